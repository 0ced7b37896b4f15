"""qwn_kv_append_rotary and qwn_kv_load_tokens on the GPU: the rotation and the
codecs against 64-bit formulas, pages byte for byte against qwn_kv_store_tokens
of rows rotated beforehand, and the attention over what was stored."""
from __future__ import annotations

import ctypes as C
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
CODECS = [1, 2, 3, 4, 5]
DTYPES = {"f32": 1, "f16": 2, "bf16": 3}
BAD_PAGE, BAD_SEQUENCE, BAD_LENGTH = 1 << 2, 1 << 3, 1 << 5


def _type(torch, name):
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def _table(torch, positions, dims):
    freq = 1.0 / (10000.0 ** (torch.arange(0, dims, 2, dtype=torch.float64, device="cuda") / max(dims, 1)))
    angle = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * freq
    return torch.cat((angle.cos(), angle.sin()), 1).float().contiguous()


def _pairs(rot, neighbours):
    return (slice(0, rot, 2), slice(1, rot, 2)) if neighbours else (slice(0, rot // 2), slice(rot // 2, rot))


def _rotated(torch, x, cs, rot, neighbours):
    """fp32, every product and sum rounded by itself: torch's elementwise operations do that."""
    y = x.float().clone()
    if rot:
        i, j = _pairs(rot, neighbours)
        a, b = x[..., i].float(), x[..., j].float()
        c, s = cs[:, None, :rot // 2], cs[:, None, rot // 2:]
        y[..., i] = a * c - b * s
        y[..., j] = b * c + a * s
    return y


def _rotated64(torch, x, cs, rot, neighbours):
    """The rotation in 64 bits, and the size of what it sums."""
    y = x.double().clone()
    size = y.abs()
    if rot:
        i, j = _pairs(rot, neighbours)
        a, b = x[..., i].double(), x[..., j].double()
        c, s = cs[:, None, :rot // 2].double(), cs[:, None, rot // 2:].double()
        y[..., i], y[..., j] = a * c - b * s, b * c + a * s
        size[..., i], size[..., j] = (a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()
    return y, size


def _held64(torch, codec, x):
    """What the cache holds of fp32 rows x, by the codec's definition in 64
    bits, and the largest distance of a stored value from it: half a step of
    the codes each way where fp32 rounds the other way, and the parameters'
    own rounding."""
    x = x.double()
    if codec == 5:
        return x.half().double(), torch.zeros_like(x)
    if codec in (1, 2):
        y = x.reshape(*x.shape[:-1], 2 if codec == 1 else 1, -1)
        top = y.abs().amax(-1, keepdim=True)
        step = torch.where(top > 0, top / 127, torch.ones_like(top))
        exact_step = step
        if codec == 2:
            step = step.half().double().clamp(2.0 ** -24, 65504.0)
        # a code's step when fp32's quotient rounds to the other side, else the scale's error on the value
        near_tie = ((y / step).abs() % 1 - 0.5).abs() < 1e-3
        code = torch.round(y / step).clamp(-127, 127)
        far = torch.where(near_tie, step, torch.zeros_like(step)) + code.abs() * exact_step * 4 * U
        if codec == 2:  # an fp16 scale whose rounding fp32 decides the other way
            far = far + code.abs() * ((exact_step - step).abs() > step * 2.0 ** -11 * 0.999) * step * 2.0 ** -10
        return (code * step).reshape(x.shape), far.expand(y.shape).reshape(x.shape)
    group = 32 if codec == 4 else 64
    y = x.reshape(*x.shape[:-1], -1, group)
    low, span = y.amin(-1, keepdim=True), y.amax(-1, keepdim=True) - y.amin(-1, keepdim=True)
    odd = torch.arange(group, device=x.device) % 2 == 1
    levels = torch.where(odd & torch.tensor(codec == 3, device=x.device), 7.0, 15.0).double()
    pos = (y - low) / span.clamp_min(1e-300) * levels
    pos = torch.where(span > 1e-8, pos, torch.zeros_like(pos))
    code = torch.floor(pos + 0.5)
    near_tie = ((pos % 1) - 0.5).abs() < 1e-4
    # the parameters are fp16, cut off: 2^-10 of them, or the smallest fp16 step
    far = (torch.where(near_tie, span / levels, torch.zeros_like(pos)) + low.abs() * 2.0 ** -10 +
           code / levels * span * 2.0 ** -10 + 2 * 2.0 ** -24 + (low.abs() + span) * 4 * U)
    return (low + code / levels * span).reshape(x.shape), far.reshape(x.shape)


HALF_ULP = {"f32": U, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def _assert_within(off, tol, what):
    bad = off > tol
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst by {float((off - tol).max())}"


class Batch:
    """A pool, and the rows of one call over some of its sequences."""

    def __init__(self, torch, codec, kind, counts, starts, kv=2, group=3, page=16, layers=2, seed=0, max_query=None,
                 spare=5, lens=None, lead=4):
        import qwanto_b200 as qb
        self.torch, self.qb = torch, qb
        self.counts, self.starts = counts, starts
        self.kv, self.hq, self.kind = kv, kv * group, kind
        n = len(counts)
        self.n, self.rows = n, sum(counts)
        lens = lens or [a + b for a, b in zip(starts, counts)]
        pages = [max(1, -(-x // page)) for x in lens]
        self.pool = qb.KvPool(codec, layers, kv, page, sum(pages) + spare, n, max(pages) + 1,
                              max_query_heads=max_query or kv * group, permutation_seed=seed + 1)
        self.twin = qb.KvPool(codec, layers, kv, page, sum(pages) + spare, n, max(pages) + 1,
                              max_query_heads=max_query or kv * group, permutation_seed=seed + 1)
        self.lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
        for p in (self.pool, self.twin):
            p.seq_append(n, counts=self.lens)
        g = torch.Generator("cuda").manual_seed(seed)
        # rows of the projection's output: `lead` values before the heads, as many and 4 more after (lead 4: rows
        # start on 4 values, lead 8 and no more after: on 16 bytes)
        self.lead = lead
        width = (self.hq + 2 * kv) * 128
        self.wide = width + 2 * lead + (4 if lead == 4 else 0)
        self.qkv = torch.full((self.rows, self.wide), float("nan"), device="cuda", dtype=_type(torch, kind))
        self.qkv[:, lead:lead + width] = torch.randn((self.rows, width), device="cuda", generator=g).to(self.qkv.dtype)
        x = self.qkv[:, lead:lead + width].view(self.rows, -1, 128) if self.rows else self.qkv.new_zeros((0, self.hq + 2 * kv, 128))
        self.q, self.k, self.v = x[:, :self.hq], x[:, self.hq:self.hq + kv], x[:, self.hq + kv:]
        self.begin = torch.tensor([0] + list(np.cumsum(counts)), dtype=torch.int32, device="cuda")
        self.first = torch.tensor(starts, dtype=torch.int32, device="cuda")
        pos = [np.arange(s, s + c) for s, c in zip(starts, counts)]
        self.pos = torch.tensor(np.concatenate(pos) if pos else [], dtype=torch.int64, device="cuda")

    def parts(self):
        """query, key, value where the rows' heads begin."""
        at = self.lead
        return self.qkv[:, at:], self.qkv[:, at + self.hq * 128:], self.qkv[:, at + (self.hq + self.kv) * 128:]

    def append(self, layer, rot, neighbours, table, out, out_kind, **over):
        q, k, v = self.parts()
        args = dict(query=q, query_heads=self.hq, query_out=out, query_out_dtype=DTYPES[out_kind], rotations=table,
                    rotary_dim=rot, max_position=0 if table is None else table.shape[0], neighbours=neighbours,
                    row_begin=self.begin, first_pos=self.first, query_stride=self.wide, key_stride=self.wide,
                    value_stride=self.wide)
        args.update(over)
        self.pool.append_rotary(layer, self.n, self.rows, DTYPES[self.kind], k, v, **args)

    def store_twin(self, layer, k, v):
        """The same rows through the fp32 entry point."""
        at = 0
        for i, (c, s) in enumerate(zip(self.counts, self.starts)):
            if c:
                self.twin.store_tokens(i, layer, s, c, k[at:at + c].contiguous(), v[at:at + c].contiguous())
            at += c
        self.torch.cuda.synchronize()

    def assert_pages_equal(self):
        t, u = self.pool.page_table(), self.twin.page_table()
        assert np.array_equal(t, u)
        for pg in sorted({int(x) for x in t.ravel() if x >= 0}):
            assert np.array_equal(self.pool.page(pg), self.twin.page(pg)), f"page {pg}"

    def close(self):
        self.pool.close()
        self.twin.close()


COUNTS = ([1, 0, 15, 16, 17, 40, 3], [0, 5, 16, 3, 31, 12, 47])  # rows of each sequence, and where they start


@pytest.mark.parametrize("codec", CODECS)
@pytest.mark.parametrize("kind,out_kind,rot,neighbours,page", [
    ("f32", "f32", 128, False, 16), ("bf16", "f32", 128, True, 32), ("f16", "bf16", 64, False, 64),
    ("bf16", "f16", 8, True, 16), ("f32", "bf16", 96, False, 16), ("f16", "f16", 0, False, 48),
    ("bf16", "bf16", 40, False, 16)])
@pytest.mark.parametrize("lead", [4, 8])
def test_ragged_rows(cuda, codec, kind, out_kind, rot, neighbours, page, lead):
    torch = cuda
    b = Batch(torch, codec, kind, *COUNTS, page=page, seed=codec * 10 + rot, lead=lead)
    try:
        # tokens that are there already must stay: fill everything first
        old = torch.randn((200, b.kv, 128), device="cuda", generator=torch.Generator("cuda").manual_seed(77))
        for p in (b.pool, b.twin):
            for i, n in enumerate(b.lens.tolist()):
                if n:
                    p.store_tokens(i, 1, 0, n, old[:n], old[-n:].contiguous())
        table = _table(torch, 128, rot) if rot else None
        out = torch.full((b.rows, b.hq, 128), float("nan"), device="cuda", dtype=_type(torch, out_kind))
        b.append(1, rot, neighbours, table, out, out_kind)
        assert b.pool.check() == 0
        cs = table[b.pos] if rot else None
        q64, size = _rotated64(torch, b.q, cs, rot, neighbours)
        # two products and a sum, then the output's rounding
        tol = 3 * U * size * bool(rot) + HALF_ULP[out_kind] * (q64.abs() + 3 * U * size) + 2.0 ** -25
        _assert_within((out.double() - q64).abs(), tol, "query")
        k32 = _rotated(torch, b.k, cs, rot, neighbours)
        b.store_twin(1, k32, b.v.float())
        b.assert_pages_equal()
        # and back: the codes' values
        for back_kind in ("f32", "bf16", "f16"):
            bk = torch.full((b.rows, b.kv, 128), float("nan"), device="cuda", dtype=_type(torch, back_kind))
            bv = torch.full_like(bk, float("nan"))
            b.pool.load_tokens(1, b.n, b.rows, DTYPES[back_kind], bk, bv, row_begin=b.begin, first_pos=b.first)
            for got, x in ((bk, k32), (bv, b.v.float())):
                want, far = _held64(torch, codec, x)
                _assert_within((got.double() - want).abs(), far + HALF_ULP[back_kind] * (want.abs() + far) + 2.0 ** -25,
                               f"held {back_kind}")
        assert b.pool.check() == 0
    finally:
        b.close()


@pytest.mark.parametrize("codec", CODECS)
@pytest.mark.parametrize("kv,group,kind", [(1, 1, "f32"), (2, 6, "bf16"), (8, 8, "f16")])
def test_one_token_each_then_attention(cuda, codec, kv, group, kind):
    """A decode step: the newest token of every sequence, then qwn_kv_decode
    over the stored rows, against softmax attention in 64 bits over the rows
    read back; the first token of a sequence is one of the steps."""
    torch = cuda
    lens = [1, 2, 16, 17, 64, 129]
    b = Batch(torch, codec, kind, [1] * 6, [n - 1 for n in lens], kv=kv, group=group, seed=kv)
    try:
        g = torch.Generator("cuda").manual_seed(4)
        for i, n in enumerate(lens):
            if n > 1:
                b.pool.store_tokens(i, 0, 0, n - 1, torch.randn((n - 1, kv, 128), device="cuda", generator=g),
                                    torch.randn((n - 1, kv, 128), device="cuda", generator=g))
        table = _table(torch, 256, 128)
        q = torch.full((6, b.hq, 128), float("nan"), device="cuda")
        b.append(0, 128, False, table, q, "f32", row_begin=None, first_pos=None)
        out = torch.empty_like(q)
        b.pool.decode(0, 6, b.hq, q, out)
        assert b.pool.check() == 0
        rows = sum(lens)
        begin = torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32, device="cuda")
        k, v = torch.empty((rows, kv, 128), device="cuda"), torch.empty((rows, kv, 128), device="cuda")
        b.pool.load_tokens(0, 6, rows, 1, k, v, row_begin=begin)
        for i, n in enumerate(lens):
            ki, vi = (t[int(begin[i]):int(begin[i + 1])].double().repeat_interleave(group, 1) for t in (k, v))
            w = torch.softmax(torch.einsum("hd,thd->ht", q[i].double(), ki) / math.sqrt(128), -1)
            want = torch.einsum("ht,thd->hd", w, vi)
            _assert_within((out[i].double() - want).abs(), 1e-4 + 1e-3 * want.abs(), f"attention of {n} tokens")
        cs = table[torch.tensor([n - 1 for n in lens], device="cuda")]
        last = torch.tensor([int(x) - 1 for x in begin[1:]], device="cuda")
        for got, x in ((k[last], _rotated(torch, b.k, cs, 128, False)), (v[last], b.v.float())):
            want, far = _held64(torch, codec, x)
            _assert_within((got.double() - want).abs(), far + U * want.abs() + 2.0 ** -25, "newest token")
    finally:
        b.close()


@pytest.mark.parametrize("lead", [4, 8])
def test_sequence_ids_in_any_order_and_newest_rows(cuda, lead):
    """seq_ids picks the sequences; without first_pos the rows are each one's newest."""
    torch = cuda
    b = Batch(torch, 2, "f32", [5, 20, 1], [30, 7, 16], seed=3, lead=lead)
    try:
        ids = torch.tensor([2, 0, 1], dtype=torch.int32, device="cuda")
        order = [1, 20, 5]  # rows per entry: sequence 2's 1, 0's ... in the order of ids
        # entry 0 -> sequence 2 (len 17), entry 1 -> sequence 0 (len 35), entry 2 -> sequence 1 (len 27)
        begin = torch.tensor([0] + list(np.cumsum(order)), dtype=torch.int32, device="cuda")
        table = _table(torch, 64, 128)
        out = torch.empty((b.rows, b.hq, 128), device="cuda")
        b.append(1, 128, False, table, out, "f32", row_begin=begin, first_pos=None, seq_ids=ids)
        assert b.pool.check() == 0
        pos, at = [], 0
        for i, c in zip((2, 0, 1), order):
            n = int(b.lens[i])
            pos += list(range(n - c, n))
        cs = table[torch.tensor(pos, device="cuda")]
        k32 = _rotated(torch, b.k, cs, 128, False)
        for i, c in zip((2, 0, 1), order):
            n = int(b.lens[i])
            b.twin.store_tokens(i, 1, n - c, c, k32[at:at + c].contiguous(), b.v[at:at + c].float().contiguous())
            at += c
        torch.cuda.synchronize()
        b.assert_pages_equal()
        bk, bv = torch.zeros((b.rows, b.kv, 128), device="cuda"), torch.zeros((b.rows, b.kv, 128), device="cuda")
        b.pool.load_tokens(1, 3, b.rows, 1, bk, None, row_begin=begin, seq_ids=ids)
        want, far = _held64(torch, 2, k32)
        _assert_within((bk.double() - want).abs(), far + U * want.abs() + 2.0 ** -25, "keys alone")
        assert not bv.any()
    finally:
        b.close()


def test_angles_apart_from_cache_positions(cuda):
    """After an eviction a token's place in the cache is not its position."""
    torch = cuda
    b = Batch(torch, 5, "f32", [9, 39], [0, 20], seed=6, lead=8)
    try:
        table = _table(torch, 5000, 128)
        angles = torch.randint(0, 5000, (b.rows,), device="cuda", dtype=torch.int32)
        out = torch.empty((b.rows, b.hq, 128), device="cuda")
        b.append(0, 128, False, table, out, "f32", rotary_pos=angles)
        assert b.pool.check() == 0
        assert torch.equal(out, _rotated(torch, b.q, table[angles.long()], 128, False))
        b.store_twin(0, _rotated(torch, b.k, table[angles.long()], 128, False), b.v.float())
        b.assert_pages_equal()
    finally:
        b.close()


@pytest.mark.parametrize("rot,neighbours", [(128, False), (64, True), (64, False), (40, False)])
@pytest.mark.parametrize("lead", [4, 8])
def test_query_in_place_and_no_query(cuda, rot, neighbours, lead):
    torch = cuda
    b = Batch(torch, 4, "f32", [63], [2], seed=9, lead=lead)
    try:
        table = _table(torch, 70, rot)
        q = b.q.contiguous().clone()
        want = _rotated(torch, q, table[b.pos], rot, neighbours)
        b.append(0, rot, neighbours, table, q, "f32", query=q, query_stride=0)
        b.append(0, rot, neighbours, table, None, "f32", query=None, query_heads=0)
        assert b.pool.check() == 0
        assert torch.equal(q, want)
    finally:
        b.close()


@pytest.mark.parametrize("lead", [4, 8])
@pytest.mark.parametrize("codec", [1, 2, 3, 4, 5])
def test_beyond_numbers_in_other_rows(cuda, codec, lead):
    """NaN and infinities of one row leave the other rows of its tile alone, and
    are stored as the fp32 entry point stores them; so is a row of zeros with a
    negative one among them."""
    torch = cuda
    b = Batch(torch, codec, "f32", [44], [3], seed=2, lead=lead)
    try:
        b.k[5, 0, 3], b.k[9, 1, 77], b.v[5, 1, 0] = float("nan"), float("inf"), float("-inf")
        b.k[20, 0], b.v[21, 1] = 0.0, 0.0
        b.v[21, 1, 40], b.v[21, 1, 100] = -0.0, 2.0
        b.v[20, 0, 64:] = float("nan")
        table = _table(torch, 64, 128)
        out = torch.empty((b.rows, b.hq, 128), device="cuda")
        b.append(0, 128, False, table, out, "f32")
        assert b.pool.check() == 0
        bk, bv = (torch.empty((b.rows, b.kv, 128), device="cuda") for _ in range(2))
        b.pool.load_tokens(0, 1, b.rows, 1, bk, bv, row_begin=b.begin, first_pos=b.first)
        keep = torch.tensor([i for i in range(44) if i not in (5, 9, 20, 21)], device="cuda")
        for got, x in ((bk, _rotated(torch, b.k, table[b.pos], 128, False)), (bv, b.v.float())):
            want, far = _held64(torch, codec, x[keep])
            _assert_within((got[keep].double() - want).abs(), far + U * want.abs() + 2.0 ** -25, "other rows")
        b.store_twin(0, _rotated(torch, b.k, table[b.pos], 128, False), b.v.float())
        b.assert_pages_equal()
    finally:
        b.close()


@pytest.mark.parametrize("lead", [4, 8])
def test_rows_that_cannot_be_stored(cuda, lead):
    """A bad sequence id, position, angle or run: latched, nothing stored, zero rows out; the others go on."""
    torch = cuda
    b = Batch(torch, 2, "f32", [4, 4, 4], [0, 3, 10], seed=1, lead=lead)
    try:
        table = _table(torch, 13, 128)  # positions 13 of sequence 2 are outside
        out = torch.full((b.rows, b.hq, 128), float("nan"), device="cuda")
        b.append(0, 128, False, table, out, "f32")
        assert b.pool.check() == BAD_LENGTH
        assert not out[11].any() and torch.equal(out[:11], _rotated(torch, b.q, table[b.pos.clamp(max=12)], 128, False)[:11])
        big = _table(torch, 64, 128)
        before = [b.pool.page(p).copy() for p in range(8)]
        for over, bits, rows in (
                ({"seq_ids": torch.tensor([0, -1, 3], dtype=torch.int32, device="cuda")}, BAD_SEQUENCE, range(4, 12)),
                ({"first_pos": torch.tensor([0, 5, -2], dtype=torch.int32, device="cuda")}, BAD_LENGTH, [6, 7, 8, 9]),
                ({"first_pos": torch.tensor([2 ** 31 - 2, 3, 10], dtype=torch.int32, device="cuda")}, BAD_LENGTH, range(4)),
                ({"row_begin": torch.tensor([0, 4, 8, 10], dtype=torch.int32, device="cuda")}, BAD_LENGTH, [10, 11]),
                ({"row_begin": torch.tensor([2, 4, 8, 12], dtype=torch.int32, device="cuda")}, BAD_LENGTH, [0, 1])):
            out.fill_(float("nan"))
            b.append(0, 128, False, big, out, "f32", **over)
            assert b.pool.check() == bits, over
            for r in range(12):
                assert out[r].any() == (r not in rows) and not out[r].isnan().any(), (over, r)
        assert len(before) == 8
        key = torch.full((b.rows, b.kv, 128), float("nan"), device="cuda")
        b.pool.load_tokens(0, 3, b.rows, 1, key, None, row_begin=b.begin,
                           first_pos=torch.tensor([0, 5, 10], dtype=torch.int32, device="cuda"))
        assert b.pool.check() == BAD_LENGTH
        assert not key[6:8].any() and not key.isnan().any() and key[:6].any() and key[8:].any()
        # an empty sequence has no newest token
        b.pool.reset()
        out.fill_(float("nan"))
        b.append(0, 128, False, big, out, "f32")
        assert b.pool.check() == BAD_LENGTH and not out.any()
    finally:
        b.close()


def test_long_cache_offsets_pass_32_bits(cuda):
    """A page whose bytes start beyond 4 GiB, and a position beyond 65536."""
    import qwanto_b200 as qb
    torch = cuda
    n = 66000  # of 16: 4125 pages
    pages = n // 16
    pool = qb.KvPool(5, 17, 8, 16, pages, 1, pages, max_query_heads=8)  # pages of 1.1 MB
    try:
        assert pool.info.page_bytes * (pages - 1) > 1 << 32
        pool.seq_append(1, counts=torch.tensor([n], dtype=torch.int32, device="cuda"))
        table = _table(torch, n, 128)
        g = torch.Generator("cuda").manual_seed(1)
        rows = 40
        x = torch.randn((rows, 24, 128), device="cuda", generator=g).bfloat16()
        out = torch.empty((rows, 8, 128), device="cuda")
        begin = torch.tensor([0, rows], dtype=torch.int32, device="cuda")
        for first in (0, 32760, n - rows):
            where = torch.tensor([first], dtype=torch.int32, device="cuda")
            pool.append_rotary(16, 1, rows, 3, x[:, 8:], x[:, 16:], query=x, query_heads=8, query_out=out, rotations=table,
                               rotary_dim=128, max_position=n, row_begin=begin, first_pos=where, query_stride=24 * 128,
                               key_stride=24 * 128, value_stride=24 * 128)
            k, v = (torch.empty((rows, 8, 128), device="cuda") for _ in range(2))
            pool.load_tokens(16, 1, rows, 1, k, v, row_begin=begin, first_pos=where)
            assert pool.check() == 0
            cs = table[first:first + rows]
            assert torch.equal(k, _rotated(torch, x[:, 8:16], cs, 128, False).half().float())
            assert torch.equal(v, x[:, 16:].float().half().float())
            assert torch.equal(out, _rotated(torch, x[:, :8], cs, 128, False))
    finally:
        pool.close()


def test_a_stream_of_its_own(cuda):
    torch = cuda
    b = Batch(torch, 1, "bf16", [300, 200], [0, 40], seed=12, lead=8)
    try:
        table = _table(torch, 512, 128)
        out = torch.empty((b.rows, b.hq, 128), device="cuda")
        s = torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            b.qkv *= 2  # written on the stream that the call reads on
            b.append(0, 128, False, table, out, "f32", stream=s)
            bk, bv = (torch.empty((b.rows, b.kv, 128), device="cuda") for _ in range(2))
            b.pool.load_tokens(0, 2, b.rows, 1, bk, bv, row_begin=b.begin, first_pos=b.first, stream=s)
            copy = bk + 0
        s.synchronize()
        k32 = _rotated(torch, b.k, table[b.pos], 128, False)
        want, far = _held64(torch, 1, k32)
        _assert_within((copy.double() - want).abs(), far + U * want.abs() + 2.0 ** -25, "keys")
        assert torch.equal(out, _rotated(torch, b.q, table[b.pos], 128, False))
    finally:
        b.close()


def test_refusals(cuda):
    from qwanto_b200 import _lib
    torch = cuda
    b = Batch(torch, 2, "bf16", [4, 4], [0, 0], seed=1)
    try:
        table = _table(torch, 64, 128)
        out = torch.empty((b.rows, b.hq, 128), device="cuda")
        q, k, v = b.parts()

        def append(**over):
            r = _lib.init(_lib.AppendRotaryRequest())
            r.num_seqs, r.num_rows, r.dtype, r.query_heads, r.query_out_dtype = 2, 8, 3, b.hq, 1
            r.rotary_dim, r.max_position, r.rotations_dev, r.row_begin_dev = 128, 64, table.data_ptr(), b.begin.data_ptr()
            r.query_stride = r.key_stride = r.value_stride = b.wide
            r.query_dev, r.key_dev, r.value_dev = q.data_ptr(), k.data_ptr(), v.data_ptr()
            r.query_out_dev = out.data_ptr()
            for key, x in over.items():
                setattr(r, key, x)
            return _lib.lib().qwn_kv_append_rotary(C.byref(b.pool.h), C.byref(r))

        assert append() == 0 and append(num_rows=0, key_dev=None) == 0
        for over in ({"layer": 2}, {"num_seqs": 3}, {"num_seqs": 0}, {"dtype": 0}, {"dtype": 4}, {"row_begin_dev": None},
                     {"rotary_dim": 4}, {"rotary_dim": 136}, {"rotary_style": 2}, {"rotations_dev": None},
                     {"rotations_dev": table.data_ptr() + 4}, {"max_position": 0}, {"query_heads": 5},
                     {"query_heads": b.hq + 2}, {"query_dev": None}, {"query_out_dev": None}, {"query_out_dtype": 9},
                     {"key_dev": None}, {"value_dev": None}, {"key_stride": 2}, {"key_stride": b.wide + 2},
                     {"key_dev": k.data_ptr() + 2}, {"query_out_dev": out.data_ptr() + 8}):
            assert append(**over) == -1, over
            assert "qwn_kv_append_rotary" in _lib.last_error()

        def load(**over):
            r = _lib.init(_lib.LoadTokensRequest())
            r.num_seqs, r.num_rows, r.dtype, r.row_begin_dev = 2, 8, 1, b.begin.data_ptr()
            r.key_out_dev = out.data_ptr()
            for key, x in over.items():
                setattr(r, key, x)
            return _lib.lib().qwn_kv_load_tokens(C.byref(b.pool.h), C.byref(r))

        assert load() == 0 and load(num_rows=0) == 0
        for over in ({"layer": 2}, {"num_seqs": 3}, {"num_seqs": 0}, {"dtype": 0}, {"row_begin_dev": None},
                     {"key_out_dev": None}, {"key_stride": 3}, {"key_stride": 258}, {"value_out_dev": out.data_ptr() + 4}):
            assert load(**over) == -1, over
            assert "qwn_kv_load_tokens" in _lib.last_error()
        assert b.pool.check() == 0
    finally:
        b.close()


@pytest.mark.parametrize("lead", [4, 8])
@pytest.mark.parametrize("codec", CODECS)
def test_rows_that_cannot_be_stored_leave_the_pages_alone(cuda, codec, lead):
    """Of a call with bad rows, the pages hold the good rows and nothing else: every
    byte of every page equals a pool's that only got the good ones."""
    torch = cuda
    counts, starts = [40, 33, 20], [0, 5, 12]
    b = Batch(torch, codec, "f32", counts, starts, seed=codec, lead=lead)
    try:
        g = torch.Generator("cuda").manual_seed(40)
        table = _table(torch, 64, 128)
        out = torch.empty((b.rows, b.hq, 128), device="cuda")
        held = sorted({int(p) for p in b.pool.page_table().ravel() if p >= 0})
        total = b.pool.total_pages

        def ints(*x):
            return torch.tensor(x, dtype=torch.int32, device="cuda")

        far = torch.arange(b.rows, device="cuda", dtype=torch.int32) % 60
        far[50], far[51] = 64, -1  # angles outside the table
        # what is wrong, the status, the rows stored: (row, sequence, position)
        normal = [(r, i, s + j) for i, (c, s, at) in enumerate(zip(counts, starts, (0, 40, 73)))
                  for j, r in enumerate(range(at, at + c))]
        cases = [
            ({"seq_ids": ints(0, -1, 3)}, BAD_SEQUENCE, [x for x in normal if x[1] == 0]),
            ({"seq_ids": ints(-2 ** 31, 1, 2 ** 31 - 1)}, BAD_SEQUENCE, [x for x in normal if x[1] == 1]),
            ({"first_pos": ints(-3, 5, 12)}, BAD_LENGTH,
             [(r, i, p - 3 if i == 0 else p) for r, i, p in normal if i or p >= 3]),
            ({"first_pos": ints(0, 5, 20)}, BAD_LENGTH,
             [(r, i, p + 8 if i == 2 else p) for r, i, p in normal if i < 2 or p + 8 < 32]),
            ({"first_pos": ints(2 ** 31 - 5, 5, 12)}, BAD_LENGTH, [x for x in normal if x[1]]),
            ({"first_pos": ints(-2 ** 31, 5, 12)}, BAD_LENGTH, [x for x in normal if x[1]]),
            ({"row_begin": ints(7, 40, 73, 80), "first_pos": ints(7, 5, 12)}, BAD_LENGTH,
             [x for x in normal if 7 <= x[0] < 80]),
            ({"rotary_pos": far}, BAD_LENGTH, [x for x in normal if x[0] not in (50, 51)]),
        ]
        for over, bits, good in cases:
            n = int(b.lens.max())
            old = torch.randn((n, b.kv, 128), device="cuda", generator=g)
            for p in (b.pool, b.twin):
                for layer in range(2):
                    for i, m in enumerate(b.lens.tolist()):
                        p.store_tokens(i, layer, 0, m, old[:m], old[-m:].contiguous())
            before = [b.pool.page(p).copy() for p in range(total)]
            b.append(1, 128, False, table, out, "f32", **over)
            assert b.pool.check() == bits, over
            angle = far.long() if "rotary_pos" in over else None
            rows = torch.tensor([r for r, _, _ in good], device="cuda")
            where = angle[rows] if angle is not None else torch.tensor([p for _, _, p in good], device="cuda")
            k32 = _rotated(torch, b.k[rows], table[where], 128, False)
            for at, (r, i, p) in enumerate(good):
                b.twin.store_tokens(i, 1, p, 1, k32[at:at + 1].contiguous(), b.v[r:r + 1].contiguous())
            torch.cuda.synchronize()
            for p in range(total):
                want = b.twin.page(p) if p in held else before[p]
                assert np.array_equal(b.pool.page(p), want), (over, p)
    finally:
        b.close()
