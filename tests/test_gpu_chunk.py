"""qwn_kv_chunk_attention on the GPU: chunks of new tokens over the paged cache
against the formula in 64 bits on the values that the cache holds."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

KINDS = ["bf16", "f16", "f32"]
CODECS = [1, 2, 3, 4, 5]
BAD_PAGE, BAD_SEQUENCE, BAD_LENGTH = 1 << 2, 1 << 3, 1 << 5


class Cache:
    """A pool with sequences of these lengths, and what it holds of them in fp32."""

    def __init__(self, torch, codec, lens, hk, page=16, seed=0, spare=0, outliers=True, layers=1, heads=None):
        import qwanto_b200 as qb
        g = torch.Generator("cuda").manual_seed(seed)
        pages = [-(-max(n, 1) // page) for n in lens]
        self.pool = qb.KvPool(codec, layers, hk, page, sum(pages) + spare, len(lens), max(pages) + spare,
                              max_query_heads=heads, permutation_seed=seed + 1)
        self.pool.seq_append(len(lens), counts=torch.tensor(lens, dtype=torch.int32, device="cuda"))
        self.kv = []
        for i, n in enumerate(lens):
            k, v = (torch.randn((n, hk, 128), device="cuda", generator=g) for _ in range(2))
            if outliers:
                k[..., ::37] *= 6
            if n:
                self.store(torch, i, k, v, layers - 1)
                k, v = self.held(torch, i, n, hk, layers - 1)
            self.kv.append((k, v))
        assert self.pool.check() == 0

    def store(self, torch, i, k, v, layer=0):
        self.pool.store_tokens(i, layer, 0, k.shape[0], k.contiguous(), v.contiguous())

    def held(self, torch, i, n, hk, layer=0):
        """The values that the codes stand for (min + code x step, and so on, in fp32)."""
        k, v = (torch.empty((n, hk, 128), device="cuda") for _ in range(2))
        ids = torch.tensor([i], dtype=torch.int32, device="cuda")
        begin = torch.tensor([0, n], dtype=torch.int32, device="cuda")
        first = torch.zeros(1, dtype=torch.int32, device="cuda")
        self.pool.load_tokens(layer, 1, n, 1, k, v, row_begin=begin, first_pos=first, seq_ids=ids)
        torch.cuda.synchronize()
        return k, v


def _step(codec, x):
    """How far a 16-bit operand may be from the value: int8 codes of one scale and fp16 are exact; of two
    scales, the ratio and its product are rounded; of a range, the step is rounded (15 times at most) and the sum."""
    if codec in (2, 5):
        return None
    if codec == 1:
        return x.abs() * 2.0 ** -10
    return (x.amax(-1, keepdim=True) - x.amin(-1, keepdim=True) + 2 * x.abs()) * 2.0 ** -11


def _begin(torch, counts, offset=0):
    b = [offset]
    for n in counts:
        b.append(b[-1] + n)
    return torch.tensor(b, dtype=torch.int32, device="cuda")


def _queries(torch, rows, hq, kind, seed=1):
    from promptmath import TYPES
    g = torch.Generator("cuda").manual_seed(seed)
    q = torch.randn((rows, hq, 128), device="cuda", generator=g)
    q[..., ::37] *= 6
    return q.to(TYPES[kind])


def _run(torch, c, q, counts, kind, workspace=True, out=None, one=False, layer=0, begin="yes", num_seqs=None, **more):
    from promptmath import TYPE_ID
    rows, hq, n = q.shape[0], q.shape[1], num_seqs or len(counts)
    if out is None:
        out = torch.full_like(q, 7)
    if isinstance(workspace, tuple):
        more |= {"workspace": workspace[0], "workspace_bytes": workspace[1]}
    elif workspace:
        size = c.pool.chunk_workspace(n, rows, hq)
        ws = torch.full((max(size, 16),), 255, dtype=torch.uint8, device="cuda")  # nothing in it matters
        more |= {"workspace": ws, "workspace_bytes": size}
    if not one:
        more["row_begin"] = _begin(torch, counts) if isinstance(begin, str) else begin
    c.pool.chunk_attention(layer, n, rows, TYPE_ID[kind], hq, q, out, **more)
    torch.cuda.synchronize()
    return out


def _check(torch, out, c, codec, q, counts, kind, firsts=None, window=0, scale=0.0, ids=None, at=0):
    from promptmath import assert_near, attend, seen
    for i, n in enumerate(counts):
        k, v = c.kv[ids[i] if ids else i]
        first = firsts[i] if firsts else k.shape[0] - n
        dk, dv = (None, None) if kind == "f32" else (_step(codec, k), _step(codec, v))
        # a cache's operands are f16, and so is P
        want, tol = attend(q[at:at + n], k, v, seen(first, n, k.shape[0], True, window), scale, kind,
                           None if kind == "f32" else 2.0 ** -11, dk, dv)
        assert_near(out[at:at + n], want, tol, f"sequence {i}")
        at += n


@pytest.mark.parametrize("split", [False, True])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("codec", CODECS)
def test_ragged_chunks(cuda, codec, kind, split):
    torch, lens, counts = cuda, [1, 333, 40, 700], [1, 20, 40, 133]
    c = Cache(torch, codec, lens, 2, seed=codec)
    q = _queries(torch, sum(counts), 12, kind)
    out = _run(torch, c, q, counts, kind, workspace=split)
    assert c.pool.check() == 0
    _check(torch, out, c, codec, q, counts, kind)


@pytest.mark.parametrize("split", [False, True])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("codec", CODECS)
def test_one_token_each(cuda, codec, kind, split):
    torch, lens = cuda, [1, 16, 17, 2049, 128, 127]
    c = Cache(torch, codec, lens, 2, page=64, seed=codec)
    q = _queries(torch, len(lens), 8, kind)
    out = _run(torch, c, q, [1] * len(lens), kind, workspace=split, one=True)
    assert c.pool.check() == 0
    _check(torch, out, c, codec, q, [1] * len(lens), kind)


@pytest.mark.parametrize("split", [False, True])
@pytest.mark.parametrize("codec", CODECS)
def test_many_rows(cuda, codec, split):
    """More than 128 rows a sequence: two tiles per block of threads."""
    torch, lens, counts = cuda, [1200, 515], [1000, 300]
    c = Cache(torch, codec, lens, 8, seed=codec)
    for kind in ("bf16", "f16"):
        q = _queries(torch, sum(counts), 32, kind)
        _check(torch, _run(torch, c, q, counts, kind, workspace=split), c, codec, q, counts, kind)


@pytest.mark.parametrize("split", [False, True])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("window", [1, 50, 128, 300, 5000])
def test_windows(cuda, window, kind, split):
    torch, lens, counts = cuda, [900, 333, 1], [200, 1, 1]
    c = Cache(torch, 2, lens, 2, seed=window)
    q = _queries(torch, sum(counts), 6, kind)
    _check(torch, _run(torch, c, q, counts, kind, workspace=split, window=window), c, 2, q, counts, kind, window=window)


@pytest.mark.parametrize("split", [False, True])
@pytest.mark.parametrize("kind", KINDS)
def test_long_context(cuda, kind, split):
    torch, lens, counts = cuda, [40000, 5], [3, 2]
    for codec in (2, 4):
        c = Cache(torch, codec, lens, 1, page=64, seed=codec)
        q = _queries(torch, sum(counts), 8, kind)
        _check(torch, _run(torch, c, q, counts, kind, workspace=split), c, codec, q, counts, kind)


@pytest.mark.parametrize("split", [False, True])
@pytest.mark.parametrize("kind", KINDS)
def test_positions_sequences_and_scale(cuda, kind, split):
    """Rows that are not the newest tokens, sequences in another order, a scale, a second layer."""
    torch, lens, counts, ids, firsts = cuda, [300, 77, 500], [30, 128, 7], [2, 0, 1], [100, 172, 0]
    c = Cache(torch, 2, lens, 2, seed=3, layers=2)
    q = _queries(torch, sum(counts), 4, kind)
    more = {"seq_ids": torch.tensor(ids, dtype=torch.int32, device="cuda"),
            "first_pos": torch.tensor(firsts, dtype=torch.int32, device="cuda")}
    out = _run(torch, c, q, counts, kind, workspace=split, layer=1, scale=0.05, **more)
    assert c.pool.check() == 0
    _check(torch, out, c, 2, q, counts, kind, firsts=firsts, ids=ids, scale=0.05)


@pytest.mark.parametrize("split", [False, True])
@pytest.mark.parametrize("kind", KINDS)
def test_rows_outside_their_sequence(cuda, kind, split):
    """They are zero and latch; rows of no sequence stay as they were."""
    torch, lens, counts = cuda, [300, 200, 50], [20, 10, 5]
    c = Cache(torch, 2, lens, 2, seed=4)
    q = _queries(torch, 45, 4, kind)
    begin = _begin(torch, counts, offset=4)
    firsts = torch.tensor([290, -4, 45], dtype=torch.int32, device="cuda")
    ids = torch.tensor([0, 1, 99], dtype=torch.int32, device="cuda")
    out = _run(torch, c, q, counts, kind, workspace=split, begin=begin, first_pos=firsts, seq_ids=ids)
    assert c.pool.check() == BAD_LENGTH | BAD_SEQUENCE
    assert (out[:4] == 7).all() and (out[39:] == 7).all()
    assert (out[14:24] == 0).all() and (out[24:28] == 0).all() and (out[34:39] == 0).all()
    _check(torch, out, c, 2, q, [10], kind, firsts=[290], at=4)
    _check(torch, out, c, 2, q, [6], kind, firsts=[0], ids=[1], at=28)


@pytest.mark.parametrize("split", [False, True])
def test_empty_sequences(cuda, split):
    torch, lens, counts = cuda, [0, 100, 0, 40], [0, 30, 0, 40]
    c = Cache(torch, 4, lens, 2, seed=5)
    q = _queries(torch, 70, 4, "bf16")
    out = _run(torch, c, q, counts, "bf16", workspace=split)
    assert c.pool.check() == 0
    _check(torch, out, c, 4, q, counts, "bf16")


@pytest.mark.parametrize("split", [False, True])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("codec", CODECS)
def test_masked_tokens_do_not_matter(cuda, codec, kind, split):
    """Infinities and NaN in later tokens (fp16 pages hold them; a range that is not finite makes NaN), and the
    bytes of slots behind the last token."""
    torch, lens, counts = cuda, [150, 333], [60, 33]
    c = Cache(torch, codec, lens, 2, seed=6)
    q = _queries(torch, sum(counts), 4, kind)
    dirty = Cache(torch, codec, [n + 40 for n in lens], 2, seed=6)
    for i, n in enumerate(lens):
        k, v = (torch.zeros((n + 40, 2, 128), device="cuda") for _ in range(2))
        k[n - 5:], v[n - 5:] = float("nan"), float("inf")
        v[n - 3] = float("nan")
        dirty.store(torch, i, k, v)
        k, v = _values(torch, i, lens, 6)
        ids = torch.tensor([i], dtype=torch.int32, device="cuda")
        dirty.pool.store_tokens(i, 0, 0, n - 5, k[:n - 5].contiguous(), v[:n - 5].contiguous())
    firsts = torch.tensor([l - n for l, n in zip(lens, counts)], dtype=torch.int32, device="cuda")
    out = _run(torch, dirty, q, counts, kind, workspace=split, first_pos=firsts)
    assert dirty.pool.check() == 0
    from promptmath import assert_near, attend, seen
    at = 0
    for i, n in enumerate(counts):
        k, v = c.kv[i]
        dk, dv = (None, None) if kind == "f32" else (_step(codec, k), _step(codec, v))
        want, tol = attend(q[at:at + n - 5], k, v, seen(lens[i] - n, n - 5, lens[i], True, 0), 0.0, kind,
                           None if kind == "f32" else 2.0 ** -11, dk, dv)
        assert_near(out[at:at + n - 5], want, tol, f"sequence {i}")
        at += n


def _values(torch, i, lens, seed):
    """What Cache stored."""
    g = torch.Generator("cuda").manual_seed(seed)
    for j, n in enumerate(lens):
        k, v = (torch.randn((n, 2, 128), device="cuda", generator=g) for _ in range(2))
        k[..., ::37] *= 6
        if j == i:
            return k, v


@pytest.mark.parametrize("kind", KINDS)
def test_values_that_are_not_finite_reach_the_rows_that_see_them(cuda, kind):
    torch, n = cuda, 300
    c = Cache(torch, 5, [n], 2, seed=7)
    k, v = c.kv[0]
    v = v.clone()
    v[270, 0, 5], v[130, 1, 9] = float("inf"), float("nan")
    c.store(torch, 0, k, v)
    q = _queries(torch, 100, 4, kind)
    for split in (False, True):
        out = _run(torch, c, q, [100], kind, workspace=split)
        assert torch.isnan(out[:, 2:, 9]).all() and torch.isfinite(out[:, 2:, :9]).all()
        assert not torch.isfinite(out[70:, :2, 5]).any() and torch.isfinite(out[:70, :2]).all()


@pytest.mark.parametrize("scale", [1e-4, 1.0, 3e4])
@pytest.mark.parametrize("codec", CODECS)
def test_small_and_large_values(cuda, codec, scale):
    """Values near the ends of what the cache's parameters hold, and queries of bf16 that fp16 cannot hold."""
    torch, n = cuda, 400
    c = Cache(torch, codec, [n], 2, seed=8)
    g = torch.Generator("cuda").manual_seed(9)
    k = torch.randn((n, 2, 128), device="cuda", generator=g)
    v = torch.rand((n, 2, 128), device="cuda", generator=g) * scale
    c.store(torch, 0, k, v)
    c.kv[0] = c.held(torch, 0, n, 2)
    q = (_queries(torch, 40, 4, "bf16").float() * 1e7).bfloat16()
    out = _run(torch, c, q, [40], "bf16", scale=1e-8)
    from promptmath import assert_near, attend, seen
    kk, vv = c.kv[0]
    dv = _step(codec, vv)
    dv = (0 if dv is None else dv) + torch.full_like(vv, 2.0 ** -24)  # halved values below f16's normal range
    want, tol = attend(q, kk, vv, seen(n - 40, 40, n, True, 0), 1e-8, "bf16", 2.0 ** -11,
                       (0 if _step(codec, kk) is None else _step(codec, kk)) + torch.full_like(kk, 2.0 ** -24), dv)
    assert_near(out, want, tol)


def test_bad_page_latches(cuda):
    torch = cuda
    c = Cache(torch, 2, [100], 2, seed=10)
    import qwanto_b200 as qb
    import numpy as np
    table = np.full((1,), 12345, dtype=np.int32)
    qb.check("h2d", qb.lib().qwn_kv_memcpy_h2d(c.pool.info.page_table_dev + 4, table.ctypes.data, 4))
    q = _queries(torch, 5, 4, "bf16")
    for split in (False, True):
        _run(torch, c, q, [5], "bf16", workspace=split)
        assert c.pool.check() == BAD_PAGE


def test_split_agrees_and_repeats(cuda):
    torch, lens, counts = cuda, [5000, 333, 2000], [4, 4, 4]
    c = Cache(torch, 2, lens, 4, seed=11)
    q = _queries(torch, 12, 16, "bf16")
    first = _run(torch, c, q, counts, "bf16")
    for _ in range(3):
        assert torch.equal(first, _run(torch, c, q, counts, "bf16"))
    whole = _run(torch, c, q, counts, "bf16", workspace=False)
    assert torch.equal(whole, _run(torch, c, q, counts, "bf16", workspace=False))
    assert (whole.float() - first.float()).abs().max() < 0.02


def test_capture_and_replay_as_the_sequences_grow(cuda):
    torch, lens = cuda, [130, 500]
    c = Cache(torch, 2, lens, 2, seed=12, spare=8)
    q = _queries(torch, 8, 4, "bf16")
    out, begin = torch.empty_like(q), _begin(torch, [4, 4])
    size = c.pool.chunk_workspace(2, 8, 4)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    _run(torch, c, q, [4, 4], "bf16")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.pool.chunk_attention(0, 2, 8, 3, 4, q, out, row_begin=begin, workspace=ws, workspace_bytes=size,
                               stream=torch.cuda.current_stream())
    for grow in (0, 1, 60):
        if grow:
            c.pool.seq_append(2, counts=torch.full((2,), grow, dtype=torch.int32, device="cuda"))
            for i in range(2):
                k, v = (torch.randn((grow, 2, 128), device="cuda") for _ in range(2))
                n = c.kv[i][0].shape[0]
                c.pool.store_tokens(i, 0, n, grow, k, v)
                c.kv[i] = c.held(torch, i, n + grow, 2)
        graph.replay()
        torch.cuda.synchronize()
        assert c.pool.check() == 0
        _check(torch, out, c, 2, q, [4, 4], "bf16")


def test_two_calls_at_once_with_a_workspace_each(cuda):
    torch, lens = cuda, [3000, 700]
    c = Cache(torch, 4, lens, 2, seed=13)
    q = _queries(torch, 6, 8, "f16")
    want = _run(torch, c, q, [3, 3], "f16")
    size, begin = c.pool.chunk_workspace(2, 6, 8), _begin(torch, [3, 3])
    spaces = [torch.empty(size, dtype=torch.uint8, device="cuda") for _ in range(3)]
    outs, streams = [torch.empty_like(q) for _ in range(3)], [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for _ in range(4):
        for o, w, s in zip(outs, spaces, streams):
            c.pool.chunk_attention(0, 2, 6, 2, 8, q, o, row_begin=begin, workspace=w, workspace_bytes=size, stream=s)
    torch.cuda.synchronize()
    for o in outs:
        assert torch.equal(o, want)


def test_agrees_with_decode(cuda):
    """One newest token of each sequence in fp32: what qwn_kv_decode computes."""
    torch, lens = cuda, [1, 40, 3000]
    for codec in CODECS:
        c = Cache(torch, codec, lens, 2, seed=codec + 20)
        q = _queries(torch, 3, 12, "f32")
        want = torch.empty_like(q)
        c.pool.decode(0, 3, 12, q, want)
        out = _run(torch, c, q, [1, 1, 1], "f32", one=True)
        assert (out - want).abs().max() <= 1e-4 + 1e-3 * want.abs().max()


def test_refusals(cuda):
    import qwanto_b200 as qb
    torch = cuda
    c = Cache(torch, 2, [100], 2, seed=15)
    q = _queries(torch, 4, 4, "bf16")
    out, begin = torch.empty_like(q), _begin(torch, [4])
    ws = torch.empty(c.pool.chunk_workspace(1, 4, 4), dtype=torch.uint8, device="cuda")
    good = dict(layer=0, num_seqs=1, num_rows=4, dtype=3, query_heads=4, query=q, output=out, row_begin=begin)
    c.pool.chunk_attention(**good)
    for bad in ({"layer": 1}, {"num_seqs": 2}, {"num_seqs": 0}, {"dtype": 0}, {"dtype": 4}, {"query_heads": 3},
                {"query_heads": 0}, {"query_heads": 18}, {"row_begin": None}, {"query": None}, {"output": None},
                {"scale": -1.0}, {"scale": float("nan")}, {"scale": float("inf")}, {"query_stride": 256},
                {"output_stride": 511}, {"query_stride": 516}, {"query": q.data_ptr() + 8}, {"output": q},
                {"output": q.data_ptr() + 512}, {"window": 1 << 31}, {"num_rows": 1 << 31},
                {"workspace": ws, "workspace_bytes": 16}, {"workspace": ws.data_ptr() + 4, "workspace_bytes": ws.numel()}):
        with pytest.raises(qb.QwnCudaError):
            c.pool.chunk_attention(**{**good, **bad})
    for bad in ((2, 4, 4), (1, 4, 3), (1, 4, 0), (1, 4, 18)):
        with pytest.raises(qb.QwnCudaError):
            c.pool.chunk_workspace(*bad)
    torch.cuda.synchronize()
    assert c.pool.check() == 0


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("codec", CODECS)
def test_same_bits_every_time(cuda, codec, kind):
    """Copies into a cached tile's room must not overtake the loads out of it: many calls, the same bits."""
    torch = cuda
    for lens, counts in (([5000], [512]), ([3000] * 8, [4] * 8), ([1200, 515], [1000, 300])):
        c = Cache(torch, codec, lens, 8, seed=codec + 40)
        q = _queries(torch, sum(counts), 32, kind)
        for split in (False, True):
            first = _run(torch, c, q, counts, kind, workspace=split)
            for _ in range(12):
                assert torch.equal(first, _run(torch, c, q, counts, kind, workspace=split))


def test_many_sequences(cuda):
    """More (tile, head) pairs than a workspace is made for, and just fewer."""
    torch = cuda
    for seqs, hk, heads in ((150, 8, 16), (700, 8, 64)):
        lens = [1 + (37 * i) % 200 for i in range(seqs)]
        c = Cache(torch, 2, lens, hk, seed=16)
        q = _queries(torch, seqs, heads, "bf16")
        out = _run(torch, c, q, [1] * seqs, "bf16", one=True)
        few = list(range(0, seqs, 29))
        from promptmath import assert_near, attend, seen
        for i in few:
            k, v = c.kv[i]
            want, tol = attend(q[i:i + 1], k, v, seen(lens[i] - 1, 1, lens[i], True, 0), 0.0, "bf16", 2.0 ** -11)
            assert_near(out[i:i + 1], want, tol, f"sequence {i}")
        runs = _run(torch, c, q, [1] * seqs, "bf16")  # as runs of one row
        assert (runs.float() - out.float()).abs().max() < 0.02
        c.pool.close()


@pytest.mark.parametrize("codec", CODECS)
def test_rows_up_to_a_quarter_of_a_tile_and_beyond(cuda, codec):
    """32 rows of a kv head are in the tile four times, 33 once; both in one call, over contexts that several
    blocks of threads share."""
    torch, lens, counts = cuda, [3000, 2999, 1500, 40, 5], [4, 5, 8, 9, 5]
    c = Cache(torch, codec, lens, 2, seed=codec + 60)
    for kind in ("bf16", "f16"):
        q = _queries(torch, sum(counts), 16, kind)
        _check(torch, _run(torch, c, q, counts, kind), c, codec, q, counts, kind)
        _check(torch, _run(torch, c, q, counts, kind, window=700), c, codec, q, counts, kind, window=700)


@pytest.mark.parametrize("codec", [2, 5])
def test_a_workspace_serves_smaller_calls(cuda, codec):
    """The workspace of the largest call is one for every smaller call, and sequences' sizes do not shrink it."""
    torch, lens = cuda, [1500, 400, 40, 900]
    c = Cache(torch, codec, lens, 8, seed=codec + 70)
    need = {(n, rows): c.pool.chunk_workspace(n, rows, 32) for n in (1, 2, 4) for rows in (1, 4, 33, 128, 4000, 1 << 20)}
    assert all(need[a] <= need[b] for a in need for b in need if a[0] <= b[0] and a[1] <= b[1])
    assert c.pool.chunk_workspace(4, 0, 32) == 0 and c.pool.chunk_workspace(0, 4, 32) == 0
    size = need[4, 1 << 20]
    ws = torch.full((size + 256,), 255, dtype=torch.uint8, device="cuda")
    for kind in KINDS:
        for counts, one in (([1, 1, 1, 1], True), ([1, 4, 2, 1], False), ([700, 33, 40, 5], False), ([400], False)):
            q = _queries(torch, sum(counts), 32, kind)
            out = _run(torch, c, q, counts, kind, workspace=(ws, size), one=one)
            _check(torch, out, c, codec, q, counts, kind)
    assert c.pool.check() == 0 and (ws[size:] == 255).all()


@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_sequences_that_overlap_write_nothing_else(cuda, kind):
    """row_begin that goes back makes more tiles than the rows do; they must stay within the workspace and the rows."""
    torch, n, rows = cuda, 64, 256
    c = Cache(torch, 2, [300] * n, 2, seed=80)
    q = _queries(torch, rows, 4, kind)
    begin = torch.tensor([0, rows] * (n // 2) + [0], dtype=torch.int32, device="cuda")
    size = c.pool.chunk_workspace(n, rows, 4)
    room = torch.full((size + (32 << 20),), 255, dtype=torch.uint8, device="cuda")
    out = torch.full((rows + 64, 4, 128), 7, dtype=q.dtype, device="cuda")
    _run(torch, c, q, None, kind, workspace=(room, size), begin=begin, num_seqs=n, out=out)
    assert (room[size:] == 255).all() and (out[rows:] == 7).all()
    assert c.pool.check() & ~BAD_LENGTH == 0
    # and the pool serves as before
    good = _queries(torch, n, 4, kind)
    _check(torch, _run(torch, c, good, [1] * n, kind), c, 2, good, [1] * n, kind)
