"""qwn_kv_append_rotary with positions on three axes: bit for bit what one axis
gives with a table of every row's own angles, and the formula in 64 bits."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

CODECS = [1, 2, 3, 4, 5]
BAD_LENGTH = 1 << 5
POSITIONS = 700
U = 2.0 ** -24


def _table(torch, dims):
    freq = 1.0 / (10000.0 ** (torch.arange(0, dims, 2, dtype=torch.float64, device="cuda") / dims))
    angle = torch.arange(POSITIONS, dtype=torch.float64, device="cuda")[:, None] * freq
    return torch.cat((angle.cos(), angle.sin()), 1).float().contiguous()


class Batch:
    def __init__(self, torch, codec, kind, counts, firsts, hk=2, group=3, lead=0, seed=0):
        import qwanto_b200 as qb
        from promptmath import TYPE_ID, TYPES
        g = torch.Generator("cuda").manual_seed(seed)
        self.torch, self.counts, self.hk, self.hq, self.rows = torch, counts, hk, hk * group, sum(counts)
        self.kind, self.dtype, self.type = kind, TYPE_ID[kind], TYPES[kind]
        self.wide = (group + 2) * hk * 128 + lead  # rows off the 16-byte grid go one by one
        self.qkv = torch.randn((self.rows, self.wide), device="cuda", generator=g).to(self.type)
        self.lens = [f + n for f, n in zip(firsts, counts)]
        pages = [-(-n // 16) for n in self.lens]
        self.make = lambda: qb.KvPool(codec, 1, hk, 16, sum(pages), len(counts), max(pages), max_query_heads=self.hq)
        b = [0]
        for n in counts:
            b.append(b[-1] + n)
        self.begin = torch.tensor(b, dtype=torch.int32, device="cuda")
        self.pos = torch.randint(0, POSITIONS, (3, self.rows), device="cuda", generator=g).int()

    def append(self, dims, neighbours, table, pos, sections, one=False, out_kind="f32"):
        from promptmath import TYPE_ID, TYPES
        torch, q = self.torch, self.hq * 128
        pool = self.make()
        pool.seq_append(len(self.counts), counts=torch.tensor(self.lens, dtype=torch.int32, device="cuda"))
        out = torch.full((self.rows, self.hq, 128), 5.0, dtype=TYPES[out_kind], device="cuda")
        pool.append_rotary(0, len(self.counts), self.rows, self.dtype, self.qkv[:, q:], self.qkv[:, q + self.hk * 128:],
                           query=self.qkv, query_heads=self.hq, query_out=out, query_out_dtype=TYPE_ID[out_kind],
                           rotations=table, rotary_dim=dims, max_position=table.shape[0], neighbours=neighbours,
                           row_begin=None if one else self.begin, rotary_pos=pos, rotary_sections=sections,
                           query_stride=self.wide, key_stride=self.wide, value_stride=self.wide)
        k, v = (torch.empty((self.rows, self.hk, 128), device="cuda") for _ in range(2))
        pool.load_tokens(0, len(self.counts), self.rows, 1, k, v, row_begin=None if one else self.begin)
        status = pool.check()
        pool.close()
        return out, k, v, status

    def own_angles(self, table, sections):
        """A table with a row for each row of the batch."""
        torch = self.torch
        axis = torch.repeat_interleave(torch.arange(3, device="cuda"), torch.tensor(sections, device="cuda")).repeat(2)
        return table.gather(0, self.pos.long()[axis].T).contiguous()


def _same(torch, a, b):
    for x, y in zip(a[:3], b[:3]):
        assert torch.equal(x, y)
    assert a[3] == b[3] == 0


@pytest.mark.parametrize("lead", [0, 4])
@pytest.mark.parametrize("neighbours", [False, True])
@pytest.mark.parametrize("sections", [(16, 24, 24), (64, 0, 0), (0, 32, 32), (4, 4, 8), (12, 20, 16), (0, 0, 4)])
def test_sections(cuda, sections, neighbours, lead):
    torch, dims = cuda, 2 * sum(sections)
    b = Batch(torch, 2, "bf16", [40, 1, 77], [0, 30, 5], lead=lead, seed=dims)
    table = _table(torch, dims)
    got = b.append(dims, neighbours, table, b.pos, sections)
    alone = torch.arange(b.rows, dtype=torch.int32, device="cuda")
    _same(torch, got, b.append(dims, neighbours, b.own_angles(table, sections), alone, None))
    # and in 64 bits: a pair is a complex number, its rotation a product
    x = b.qkv[:, :b.hq * 128].double().reshape(b.rows, b.hq, 128)
    cs = b.own_angles(table, sections).double()
    turn = torch.complex(cs[:, :dims // 2], cs[:, dims // 2:])[:, None]
    i, j = (slice(0, dims, 2), slice(1, dims, 2)) if neighbours else (slice(0, dims // 2), slice(dims // 2, dims))
    z = torch.complex(x[..., i], x[..., j])
    size = (z.real.abs() + z.imag.abs()) * 1.0
    want = x.clone()
    want[..., i], want[..., j] = (z * turn).real, (z * turn).imag
    tol = torch.zeros_like(x)
    tol[..., i] = tol[..., j] = 3 * U * size  # two products and a sum, each rounded
    assert ((got[0].double() - want).abs() <= tol).all()


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("codec", CODECS)
def test_codecs_and_types(cuda, codec, kind):
    torch, sections = cuda, (16, 24, 24)
    table = _table(torch, 128)
    for one, counts, firsts in ((False, [130, 3, 16], [7, 0, 100]), (True, [1, 1, 1], [0, 15, 200])):
        b = Batch(torch, codec, kind, counts, firsts, seed=codec)
        alone = torch.arange(b.rows, dtype=torch.int32, device="cuda")
        got = b.append(128, False, table, b.pos, sections, one=one, out_kind=kind)
        _same(torch, got, b.append(128, False, b.own_angles(table, sections), alone, None, one=one, out_kind=kind))


@pytest.mark.parametrize("lead", [0, 4])
@pytest.mark.parametrize("axis", [0, 1, 2])
def test_positions_outside_the_table(cuda, axis, lead):
    """They matter on axes that have pairs only; such a row is zero and stores nothing."""
    torch = cuda
    b = Batch(torch, 2, "f32", [20, 18], [0, 0], lead=lead, seed=axis)
    table = _table(torch, 128)
    for bad in (-1, POSITIONS):
        b.pos[:, 9] = 3
        good = b.append(128, False, table, b.pos, (16, 24, 24))
        b.pos[axis, 9] = bad
        out, k, v, status = b.append(128, False, table, b.pos, (16, 24, 24))
        assert status == BAD_LENGTH and not out[9].any()
        keep = torch.arange(b.rows, device="cuda") != 9
        assert torch.equal(out[keep], good[0][keep]) and torch.equal(k[keep], good[1][keep])
        none = [32, 32, 32]
        none[axis] = 0
        assert b.append(128, False, table, b.pos, none)[3] == 0


def test_refusals(cuda):
    import qwanto_b200 as qb
    torch = cuda
    b = Batch(torch, 2, "bf16", [4, 4], [0, 0])
    table = _table(torch, 128)
    assert b.append(128, False, table, b.pos, (16, 24, 24))[3] == 0
    for sections in ((16, 24, 20), (18, 22, 24), (64, 4, 0), (0, 0, 60), (2, 2, 60)):
        with pytest.raises(qb.QwnCudaError):
            b.append(128, False, table, b.pos, sections)
    for sections in ((-4, 34, 34), (256, 0, 0)):
        with pytest.raises(ValueError):
            b.append(128, False, table, b.pos, sections)
    with pytest.raises(qb.QwnCudaError):
        b.append(128, False, table, None, (16, 24, 24))
