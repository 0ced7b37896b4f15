"""Outputs that share a buffer with inputs: rows side by side and rows in place
give what separate buffers give."""
from __future__ import annotations

import ctypes as C

import pytest

pytestmark = pytest.mark.gpu

DTYPES = {"f32": 1, "f16": 2, "bf16": 3}


def _type(torch, name):
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


@pytest.mark.parametrize("kind", sorted(DTYPES))
@pytest.mark.parametrize("rows,width", [(1, 64), (700, 4096), (2500, 257)])
@pytest.mark.parametrize("where", ["residual", "x", "beside x", "one wide row"])
def test_norm_residual_shares_a_buffer(cuda, kind, rows, width, where):
    import qwanto_b200 as qb
    torch = cuda
    if where == "one wide row":
        rows = 1
    dt = _type(torch, kind)
    g = torch.Generator("cuda").manual_seed(rows + width)
    both = torch.randn((rows, 2 * width), device="cuda", generator=g).to(dt)
    other = torch.randn((rows, width), device="cuda", generator=g).to(dt)
    x, beside = both[:, :width], both[:, width:]
    want = [torch.empty((rows, width), dtype=torch.int8, device="cuda"), torch.empty(rows, device="cuda"),
            torch.empty((rows, width), device="cuda", dtype=dt)]
    qb.rmsnorm_q8(x, rows, width, DTYPES[kind], want[0], want[1], residual=other, residual_out=want[2],
                  x_stride=2 * width)
    torch.cuda.synchronize()
    out, stride = {"residual": (other, width), "x": (x, 2 * width), "beside x": (beside, 2 * width),
                   "one wide row": (x, 0)}[where]
    codes, scales = torch.empty_like(want[0]), torch.empty_like(want[1])
    qb.rmsnorm_q8(x, rows, width, DTYPES[kind], codes, scales, residual=other, residual_out=out, x_stride=2 * width,
                  residual_out_stride=stride)
    torch.cuda.synchronize()
    assert torch.equal(codes, want[0]) and torch.equal(scales, want[1]) and torch.equal(out, want[2])


def _pool(qb, torch, rows, kv=2, hq=6):
    pool = qb.KvPool(2, 1, kv, 16, 64, 1, 64, max_query_heads=hq)
    pool.seq_append(1, counts=torch.tensor([rows], dtype=torch.int32, device="cuda"))
    return pool


@pytest.mark.parametrize("kind,out_kind", [("f32", "f32"), ("bf16", "bf16"), ("f16", "bf16"), ("bf16", "f16")])
@pytest.mark.parametrize("rows,fused", [(70, False), (1, True)])
@pytest.mark.parametrize("rot,neighbours", [(128, False), (64, False), (96, True)])
def test_queries_in_place(cuda, kind, out_kind, rows, fused, rot, neighbours):
    """Contiguous queries, or one row of a projection's buffer, replaced by values of the same size."""
    import qwanto_b200 as qb
    torch = cuda
    g = torch.Generator("cuda").manual_seed(rows + rot)
    qkv = torch.randn((rows, 10 * 128), device="cuda", generator=g).to(_type(torch, kind))
    table = torch.randn((128, rot), device="cuda", generator=g)
    begin = torch.tensor([0, rows], dtype=torch.int32, device="cuda")
    got = []
    for in_place in (False, True):
        src = qkv.clone()
        q = src if fused else src[:, :768].contiguous()
        out = q.view(_type(torch, out_kind)) if in_place else torch.empty((rows, 768), device="cuda", dtype=_type(torch, out_kind))
        pool = _pool(qb, torch, rows)
        pool.append_rotary(0, 1, rows, DTYPES[kind], src[:, 768:], src[:, 1024:], query=q, query_heads=6, query_out=out,
                           query_out_dtype=DTYPES[out_kind], rotations=table, rotary_dim=rot, max_position=128,
                           neighbours=neighbours, row_begin=begin, query_stride=1280 if fused else 0, key_stride=1280,
                           value_stride=1280)
        assert pool.check() == 0
        got.append((out[:, :768].clone(), [pool.page(int(p)).copy() for p in pool.page_table().ravel() if p >= 0]))
        assert torch.equal(src[:, 768:].view(torch.uint8), qkv[:, 768:].view(torch.uint8))
        pool.close()
    assert torch.equal(got[0][0].view(torch.uint8), got[1][0].view(torch.uint8))
    assert len(got[0][1]) == len(got[1][1]) and all((a == b).all() for a, b in zip(got[0][1], got[1][1]))


def test_queries_over_rows_still_read_are_refused(cuda):
    """With a projection's stride, or another size of value, a row's output lies on
    other rows' query, key and value."""
    import qwanto_b200 as qb
    from qwanto_b200 import _lib
    torch = cuda
    rows, wide = 8, 10 * 128
    qkv = torch.zeros((rows + 1, wide), device="cuda", dtype=torch.bfloat16)
    far = torch.zeros((rows, 768), device="cuda")
    table = torch.zeros((64, 128), device="cuda")
    pool = _pool(qb, torch, rows)
    base = qkv.data_ptr()
    begin = torch.tensor([0, rows], dtype=torch.int32, device="cuda")

    def append(**over):
        r = _lib.init(_lib.AppendRotaryRequest())
        r.num_seqs, r.num_rows, r.dtype, r.query_heads, r.query_out_dtype = 1, rows, 3, 6, 1
        r.rotary_dim, r.max_position, r.rotations_dev, r.row_begin_dev = 128, 64, table.data_ptr(), begin.data_ptr()
        r.query_stride = r.key_stride = r.value_stride = wide
        r.query_dev, r.key_dev, r.value_dev, r.query_out_dev = base, base + 768 * 2, base + 1024 * 2, far.data_ptr()
        for key, x in over.items():
            setattr(r, key, x)
        return _lib.lib().qwn_kv_append_rotary(C.byref(pool.h), C.byref(r))

    try:
        assert append() == 0
        apart = {"query_dev": far.data_ptr(), "query_stride": 0}  # contiguous bf16 queries
        assert append(**apart, query_out_dtype=3) == 0
        for over in ({"query_out_dev": base, "query_out_dtype": 3},  # in place, rows of the projection apart
                     {"query_out_dev": base}, {**apart},  # values twice as large
                     {**apart, "query_out_dtype": 3, "query_out_dev": far.data_ptr() + 768 * 2},  # a row further
                     {**apart, "query_out_dev": base + 1024 * 2}, {"query_out_dev": base + wide * 2 * (rows - 1) + 768 * 2}):
            assert append(**over) == -1, over
            assert "overlaps" in _lib.last_error()
        # with no query rows nothing is written beside the pages
        assert append(query_heads=0, query_out_dev=base) == 0
        # a row of its own: the last one is outside the rows read
        assert append(num_rows=1, row_begin_dev=None, query_out_dev=base, query_out_dtype=3) == 0
        assert append(query_out_dev=base + wide * 2 * rows, num_rows=1, row_begin_dev=None, query_out_dtype=3) == 0
        assert pool.check() == 0
    finally:
        pool.close()
