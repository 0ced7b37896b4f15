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
