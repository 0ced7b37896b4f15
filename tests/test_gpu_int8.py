"""qwn_rmsnorm_q8 and qwn_matmul_q8 on the GPU against 64-bit formulas."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24  # half a unit in fp32's last place, relative
DTYPES = {"f32": 1, "f16": 2, "bf16": 3}
HALF_ULP = {"f32": U, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}  # of a value of the type, relative
# fp32's smallest steps near zero: subnormal results are rounded absolutely
TINY = {"f32": 2.0 ** -149, "f16": 2.0 ** -24, "bf16": 2.0 ** -133}


def _type(torch, name):
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def _rows(torch, g, rows, width, stride, offset, dtype, scale=1.0):
    """[rows][width] values in a buffer of its own stride, `offset` values in; the gaps are NaN."""
    buf = torch.full((rows * stride + offset + 16,), float("nan"), device="cuda", dtype=dtype)
    v = buf[offset:offset + rows * stride].view(rows, stride)[:, :width]
    v.copy_((torch.randn((rows, width), device="cuda", generator=g) * scale).to(dtype))
    return v


# error of y in fp32: the sum of squares is at most 8 x 8 terms in a row per
# thread and 10 levels of a tree, each term's square and h itself rounded
# (76 U, half of it through the root), then the mean, the root, two products:
# below 48 U in all; the scale adds a division.
Y_REL = 48 * U


def _check_norm(torch, x, residual, weight, eps, norm, codes, scales, out_rows, out_kind, residual_out):
    h32 = x.float() + residual.float() if residual is not None else x.float()
    if residual_out is not None:
        assert torch.equal(residual_out, h32.to(x.dtype)), "the residual is h rounded once"
    h = x.double() + (residual.double() if residual is not None else 0)
    y = h / (h.square().mean(-1, keepdim=True) + eps).sqrt() if norm else h
    if weight is not None:
        y = y * weight.double()
    top = y.abs().amax(-1)
    s = torch.where(top > 0, top / 127, torch.ones_like(top))
    assert ((scales.double() - s).abs() <= (Y_REL + 2 * U) * s).all()
    # the code is the nearest whole number to y / scale, up to y's and the scale's errors
    off = (codes.double() - y / s[:, None]).abs()
    assert (off <= 0.5 + 127 * 2 * (Y_REL + 2 * U)).all(), float(off.max())
    assert int(codes.abs().max()) <= 127
    if out_rows is not None:
        want = (codes.float() * scales[:, None]).to(_type(torch, out_kind))
        assert torch.equal(out_rows, want), "rows_out is code x scale"


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,width,pad,offset", [(1, 1, 0, 0), (3, 7, 0, 0), (2, 64, 64, 0), (5, 100, 4, 0),
                                                   (4, 127, 0, 1), (33, 1536, 0, 0), (3, 2049, 7, 3), (2, 4096, 16, 0),
                                                   (2, 6144, 0, 8), (1, 12288, 0, 0), (2, 20011, 5, 1),
                                                   (2, 32768, 0, 0), (2, 32767, 0, 0), (300, 4099, 0, 0), (301, 9000, 0, 1),
                                                   (300, 1000, 24, 0), (2049, 257, 0, 0), (2051, 640, 0, 0),
                                                   (2048, 64, 0, 1), (3000, 1, 0, 0), (2500, 380, 4, 4)])
@pytest.mark.parametrize("residual,weighted,norm", [(True, True, True), (False, True, True), (True, False, False)])
def test_rmsnorm(cuda, kind, rows, width, pad, offset, residual, weighted, norm):
    import qwanto_b200 as qb
    torch = cuda
    dt = _type(torch, kind)
    g = torch.Generator("cuda").manual_seed(rows * 100003 + width)
    stride = width + pad
    x = _rows(torch, g, rows, width, stride, offset, dt)
    r = _rows(torch, g, rows, width, stride, offset, dt, 3.0) if residual else None
    w = _rows(torch, g, 1, width, width, offset, dt)[0] if weighted else None
    codes = torch.full((rows * stride + offset,), 77, dtype=torch.int8, device="cuda")
    cv = codes[offset:].view(rows, stride)
    scales = torch.full((rows,), float("nan"), device="cuda")
    out_kind = {"f32": "bf16", "f16": "f32", "bf16": "f16"}[kind]
    back = torch.full((rows * stride + offset,), float("nan"), device="cuda", dtype=_type(torch, out_kind))
    bv = back[offset:].view(rows, stride)
    ro = torch.full((rows, width), float("nan"), device="cuda", dtype=dt) if residual else None
    qb.rmsnorm_q8(x, rows, width, DTYPES[kind], cv, scales, weight=w, eps=1e-5, residual=r, residual_out=ro,
                  norm=norm, x_stride=stride, residual_stride=stride if residual else 0, codes_stride=stride,
                  rows_out=bv, rows_dtype=DTYPES[out_kind], rows_stride=stride)
    torch.cuda.synchronize()
    _check_norm(torch, x, r, w, 1e-5, norm, cv[:, :width], scales, bv[:, :width], out_kind, ro)
    if pad:  # the gaps between rows are left alone
        assert (cv[:, width:] == 77).all() and bv[:, width:].isnan().all()


def test_rmsnorm_in_place_on_a_stream(cuda):
    """residual_out may be the residual; a call on a stream of its own is ordered with that stream's work."""
    import qwanto_b200 as qb
    torch = cuda
    g = torch.Generator("cuda").manual_seed(5)
    x = torch.randn((700, 4096), device="cuda", generator=g).bfloat16()
    r = torch.randn((700, 4096), device="cuda", generator=g).bfloat16()
    before = r.clone()
    codes = torch.empty((700, 4096), dtype=torch.int8, device="cuda")
    scales = torch.empty(700, device="cuda")
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        x2 = x * 2  # the call reads what this stream writes
        qb.rmsnorm_q8(x2, 700, 4096, 3, codes, scales, residual=r, residual_out=r, stream=s)
        total = r.float() + 0
    s.synchronize()
    _check_norm(torch, x2, before, None, 1e-6, True, codes, scales, None, None, r)
    assert torch.equal(total, (x2.float() + before.float()).bfloat16().float())


def test_rmsnorm_rows_of_zeros_and_beyond_numbers(cuda):
    import qwanto_b200 as qb
    torch = cuda
    inf, nan = float("inf"), float("nan")
    x = torch.randn((6, 300), device="cuda", generator=torch.Generator("cuda").manual_seed(9))
    x[0] = 0.0
    x[1, 17] = nan
    x[2, 299] = -inf
    x[4] = 1e-30  # squares vanish beside eps
    for norm in (True, False):
        codes = torch.full((6, 300), 9, dtype=torch.int8, device="cuda")
        scales = torch.full((6,), nan, device="cuda")
        rows = torch.full((6, 300), nan, device="cuda")
        qb.rmsnorm_q8(x, 6, 300, 1, codes, scales, norm=norm, rows_out=rows, rows_dtype=1)
        torch.cuda.synchronize()
        assert scales[0] == 1.0 and not codes[0].any()
        if norm:  # the mean is not a number or not finite: nothing of the row is, or only zeros
            for i in (1, 2):
                assert scales[i] == 1.0 and not codes[i].any() and not rows[i].any()
        else:
            for i, j in ((1, 17), (2, 299)):
                fine = x[i].isfinite()
                top = float(x[i][fine].abs().max())
                assert abs(float(scales[i]) - top / 127) <= 2 * U * top and codes[i, j] == 0
                assert ((codes[i].double() - x[i].double() / (top / 127)).abs()[fine] <= 0.5 + 1e-4).all()
        for i in (3, 5):
            y = x[i].double()
            if norm:
                y = y / (y.square().mean() + 1e-6).sqrt()
            assert ((codes[i].double() - y / (y.abs().max() / 127)).abs() <= 0.5 + 127 * 2 * (Y_REL + 2 * U)).all()
        assert (codes[4] == 127).all()


@pytest.mark.parametrize("kind", sorted(DTYPES))
@pytest.mark.parametrize("width", [8, 257, 4096, 16384])
def test_rows_beyond_numbers_of_every_type_and_width(cuda, kind, width):
    import qwanto_b200 as qb
    torch = cuda
    dt, inf, nan = _type(torch, kind), float("inf"), float("nan")
    x = torch.randn((6, width), device="cuda", generator=torch.Generator("cuda").manual_seed(width)).to(dt)
    x[0] = 0.0
    x[1, 0], x[1, width - 1] = nan, inf
    x[2] = -inf
    x[3] = float(torch.finfo(dt).tiny)  # its scale's inverse overflows in fp32
    x[3, 1] = 0.0
    codes = torch.full((6, width), 9, dtype=torch.int8, device="cuda")
    scales = torch.full((6,), nan, device="cuda")
    rows = torch.full((6, width), nan, device="cuda")
    qb.rmsnorm_q8(x, 6, width, DTYPES[kind], codes, scales, norm=False, rows_out=rows, rows_dtype=1)
    torch.cuda.synchronize()
    assert rows.isfinite().all()
    for i in (0, 2):
        assert scales[i] == 1.0 and not codes[i].any() and not rows[i].any()
    assert codes[3, 1] == 0 and (codes[3].abs().sum() == 127 * (width - 1))
    for i in (1, 4, 5):
        fine = x[i].isfinite()
        top = float(x[i][fine].abs().max())
        assert abs(float(scales[i]) - top / 127) <= 2 * U * top and not codes[i][~fine].any()
        assert ((codes[i].double() - x[i].double() / (top / 127)).abs()[fine] <= 0.5 + 1e-4).all()
    # rows of zeros have no root without eps; a value that is none spoils its row's mean alone
    qb.rmsnorm_q8(x, 6, width, DTYPES[kind], codes, scales, eps=0.0)
    torch.cuda.synchronize()
    for i in (0, 1, 2):
        assert scales[i] == 1.0 and not codes[i].any()
    assert scales[4:].isfinite().all() and (codes[4:].abs().amax(1) == 127).all()


# ---- products -------------------------------------------------------------------

def _codes(torch, g, rows, k, low=-127):
    stride = -(-k // 16) * 16 + 16
    buf = torch.full((rows, stride), 99, dtype=torch.int8, device="cuda")  # the gaps must not count
    buf[:, :k] = torch.randint(low, 128, (rows, k), device="cuda", generator=g).to(torch.int8)
    return buf, stride


def _check_matmul(torch, x, w, sx, sw, bias, kind, out):
    acc = x.double() @ w.double().T  # whole numbers below 2^53: exact
    y = acc * torch.outer(sx.double(), sw.double())
    # the sum's conversion, two products, the bias' sum in fp32, then the output's rounding
    size = y.abs() + (bias.double().abs() if bias is not None else 0)
    if bias is not None:
        y = y + bias.double()
    tol = 4 * U * size + HALF_ULP[kind] * (y.abs() + 4 * U * size) + TINY[kind]
    off = (out.double() - y).abs()
    assert (off <= tol).all(), f"{int((off > tol).sum())} of {off.numel()} off, worst {float((off - tol).max())}"


SHAPES = [(1, 1, 1), (1, 1536, 2048), (2, 15, 7), (3, 16, 8), (1, 17, 129), (8, 4096, 128), (15, 127, 1000), (16, 128, 128),
          (17, 129, 127), (31, 300, 257), (32, 4096, 640), (33, 64, 384), (63, 1000, 100), (64, 2048, 256),
          (65, 511, 513), (100, 4099, 255), (127, 96, 1024), (128, 640, 128), (129, 256, 129), (200, 1536, 300),
          (255, 80, 65), (256, 1024, 512), (257, 513, 1023), (300, 4100, 77), (511, 200, 640), (513, 384, 2049),
          (1000, 130, 1000), (2049, 1111, 513), (4096, 256, 16)]


@pytest.mark.parametrize("m,k,n", SHAPES)
def test_matmul(cuda, m, k, n):
    import qwanto_b200 as qb
    torch = cuda
    g = torch.Generator("cuda").manual_seed(m * 7919 + k * 31 + n)
    x, stride = _codes(torch, g, m, k)
    w = torch.randint(-128, 128, (n, k + 3), device="cuda", generator=g).to(torch.int8)
    sx = torch.rand(m, device="cuda", generator=g) * 0.03
    sw = torch.rand(n, device="cuda", generator=g) * 0.01
    bias = torch.randn(n, device="cuda", generator=g)
    for kind, b, pad in (("f32", bias, 0), ("f16", None, 5), ("bf16", bias, 1)):
        with_gap = torch.full((m, n + pad), float("nan"), device="cuda", dtype=_type(torch, kind))
        mm = qb.MatmulQ8(w, n, k, sw, b, weight_stride=k + 3)
        try:
            mm(x, sx, m, with_gap, DTYPES[kind], codes_stride=stride, out_stride=n + pad)
            assert mm.check() == 0
        finally:
            mm.close()
        _check_matmul(torch, x[:, :k], w[:, :k], sx, sw, b, kind, with_gap[:, :n])
        assert with_gap[:, n:].isnan().all()


@pytest.mark.parametrize("m", [1, 40, 300])
def test_matmul_whole_numbers_are_exact(cuda, m):
    """Scales of one and sums below 2^24: the fp32 output is the integer sum."""
    import qwanto_b200 as qb
    torch = cuda
    g = torch.Generator("cuda").manual_seed(m)
    k, n = 1000, 333
    x, stride = _codes(torch, g, m, k, -128)
    w = torch.randint(-128, 128, (n, k), device="cuda", generator=g).to(torch.int8)
    one = torch.ones(max(m, n), device="cuda")
    out = torch.empty((m, n), device="cuda")
    mm = qb.MatmulQ8(w, n, k, one)
    mm(x, one, m, out, 1, codes_stride=stride)
    assert mm.check() == 0
    assert torch.equal(out.double(), x[:, :k].double() @ w.double().T)


@pytest.mark.parametrize("m", [1, 64, 130, 600])
def test_matmul_largest_sum(cuda, m):
    """The longest row of -128 times -128 stays within int32."""
    import qwanto_b200 as qb
    torch = cuda
    k, n = 131071, 130
    x = torch.full((m, k + 1), -128, dtype=torch.int8, device="cuda")
    w = torch.full((n, k), -128, dtype=torch.int8, device="cuda")
    w[1] = 127
    one = torch.ones(max(m, n), device="cuda")
    out = torch.empty((m, n), device="cuda")
    mm = qb.MatmulQ8(w, n, k, one)
    mm(x, one, m, out, 1, codes_stride=k + 1)
    assert mm.check() == 0
    want = torch.full((n,), 128.0 * 128 * k, dtype=torch.float64, device="cuda")
    want[1] = -128.0 * 127 * k
    assert torch.equal(out, want.float().expand(m, n))  # one rounding of the exact sum


def test_matmul_beyond_numbers_stay_in_their_row(cuda):
    import qwanto_b200 as qb
    torch = cuda
    g = torch.Generator("cuda").manual_seed(3)
    x, stride = _codes(torch, g, 20, 256)
    w = torch.randint(-127, 128, (200, 256), device="cuda", generator=g).to(torch.int8)
    sx, sw = torch.ones(20, device="cuda"), torch.ones(200, device="cuda")
    sx[7], sw[11] = float("nan"), float("inf")
    mm = qb.MatmulQ8(w, 200, 256, sw)
    out = torch.zeros((20, 200), device="cuda")
    mm(x, sx, 20, out, 1, codes_stride=stride)
    assert mm.check() == 0
    keep_r = torch.tensor([i for i in range(20) if i != 7], device="cuda")
    keep_c = torch.tensor([j for j in range(200) if j != 11], device="cuda")
    assert out[7].isnan().all()
    assert not out[keep_r][:, keep_c].isnan().any() and not out[keep_r][:, keep_c].isinf().any()


def test_matmul_two_streams_share_a_handle(cuda):
    import qwanto_b200 as qb
    torch = cuda
    g = torch.Generator("cuda").manual_seed(8)
    n, k = 640, 2048
    w = torch.randint(-127, 128, (n, k), device="cuda", generator=g).to(torch.int8)
    sw = torch.rand(n, device="cuda", generator=g) * 0.01
    mm = qb.MatmulQ8(w, n, k, sw)
    jobs = []
    for i, m in enumerate((1, 48, 500, 3)):
        x, stride = _codes(torch, g, m, k)
        jobs.append((x, stride, torch.rand(m, device="cuda", generator=g), torch.empty((m, n), device="cuda"), m))
    streams = [torch.cuda.Stream() for _ in jobs]
    torch.cuda.synchronize()
    for _ in range(5):
        for s, (x, stride, sx, out, m) in zip(streams, jobs):
            mm(x, sx, m, out, 1, codes_stride=stride, stream=s)
    assert mm.check() == 0
    for x, _, sx, out, m in jobs:
        _check_matmul(torch, x[:, :k], w, sx, sw, None, "f32", out)


@pytest.mark.parametrize("k", [1, 100, 1000, 4097])
def test_matmul_of_one_row_needs_no_aligned_stride(cuda, k):
    import qwanto_b200 as qb
    torch = cuda
    g = torch.Generator("cuda").manual_seed(k)
    x = torch.randint(-128, 128, (1, k), device="cuda", generator=g).to(torch.int8)
    w = torch.randint(-128, 128, (70, k), device="cuda", generator=g).to(torch.int8)
    sx, sw = torch.rand(1, device="cuda", generator=g), torch.rand(70, device="cuda", generator=g) * 0.01
    out = torch.full((1, 70), float("nan"), device="cuda")
    mm = qb.MatmulQ8(w, 70, k, sw)
    mm(x, sx, 1, out, 1)
    assert mm.check() == 0
    _check_matmul(torch, x, w, sx, sw, None, "f32", out)


def test_matmul_refusals(cuda):
    import qwanto_b200 as qb
    from qwanto_b200 import _lib
    torch = cuda
    w = torch.zeros((8, 40), dtype=torch.int8, device="cuda")
    mm = qb.MatmulQ8(w, 8, 40, torch.ones(8, device="cuda"))
    x = torch.zeros((4, 64), dtype=torch.int8, device="cuda")
    sx, out = torch.ones(4, device="cuda"), torch.zeros((4, 8), device="cuda")

    def call(**over):
        r = _lib.init(_lib.MatmulQ8Request())
        r.rows, r.out_dtype, r.codes_stride = 4, 1, 64
        r.codes_dev, r.scales_dev, r.out_dev = x.data_ptr(), sx.data_ptr(), out.data_ptr()
        for key, v in over.items():
            setattr(r, key, v)
        return _lib.lib().qwn_matmul_q8(C.byref(mm.h), C.byref(r))

    assert call() == 0 and call(rows=0, codes_dev=None) == 0
    for over in ({"out_dtype": 0}, {"codes_stride": 32}, {"codes_stride": 56}, {"codes_dev": x.data_ptr() + 8},
                 {"codes_dev": None}, {"scales_dev": None}, {"out_dev": None}, {"out_stride": 7},
                 {"out_dev": out.data_ptr() + 2}, {"scales_dev": sx.data_ptr() + 1}):
        assert call(**over) == -1, over
        assert "qwn_matmul_q8" in _lib.last_error()
    with pytest.raises(qb.QwnCudaError):
        qb.MatmulQ8(w, 8, 131072, sx)
    assert mm.check() == 0
    mm.close()


def test_products_of_both_kinds_one_behind_the_other(cuda):
    """Every launch starts while the one before it runs, each with tensor memory
    of its own: few tokens, a cluster per tile, pairs with narrow and wide tiles,
    on one stream and on three at once."""
    import qwanto_b200 as qb
    torch = cuda
    g = torch.Generator("cuda").manual_seed(21)
    products = []
    for n, k in ((2048, 128), (4096, 1536), (1000, 4096), (20000, 256)):
        w = torch.randint(-127, 128, (n, k), device="cuda", generator=g).to(torch.int8)
        sw = torch.rand(n, device="cuda", generator=g) * 0.01
        products.append((qb.MatmulQ8(w, n, k, sw), w, sw))
    jobs = []
    for m in (1, 600, 33, 2, 257, 128, 64, 1500, 16):
        for mm, w, sw in products:
            x, stride = _codes(torch, g, m, mm.in_features)
            jobs.append((mm, w, sw, x, stride, torch.rand(m, device="cuda", generator=g), m))
    torch.cuda.synchronize()
    for streams in ([None], [torch.cuda.Stream() for _ in range(3)]):
        outs = [torch.full((j[6], j[0].out_features), float("nan"), device="cuda") for j in jobs]
        torch.cuda.synchronize()
        for _ in range(3):
            for i, (mm, _, _, x, stride, sx, m) in enumerate(jobs):
                mm(x, sx, m, outs[i], 1, codes_stride=stride, stream=streams[i % len(streams)])
        torch.cuda.synchronize()
        for (mm, w, sw, x, _, sx, m), out in zip(jobs, outs):
            assert mm.check() == 0
            _check_matmul(torch, x[:, :mm.in_features], w, sx, sw, None, "f32", out)
    for mm, _, _ in products:
        mm.close()
