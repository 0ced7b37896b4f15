"""The int8 norm's codes against the rule itself, in fp32 on the host: without
the norm every step of it is one rounded operation, so codes, scales and rows
agree bit for bit."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

DTYPES = {"f32": 1, "f16": 2, "bf16": 3}


def _type(torch, name):
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def _rule(y):
    """Codes and scales of fp32 rows: scale = max|y| / 127 (1 if that is 0), code = y / scale to the nearest, ties to even."""
    top = np.abs(y).max(1)
    scale = top / np.float32(127)
    scale[scale == 0] = 1
    return np.clip(np.rint(y / scale[:, None]), -127, 127).astype(np.int8), scale


def _tied(torch, g, rows, width, dt):
    """Rows with values at half codes of their own maximum, where a rounding of the quotient decides."""
    top = (1 + torch.rand((rows, 1), device="cuda", generator=g)) * 2.0 ** torch.randint(-3, 8, (rows, 1), device="cuda", generator=g)
    half = torch.randint(-127, 127, (rows, width), device="cuda", generator=g) + 0.5
    x = half / 127 * top.to(dt).float()
    x[:, 0] = top[:, 0].to(dt).float()
    return x.to(dt)


# widths and counts of rows that reach every kernel: one chunk of 16 bytes per thread and two, four, eight,
# sixteen; a warp per row; rows off the 16-byte grid
@pytest.mark.parametrize("kind", sorted(DTYPES))
@pytest.mark.parametrize("rows,width,offset", [(2, 176, 0), (40, 4096, 0), (400, 2048, 0), (400, 6144, 0), (300, 14336, 0),
                                               (5, 16384, 0), (3, 32768, 0), (2048, 256, 0), (2050, 512, 0), (2049, 768, 0),
                                               (3, 1001, 1), (500, 2047, 0), (300, 9001, 3), (2048, 255, 1), (3, 32767, 0)])
@pytest.mark.parametrize("residual,weighted", [(False, False), (True, False), (False, True)])
def test_codes_follow_the_rule_at_ties(cuda, kind, rows, width, offset, residual, weighted):
    import qwanto_b200 as qb
    torch = cuda
    dt = _type(torch, kind)
    g = torch.Generator("cuda").manual_seed(rows * 7 + width)
    x = torch.zeros(rows * width + offset, device="cuda", dtype=dt)[offset:].view(rows, width)
    x.copy_(_tied(torch, g, rows, width, dt))
    r = torch.randint(-3, 4, (rows, width), device="cuda", generator=g).to(dt) if residual else None
    w = (2.0 ** torch.randint(-2, 3, (width,), device="cuda", generator=g)).to(dt) if weighted else None
    codes = torch.full((rows, width), 77, dtype=torch.int8, device="cuda")
    scales = torch.full((rows,), float("nan"), device="cuda")
    back = torch.full((rows, width), float("nan"), device="cuda")
    qb.rmsnorm_q8(x, rows, width, DTYPES[kind], codes, scales, weight=w, residual=r, norm=False, rows_out=back, rows_dtype=1)
    y = x.float()
    if residual:
        y = y + r.float()
    if weighted:
        y = y * w.float()
    want, scale = _rule(y.cpu().numpy())
    assert np.array_equal(scales.cpu().numpy(), scale)
    got = codes.cpu().numpy()
    assert np.array_equal(got, want), f"{int((got != want).sum())} of {want.size} codes"
    assert np.array_equal(back.cpu().numpy(), want.astype(np.float32) * scale[:, None])


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("width", [64, 257, 4096])
def test_codes_follow_the_rule_near_the_smallest_numbers(cuda, kind, width):
    """Maxima down to the smallest number: scales with few bits, or none."""
    import qwanto_b200 as qb
    torch = cuda
    dt = _type(torch, kind)
    tops = [2.0 ** -e for e in (90, 99, 100, 101, 118, 119, 121, 126, 130, 133)] + ([2.0 ** -140, 3 * 2.0 ** -143, 2.0 ** -149]
                                                                                    if kind == "f32" else [])
    g = torch.Generator().manual_seed(width)
    x = (torch.rand((len(tops), width), generator=g, dtype=torch.float64) * 2 - 1) * torch.tensor(tops, dtype=torch.float64)[:, None]
    x[:, 1] = torch.tensor(tops, dtype=torch.float64)
    x = x.to(dt)
    want, scale = _rule(x.float().numpy())
    codes = torch.full((len(tops), width), 77, dtype=torch.int8, device="cuda")
    scales = torch.full((len(tops),), float("nan"), device="cuda")
    qb.rmsnorm_q8(x.cuda(), len(tops), width, DTYPES[kind], codes, scales, norm=False)
    assert np.array_equal(scales.cpu().numpy(), scale)
    assert np.array_equal(codes.cpu().numpy(), want)


def _hard_rows():
    """(maximum, value) whose quotient value / (maximum / 127) lies within four 2^-24ths of a unit in the last place of
    the middle between a half code and its neighbour in fp32, so that only a correctly rounded quotient is on the right
    side: with 24-bit whole numbers a, b and the middle N / 2, a 2^j = b N + D for a small D, which b solves modulo 2^j."""
    rows = []
    for k in range(127):
        e = int(np.floor(np.log2(k + 0.5)))
        for side in (1, -1):
            n = (2 * k + 1) * 2 ** (23 - e) + side
            for j in (23, 24, 25):
                for d in (-4, -3, -2, -1, 1, 2, 3, 4):
                    b0 = -d * pow(n, -1, 2 ** j) % 2 ** j
                    for b in (b0, b0 + 2 ** 23):
                        if not 2 ** 23 <= b < 2 ** 24 or (b * n + d) % 2 ** j:
                            continue
                        a = (b * n + d) >> j
                        if not 2 ** 23 <= a <= 2 ** 24:
                            continue
                        s, y = np.float32(b * 2.0 ** -24), np.float32(a * 2.0 ** (j + e - 48))
                        top = np.float32(127 * float(s))
                        for t in (top, np.nextafter(top, np.float32(0)), np.nextafter(top, np.float32(999))):
                            if t / np.float32(127) == s and y <= t:
                                rows.append((t, y))
                                break
    return np.array(rows, dtype=np.float32)


@pytest.mark.parametrize("power", [0, 100, -80])
def test_codes_follow_the_rule_in_the_hardest_quotients(cuda, power):
    import qwanto_b200 as qb
    torch = cuda
    pairs = _hard_rows()
    assert len(pairs) > 100
    n, width = len(pairs), 64
    x = np.zeros((n, width), dtype=np.float32)
    x[:, 5], x[:, 6], x[:, 7] = pairs[:, 0], pairs[:, 1], -pairs[:, 1]
    x = np.ldexp(x, power).astype(np.float32)
    want, scale = _rule(x)
    codes = torch.full((n, width), 77, dtype=torch.int8, device="cuda")
    scales = torch.full((n,), float("nan"), device="cuda")
    qb.rmsnorm_q8(torch.from_numpy(x).cuda(), n, width, 1, codes, scales, norm=False)
    assert np.array_equal(scales.cpu().numpy(), scale)
    assert np.array_equal(codes.cpu().numpy(), want)
