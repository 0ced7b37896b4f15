"""The int8 and rotary entry points without a GPU: structure layouts equal
their ctypes mirrors, and arguments are refused before any device work."""
import ctypes as C
import os
import subprocess
import tempfile

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
INVALID, MISMATCH = -1, -2


def _mirrors():
    from qwanto_b200 import _lib
    return {"QwnKvAppendRotaryRequest": _lib.AppendRotaryRequest, "QwnKvLoadTokensRequest": _lib.LoadTokensRequest,
            "QwnRmsNormQ8Request": _lib.RmsNormQ8Request, "QwnMatmulQ8Options": _lib.MatmulQ8Options,
            "QwnMatmulQ8Request": _lib.MatmulQ8Request, "QwnMatmulQ8Handle": _lib.Handle}


def test_struct_layouts():
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "qwn_kv_b200.h"', "int main(void){"]
    for name, cls in _mirrors().items():
        lines.append(f'printf("{name} %zu\\n", sizeof({name}));')
        lines += [f'printf("{name}.{f[0]} %zu\\n", offsetof({name}, {f[0]}));' for f in cls._fields_]
    lines.append("return 0;}")
    with tempfile.TemporaryDirectory() as d:
        src, exe = os.path.join(d, "p.c"), os.path.join(d, "p")
        open(src, "w").write("\n".join(lines))
        subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), src, "-o", exe], check=True)
        text = subprocess.run([exe], check=True, capture_output=True, text=True).stdout
    got = dict(line.rsplit(" ", 1) for line in text.strip().splitlines())
    for name, cls in _mirrors().items():
        assert int(got[name]) == C.sizeof(cls), name
        for f in cls._fields_:
            assert int(got[f"{name}.{f[0]}"]) == getattr(cls, f[0]).offset, f"{name}.{f[0]}"


def test_capability_bits():
    import qwanto_b200
    from qwanto_b200 import _lib
    bits = qwanto_b200.CudaContext.query().capability_bits
    assert bits & _lib.CAP_ROTARY_KV and bits & _lib.CAP_INT8_LINEAR


def _norm(**over):
    from qwanto_b200 import _lib
    r = _lib.init(_lib.RmsNormQ8Request())
    r.rows, r.width, r.dtype, r.eps = 2, 64, 1, 1e-6
    r.x_dev, r.codes_dev, r.scales_dev = 4096, 8192, 12288
    for k, v in over.items():
        setattr(r, k, v)
    return r


@pytest.mark.parametrize("over", [{"dtype": 0}, {"dtype": 4}, {"mode": 2}, {"width": 0}, {"width": 32769},
                                  {"eps": -1.0}, {"eps": float("nan")}, {"eps": float("inf")}, {"x_dev": None},
                                  {"codes_dev": None}, {"scales_dev": None}, {"x_stride": 63}, {"codes_stride": 1},
                                  {"x_dev": 4097}, {"scales_dev": 12290}, {"rows_out_dev": 4096, "rows_dtype": 0},
                                  {"rows_out_dev": 4097, "rows_dtype": 3}, {"residual_dev": 4098}])
def test_rmsnorm_refuses(over):
    from qwanto_b200 import _lib
    assert _lib.lib().qwn_rmsnorm_q8(C.byref(_norm(**over))) == INVALID
    assert "qwn_rmsnorm_q8" in _lib.last_error()


def test_rmsnorm_header_and_empty():
    from qwanto_b200 import _lib
    r = _norm(rows=0, x_dev=None, codes_dev=None, scales_dev=None)
    assert _lib.lib().qwn_rmsnorm_q8(C.byref(r)) == 0  # nothing to do
    r = _norm()
    r.header.struct_size -= 8
    assert _lib.lib().qwn_rmsnorm_q8(C.byref(r)) == MISMATCH
    r = _norm()
    r.header.abi_version = 7
    assert _lib.lib().qwn_rmsnorm_q8(C.byref(r)) == MISMATCH
    assert _lib.lib().qwn_rmsnorm_q8(None) == MISMATCH


@pytest.mark.parametrize("over", [{"out_features": 0}, {"in_features": 0}, {"in_features": 131072},
                                  {"out_features": 1 << 31}, {"weight_dev": None}, {"scales_dev": None},
                                  {"weight_stride": 63}])
def test_matmul_create_refuses(over):
    from qwanto_b200 import _lib
    o = _lib.init(_lib.MatmulQ8Options())
    o.out_features, o.in_features, o.weight_dev, o.scales_dev = 16, 64, 4096, 8192
    for k, v in over.items():
        setattr(o, k, v)
    h = _lib.init(_lib.Handle())
    assert _lib.lib().qwn_matmul_q8_create(C.byref(o), C.byref(h)) == INVALID
    assert not h.opaque


def test_calls_without_a_handle():
    from qwanto_b200 import _lib
    L = _lib.lib()
    h = _lib.init(_lib.Handle())
    bits = C.c_uint32(0)
    assert L.qwn_matmul_q8(C.byref(h), C.byref(_lib.init(_lib.MatmulQ8Request()))) == INVALID
    assert L.qwn_matmul_q8_destroy(C.byref(h)) == INVALID
    assert L.qwn_matmul_q8_check(C.byref(h), C.byref(bits)) == INVALID
    assert L.qwn_kv_append_rotary(C.byref(h), C.byref(_lib.init(_lib.AppendRotaryRequest()))) == INVALID
    assert L.qwn_kv_load_tokens(C.byref(h), C.byref(_lib.init(_lib.LoadTokensRequest()))) == INVALID


@pytest.mark.parametrize("over", [{"residual_out_dev": 4096, "residual_out_stride": 128},
                                  {"residual_dev": 65536, "residual_out_dev": 65536, "residual_stride": 96},
                                  {"residual_dev": 65536, "residual_out_dev": 65536 + 256},
                                  {"residual_out_dev": 4096 + 4}, {"residual_out_dev": 4096 - 252},
                                  {"x_stride": 100, "residual_out_dev": 4096 + 256, "residual_out_stride": 100},
                                  {"weight_dev": 65536, "residual_out_dev": 65536 + 128}])
def test_rmsnorm_refuses_a_residual_over_rows_still_read(over):
    """In place is the same rows; any other overlap is a row that another row's output may have replaced."""
    from qwanto_b200 import _lib
    assert _lib.lib().qwn_rmsnorm_q8(C.byref(_norm(**over))) == INVALID
    assert "overlaps" in _lib.last_error()


def test_rows_meet_where_they_share_a_byte():
    """The library's test of overlap against sets of bytes."""
    import random
    rng = random.Random(5)
    cases = []
    for i in range(4000):
        spans = []
        same = rng.randrange(1, 30)
        for _ in range(2):
            size = rng.randrange(1, 12)
            stride = max(size, same) if i % 2 else size + rng.randrange(0, 20)
            spans.append((rng.randrange(100, 220), stride, size, rng.randrange(1, 7)))
        cases.append(spans)
    lines = "\n".join(" ".join(str(v) for s in c for v in s) for c in cases)
    code = """#include <cstdio>
#include "row_span.h"
int main() {
    qkv::RowSpan s[2];
    unsigned long v[8];
    while (scanf("%lu %lu %lu %lu %lu %lu %lu %lu", v, v + 1, v + 2, v + 3, v + 4, v + 5, v + 6, v + 7) == 8) {
        for (int i = 0; i < 2; i++) s[i] = {v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]};
        putchar('0' + qkv::rows_meet(s[0], s[1]));
    }
}
"""
    with tempfile.TemporaryDirectory() as d:
        src, exe = os.path.join(d, "p.cpp"), os.path.join(d, "p")
        open(src, "w").write(code)
        subprocess.run(["g++", "-std=c++17", "-I", os.path.join(ROOT, "qwanto_b200", "csrc"), src, "-o", exe], check=True)
        got = subprocess.run([exe], check=True, input=lines, capture_output=True, text=True).stdout
    held = lambda s: {s[0] + r * s[1] + b for r in range(s[3]) for b in range(s[2])}  # noqa: E731
    want = "".join(str(int(bool(held(a) & held(b)))) for a, b in cases)
    assert got == want and "0" in got and "1" in got
