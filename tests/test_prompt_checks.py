"""The prompt attention's entry points without a GPU: structure layouts equal
their ctypes mirrors, and arguments are refused before any device work."""
import ctypes as C
import os
import subprocess
import tempfile

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
OK, INVALID = 0, -1


def test_struct_layouts():
    from qwanto_b200 import _lib
    mirrors = {"QwnKvChunkAttentionRequest": _lib.ChunkAttentionRequest,
               "QwnPromptAttentionRequest": _lib.PromptAttentionRequest}
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "qwn_kv_b200.h"', "int main(void){"]
    for name, cls in mirrors.items():
        lines.append(f'printf("{name} %zu\\n", sizeof({name}));')
        lines += [f'printf("{name}.{f[0]} %zu\\n", offsetof({name}, {f[0]}));' for f in cls._fields_]
    lines.append("return 0;}")
    with tempfile.TemporaryDirectory() as d:
        src, exe = os.path.join(d, "p.c"), os.path.join(d, "p")
        open(src, "w").write("\n".join(lines))
        subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), src, "-o", exe], check=True)
        text = subprocess.run([exe], check=True, capture_output=True, text=True).stdout
    got = dict(line.rsplit(" ", 1) for line in text.strip().splitlines())
    for name, cls in mirrors.items():
        assert int(got[name]) == C.sizeof(cls), name
        for f in cls._fields_:
            assert int(got[f"{name}.{f[0]}"]) == getattr(cls, f[0]).offset, f"{name}.{f[0]}"


def test_capability_bit():
    import qwanto_b200
    from qwanto_b200 import _lib
    assert qwanto_b200.CudaContext.query().capability_bits & _lib.CAP_PROMPT_ATTENTION


def _request(**over):
    from qwanto_b200 import _lib
    r = _lib.init(_lib.PromptAttentionRequest())
    r.num_seqs, r.num_rows, r.dtype, r.query_heads, r.kv_heads, r.causal = 2, 10, 3, 8, 2, 1
    r.row_begin_dev, r.query_dev, r.key_dev, r.value_dev, r.output_dev = 64, 1 << 20, 2 << 20, 3 << 20, 4 << 20
    for k, v in over.items():
        setattr(r, k, v)
    return r


BAD = [{"dtype": 0}, {"dtype": 4}, {"num_rows": 1 << 31}, {"query_heads": 7}, {"query_heads": 0}, {"kv_heads": 0},
       {"query_heads": 65538}, {"num_seqs": 0}, {"row_begin_dev": None}, {"num_seqs": 1 << 31}, {"scale": -0.5},
       {"scale": float("nan")}, {"scale": float("inf")}, {"window": 1 << 31}, {"causal": 0, "window": 5},
       {"query_dev": None}, {"key_dev": None}, {"value_dev": None}, {"output_dev": None}, {"query_stride": 1023},
       {"key_stride": 255}, {"value_stride": 255}, {"output_stride": 1020}, {"query_stride": 1028},
       {"key_stride": 260}, {"value_stride": 260}, {"output_stride": 1028}, {"query_dev": (1 << 20) + 8},
       {"key_dev": (2 << 20) + 8}, {"value_dev": (3 << 20) + 2}, {"output_dev": (4 << 20) + 8},
       {"dtype": 1, "query_stride": 1026}, {"output_dev": 1 << 20}, {"output_dev": (2 << 20) + 2 * 256 * 9},
       {"output_dev": (3 << 20) - 2 * 1024 * 10 + 16}]


@pytest.mark.parametrize("over", BAD)
def test_refused(over):
    import qwanto_b200
    from qwanto_b200 import _lib
    assert qwanto_b200.lib().qwn_prompt_attention(C.byref(_request(**over))) == INVALID
    assert _lib.last_error()


def test_header_and_null():
    import qwanto_b200
    r = _request()
    r.header.struct_size -= 8
    assert qwanto_b200.lib().qwn_prompt_attention(C.byref(r)) == INVALID
    assert qwanto_b200.lib().qwn_prompt_attention(None) == INVALID


def test_no_rows_is_no_work():
    import qwanto_b200
    assert qwanto_b200.lib().qwn_prompt_attention(C.byref(_request(num_rows=0, num_seqs=0))) == OK


def test_chunk_needs_a_pool():
    import qwanto_b200
    from qwanto_b200 import _lib
    lib, h, n = qwanto_b200.lib(), _lib.init(_lib.Handle()), C.c_uint64(0)
    r = _lib.init(_lib.ChunkAttentionRequest())
    for handle in (C.byref(h), None):
        assert lib.qwn_kv_chunk_attention(handle, C.byref(r)) == INVALID
        assert lib.qwn_kv_chunk_workspace(handle, 1, 1, 1, C.byref(n)) == INVALID
