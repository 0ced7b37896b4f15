"""The prompt attention's entry points without a GPU: structure layouts equal
their ctypes mirrors, and arguments are refused before any device work."""
import ctypes as C
import os
import re
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


def _kernel_source():
    text = open(os.path.join(ROOT, "qwanto_b200", "csrc", "prompt_tile.cuh")).read()
    return re.sub(r"//[^\n]*", "", text)


def _body(text, start):
    """The text from the first brace behind `start` to the matching one."""
    at = text.index("{", text.index(start))
    depth = 0
    for i in range(at, len(text)):
        depth += {"{": 1, "}": -1}.get(text[i], 0)
        if depth == 0:
            return text[at:i + 1]
    raise AssertionError(start)


def test_the_next_launch_starts_after_tensor_memory_is_held():
    """What a run could only show by hanging is read: see the products' tests."""
    body = _body(_kernel_source(), "prompt_tile_kernel(")
    assert body.count("launch_dependents()") == 1
    assert body.index("tmem_alloc<") < body.index("__syncthreads()") < body.index("launch_dependents()")
    # no role polls a barrier before the previous launch has ended
    waits = body.index("wait_previous()")
    for role in ("roles.soften()", "roles.help()", "roles.multiply()", "roles.load(", "roles.plan()"):
        assert body.count(role) == 1 and waits < body.index(role)


def test_every_wait_is_bounded():
    text = _kernel_source()
    assert "kWaitLimit" in _body(text, "at_wait(volatile int &give_up")
    # no named barrier, which one role could leave and another wait at; the block's own only where all meet
    assert "bar.sync" not in text and text.count("__syncthreads()") == 2
    # the only other poll, of the copies' lanes, gives up alike
    polls = [m.start() for m in re.finditer(r"mbar_try_wait\(", text)]
    assert len(polls) == 2
    assert "it >= kWaitLimit" in text[polls[1]:polls[1] + 1500]


def test_registers_are_shared_out_from_what_a_block_starts_with():
    """A warpgroup that asks for more than the others gave back waits for good."""
    text = _kernel_source()
    assert "2 * kSoftmaxRegs + kHelpers / 4 * kHelperRegs + kOtherRegs <= kThreads / 128 * kLaunchRegs" in text
    assert "at.numRegs < AtShape<SRC, PARTS, TILES>::kLaunchRegs" in _body(text, "cudaError_t prepare_tile_kernel(")


def test_cached_tiles_are_given_back_behind_a_proxy_fence():
    text = _kernel_source()
    body = _body(text, "auto give_back")
    assert body.index("fence_proxy_async_shared()") < body.index("warp_arrive(&sh.rawempty")
    assert text.count("sh.rawempty[r], lane") == 1
