"""The product kernels' hand-overs, as their source states them: what must come
before what for a launch never to wait for a later one.  A run could only show the
opposite by hanging, so these are read, not run."""
import os
import re

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
KERNELS = ["matmul_q8_split_kernel", "matmul_q8_pair_kernel"]


def _source(name):
    text = open(os.path.join(ROOT, "qwanto_b200", "csrc", name)).read()
    return re.sub(r"//[^\n]*", "", text)


def _body(text, name):
    """The function's text from its first brace to the matching one."""
    at = text.index("{", re.search(rf"\b{name}\s*\(", text).end())
    depth = 0
    for i in range(at, len(text)):
        depth += {"{": 1, "}": -1}.get(text[i], 0)
        if depth == 0:
            return text[at:i + 1]
    raise AssertionError(name)


@pytest.mark.parametrize("kernel", KERNELS)
def test_the_next_launch_starts_after_tensor_memory_is_held(kernel):
    """A CTA of the next launch that held columns while this one's allocation waits
    for them would wait for this launch's end: both for good."""
    body = _body(_source("matmul_q8.cu"), kernel)
    starts = [m.start() for m in re.finditer(r"\blaunch_dependents\(\)", body)]
    assert len(starts) == 1
    assert body.index("tmem_alloc<") < body.index("__syncthreads()") < starts[0]


def test_the_permit_to_allocate_is_given_up_at_once():
    text = _source("tcgen05.cuh")
    alloc, free = _body(text, "tmem_alloc"), _body(text, "tmem_free")
    for group in ("cta_group::1", "cta_group::2"):
        assert alloc.index(f"tcgen05.alloc.{group}") < alloc.index(f"tcgen05.relinquish_alloc_permit.{group}")
    assert "relinquish" not in free


def _branch(body, start):
    """The block behind a condition."""
    at = body.index("{", body.index(start))
    depth = 0
    for i in range(at, len(body)):
        depth += {"{": 1, "}": -1}.get(body[i], 0)
        if depth == 0:
            return body[at:i + 1]
    raise AssertionError(start)


@pytest.mark.parametrize("kernel", KERNELS)
def test_no_bounded_wait_counts_the_previous_launch(kernel):
    """Every role that polls a barrier which depends on the previous launch waits for
    that launch first: its running time must not use up the limit."""
    body = _body(_source("matmul_q8.cu"), kernel)
    for role in ("if (warp == 0)", "if (warp == 1", "if (warp >= 2)"):
        block = _branch(body[body.index("launch_dependents()"):], role)
        assert "mbar_wait" in block, role
        assert block.index("wait_previous()") < block.index("mbar_wait"), role


@pytest.mark.parametrize("kernel", KERNELS)
def test_copies_land_whichever_role_gives_up(kernel):
    """The loading warp waits for its last copies whether or not it was the one that gave up."""
    block = _branch(_body(_source("matmul_q8.cu"), kernel), "if (warp == 0)")
    drain = block[block.rindex("wait_previous()"):]
    waits = [m.start() for m in re.finditer(r"mbar_wait_\w+\(&full\[", drain)]
    assert waits
    condition = re.findall(r"if \((?:[^()]|\([^()]*\))*\bone\b(?:[^()]|\([^()]*\))*\)", drain[:waits[0]])[-1]
    assert "ok" not in condition, condition


@pytest.mark.parametrize("kernel,last", [("matmul_q8_split_kernel", "mbar_wait_bounded(&done"),
                                         ("matmul_q8_pair_kernel", "mbar_wait_cluster(&acc_full[")])
def test_products_end_before_their_tensor_memory_goes(kernel, last):
    """The warp that issues the products waits for the last of them, also when the warps that read them gave up."""
    block = _branch(_body(_source("matmul_q8.cu"), kernel), "if (warp == 1 &&" if "pair" in kernel else "else if (warp == 1)")
    assert last in block[block.rindex("mma_commit"):]
