"""The attention block of examples/attention_block.py -- norm, int8 products,
rotated append, attention, output product -- against its formula in 64 bits,
over a ragged prompt, a second prompt on top of it, and decode steps."""
from __future__ import annotations

import importlib.util
import math
import os

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _example():
    spec = importlib.util.spec_from_file_location("attention_block",
                                                  os.path.join(ROOT, "examples", "attention_block.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


class Plain:
    """The block in 64 bits: int8 weights as they are, everything else unrounded."""

    def __init__(self, torch, b):
        self.torch, self.b = torch, b
        self.cache = {}

    def run(self, x, residual, counts):
        torch, b = self.torch, self.b
        h = x.double() + residual.double()
        y = h / (h.square().mean(-1, keepdim=True) + 1e-6).sqrt() * b.norm.double()
        w, s = b.wqkv
        z = (y @ (w.double() * s.double()[:, None]).T).view(len(y), -1, 128)
        q, k, v = z[:, :b.hq], z[:, b.hq:b.hq + b.hk], z[:, b.hq + b.hk:]
        out, at = torch.empty_like(q), 0
        for i, n in enumerate(counts):
            old = self.cache.get(i)
            p = 0 if old is None else len(old[0])
            cs = b.table[p:p + n, None, :].double()
            turn = lambda t: torch.cat((t[..., :64] * cs[..., :64] - t[..., 64:] * cs[..., 64:],  # noqa: E731
                                        t[..., 64:] * cs[..., :64] + t[..., :64] * cs[..., 64:]), -1)
            kk, vv = turn(k[at:at + n]), v[at:at + n]
            if old is not None:
                kk, vv = torch.cat((old[0], kk)), torch.cat((old[1], vv))
            self.cache[i] = kk, vv
            g = b.hq // b.hk
            sc = torch.einsum("qhd,khd->hqk", turn(q[at:at + n]), kk.repeat_interleave(g, 1)) / math.sqrt(128)
            future = torch.arange(p + n, device="cuda") > torch.arange(p, p + n, device="cuda")[:, None]
            out[at:at + n] = torch.einsum("hqk,khd->qhd", sc.masked_fill(future, -torch.inf).softmax(-1),
                                          vv.repeat_interleave(g, 1))
            at += n
        w, s = b.wout
        return h, out.flatten(1) @ (w.double() * s.double()[:, None]).T


# What the block rounds, as parts of the rms of what it rounds: the activations'
# codes before each product (a step of max / 127, max about 4 rms: 0.009 rms),
# the projection and the output to bf16 (0.002 each), K and V to the cache: int8
# per head 0.009, per 64 0.007, fp16 nothing; 4 bits a step of a group's range
# (4.2 rms) / 15: 0.08, 3.5 bits: 0.08 and, in the odd dims, 0.2.  K's error moves
# the softmax by about itself at scores near 1.  The parts add up in squares over
# both products and both of K and V.
BOUND = {1: 0.03, 2: 0.03, 3: 0.35, 4: 0.2, 5: 0.025}


@pytest.mark.parametrize("codec", [1, 2, 3, 4, 5])
def test_block_against_its_formula(cuda, codec):
    torch = cuda
    m = _example()
    b = m.AttentionBlock(640, 12, 2, 4, 300, codec, max_rows=512, seed=codec)
    try:
        plain = Plain(torch, b)
        g = torch.Generator("cuda").manual_seed(7)
        rows = lambda n: torch.randn((n, 640), device="cuda", generator=g).bfloat16()  # noqa: E731
        for counts in ([70, 1, 16, 33], [5, 47, 1, 16]):
            x, r = rows(sum(counts)), rows(sum(counts))
            want_r, want = plain.run(x, r, counts)
            got = b.prompt(x, r, counts)
            assert b.check() == 0
            assert torch.equal(r, want_r.float().bfloat16())
            off = float((got.double() - want).norm() / want.norm())
            assert off <= BOUND[codec], off
        for _ in range(3):
            x, r = rows(4), rows(4)
            want_r, want = plain.run(x, r, [1] * 4)
            got = b.step(x, r)
            assert b.check() == 0
            assert torch.equal(r, want_r.float().bfloat16())
            off = float((got.double() - want).norm() / want.norm())
            assert off <= BOUND[codec], off
    finally:
        b.close()


def test_steps_on_a_stream_equal_steps_with_waits(cuda):
    """The kernels start before their predecessors end (programmatic launches):
    a run with a wait after every call gives the same bits."""
    torch = cuda
    m = _example()
    outs = []
    for wait in (False, True):
        b = m.AttentionBlock(1024, 8, 2, 3, 200, 2, max_rows=128, seed=1)
        g = torch.Generator("cuda").manual_seed(3)
        x = torch.randn((3, 1024), device="cuda", generator=g).bfloat16()
        r = torch.randn((3, 1024), device="cuda", generator=g).bfloat16()
        if wait:
            for name in ("project", "store", "output"):
                plain = getattr(b, name)
                setattr(b, name, lambda *a, f=plain: (f(*a), torch.cuda.synchronize())[0])
        torch.cuda.synchronize()
        for _ in range(40):
            x = b.step(x, r)
        assert b.check() == 0
        outs.append((x, r))
        b.close()
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])


def test_attention_after_these_calls_waits_for_them(cuda):
    """qwn_kv_decode starts early behind another layer's attention, never behind
    a call that lets the next kernel start: layers back to back, each layer's
    query and new rows written by a product just before it."""
    import qwanto_b200 as qb
    torch = cuda
    layers, hq, hk, seqs = 6, 8, 2, 5
    pool = qb.KvPool(2, layers, hk, 16, 200, seqs, 40, max_query_heads=hq)
    try:
        g = torch.Generator("cuda").manual_seed(2)
        pool.prefill_synthetic(list(range(seqs)), [100, 17, 300, 64, 200], 5)
        wide = (hq + 2 * hk) * 128
        w = torch.randint(-127, 128, (wide, 4096), device="cuda", generator=g).to(torch.int8)
        mm = qb.MatmulQ8(w, wide, 4096, torch.full((wide,), 1e-5, device="cuda"))
        codes = torch.randint(-127, 128, (layers, seqs, 4096), device="cuda", generator=g).to(torch.int8)
        scales = torch.rand((layers, seqs), device="cuda", generator=g)
        got = []
        for wait in (True, False):
            for rep in range(1 if wait else 5):
                qkv = torch.zeros((seqs, wide), device="cuda")  # one buffer for all layers
                outs = torch.zeros((layers, seqs, hq, 128), device="cuda")
                torch.cuda.synchronize()
                for layer in range(layers):
                    mm(codes[layer], scales[layer], seqs, qkv, 1)
                    if wait:
                        torch.cuda.synchronize()
                    q = qkv[:, :hq * 128].contiguous()
                    pool.decode(layer, seqs, hq, q, outs[layer])
                    if wait:
                        torch.cuda.synchronize()
                torch.cuda.synchronize()
                got.append(outs)
        for o in got[1:]:
            assert torch.equal(o, got[0])
        # the product writes the query rows that the attention reads, nothing between them
        wq = qb.MatmulQ8(w[:hq * 128].contiguous(), hq * 128, 4096, torch.full((hq * 128,), 1e-5, device="cuda"))
        got = []
        for wait in (True, False):
            for rep in range(1 if wait else 5):
                q = torch.zeros((seqs, hq * 128), device="cuda")
                outs = torch.zeros((layers, seqs, hq, 128), device="cuda")
                torch.cuda.synchronize()
                for layer in range(layers):
                    wq(codes[layer], scales[layer], seqs, q, 1)
                    if wait:
                        torch.cuda.synchronize()
                    pool.decode(layer, seqs, hq, q, outs[layer])
                    if wait:
                        torch.cuda.synchronize()
                torch.cuda.synchronize()
                got.append(outs)
        for o in got[1:]:
            assert torch.equal(o, got[0])
        assert pool.check() == 0 and mm.check() == 0 and wq.check() == 0
    finally:
        pool.close()


def test_one_product_writes_the_queries_of_several_layers(cuda):
    """The second of two attention launches starts behind the first one's start,
    not behind its end: the first lets it start only once what came before both
    has ended."""
    import qwanto_b200 as qb
    torch = cuda
    layers, hq, hk, seqs, k = 6, 8, 2, 2, 131056
    pool = qb.KvPool(2, layers, hk, 16, 64, seqs, 16, max_query_heads=hq)
    try:
        g = torch.Generator("cuda").manual_seed(2)
        pool.prefill_synthetic(list(range(seqs)), [100, 17], 5)
        ids = torch.tensor([1, 0], dtype=torch.int32, device="cuda")
        w = torch.randint(-127, 128, (hq * 128, k), device="cuda", generator=g).to(torch.int8)
        mm = qb.MatmulQ8(w, hq * 128, k, torch.full((hq * 128,), 1e-7, device="cuda"))
        codes = torch.randint(-127, 128, (layers * seqs, k), device="cuda", generator=g).to(torch.int8)
        scales = torch.rand(layers * seqs, device="cuda", generator=g)
        got = []
        for wait in (True, False):
            for seq_ids in (None, ids):
                q = torch.zeros((layers, seqs, hq * 128), device="cuda")
                outs = torch.zeros((layers, seqs, hq, 128), device="cuda")
                torch.cuda.synchronize()
                mm(codes, scales, layers * seqs, q, 1)
                for layer in range(layers):
                    if wait:
                        torch.cuda.synchronize()
                    pool.decode(layer, seqs, hq, q[layer], outs[layer], seq_ids=seq_ids)
                torch.cuda.synchronize()
                got.append(outs)
        assert torch.equal(got[0], got[2]) and torch.equal(got[1], got[3])
        assert pool.check() == 0 and mm.check() == 0
    finally:
        pool.close()
