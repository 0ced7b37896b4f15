"""A decoder layer's attention half around the paged cache, on device buffers:

    norm -> int8 -> query/key/value product -> rotation and append -> attention
         -> int8 -> output product -> residual of the next norm

Prompts of several sequences go through it in one ragged batch; their attention
is a plain torch softmax over the cache's own rows (``KvPool.load_tokens``), so
that a prompt may follow on tokens that are cached already.  Then every
sequence decodes one token at a time through ``KvPool.decode``.

    python examples/attention_block.py [--codec 1..5] [--steps N]
"""
from __future__ import annotations

import argparse
import math
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import qwanto_b200 as qb  # noqa: E402

HEAD = 128
EPS = 1e-6


def quantise_rows(w):
    """fp32 [n][k] -> int8 codes and a scale per row."""
    scale = w.abs().amax(1) / 127
    return (w / scale[:, None]).round().clamp(-127, 127).to(torch.int8), scale


def rotations(positions, dims=HEAD, base=1e6):
    """The rotation table: cosines of each position's dims / 2 angles, then their sines."""
    freq = 1.0 / (base ** (torch.arange(0, dims, 2, dtype=torch.float64) / dims))
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * freq
    return torch.cat((angle.cos(), angle.sin()), 1).float().cuda().contiguous()


class AttentionBlock:
    """One layer's weights, its cache pool and the buffers of its widest batch."""

    def __init__(self, width, query_heads, kv_heads, max_seqs, max_tokens, codec=qb.CODEC_Q8_HEAD_F16, max_rows=4096,
                 seed=0):
        g = torch.Generator("cuda").manual_seed(seed)
        self.width, self.hq, self.hk = width, query_heads, kv_heads
        qkv_width = (query_heads + 2 * kv_heads) * HEAD
        self.norm = (1 + 0.1 * torch.randn(width, device="cuda", generator=g)).bfloat16()
        self.wqkv = quantise_rows(torch.randn((qkv_width, width), device="cuda", generator=g) / math.sqrt(width))
        self.wout = quantise_rows(torch.randn((width, query_heads * HEAD), device="cuda", generator=g)
                                  / math.sqrt(query_heads * HEAD))
        self.qkv_product = qb.MatmulQ8(self.wqkv[0], qkv_width, width, self.wqkv[1])
        self.out_product = qb.MatmulQ8(self.wout[0], width, query_heads * HEAD, self.wout[1])
        pages = -(-max_tokens // 16)
        self.pool = qb.KvPool(codec, 1, kv_heads, 16, max_seqs * pages, max_seqs, pages, max_query_heads=query_heads)
        self.table = rotations(max_tokens)
        self.codes = torch.empty((max_rows, max(width, query_heads * HEAD)), dtype=torch.int8, device="cuda")
        self.scales = torch.empty(max_rows, device="cuda")
        self.qkv = torch.empty((max_rows, qkv_width), dtype=torch.bfloat16, device="cuda")
        self.query = torch.empty((max_rows, query_heads, HEAD), device="cuda")  # decode() reads fp32

    def project(self, x, residual):
        """Adds x to the residual stream in place, norms it, and fills self.qkv."""
        rows = x.shape[0]
        qb.rmsnorm_q8(x, rows, self.width, qb.DTYPE_BF16, self.codes, self.scales, weight=self.norm, eps=EPS,
                      residual=residual, residual_out=residual, codes_stride=self.codes.shape[1])
        self.qkv_product(self.codes, self.scales, rows, self.qkv, qb.DTYPE_BF16, codes_stride=self.codes.shape[1])

    def store(self, seqs, rows, row_begin=None):
        """Rotates the rows' queries and keys by their positions and stores keys and values."""
        wide, q = self.qkv.shape[1], self.hq * HEAD
        self.pool.append_rotary(0, seqs, rows, qb.DTYPE_BF16, self.qkv[:, q:], self.qkv[:, q + self.hk * HEAD:],
                                query=self.qkv, query_heads=self.hq, query_out=self.query, rotations=self.table,
                                rotary_dim=HEAD, max_position=self.table.shape[0], row_begin=row_begin,
                                query_stride=wide, key_stride=wide, value_stride=wide)

    def output(self, attended, rows):
        """Attention rows (fp32) through the output product: bf16, to be added by the next norm."""
        out = torch.empty((rows, self.width), dtype=torch.bfloat16, device="cuda")
        qb.rmsnorm_q8(attended, rows, self.hq * HEAD, qb.DTYPE_F32, self.codes, self.scales, norm=False,
                      codes_stride=self.codes.shape[1])
        self.out_product(self.codes, self.scales, rows, out, qb.DTYPE_BF16, codes_stride=self.codes.shape[1])
        return out

    def prompt(self, x, residual, counts):
        """`counts[i]` more tokens of each sequence i: rows of x and residual, sequence after sequence."""
        seqs, rows = len(counts), x.shape[0]
        begin = torch.tensor([0] + counts, device="cuda").cumsum(0).int()
        self.project(x, residual)
        self.pool.seq_append(seqs, counts=torch.tensor(counts, dtype=torch.int32, device="cuda"))
        self.store(seqs, rows, begin)
        lens = [int(n) for n in self.pool.lens()[:seqs]]
        held = torch.tensor([0] + lens, device="cuda").cumsum(0).int()
        key, value = (torch.empty((sum(lens), self.hk, HEAD), device="cuda") for _ in range(2))
        self.pool.load_tokens(0, seqs, sum(lens), qb.DTYPE_F32, key, value, row_begin=held)
        out = torch.empty((rows, self.hq, HEAD), device="cuda")
        at = 0
        for i, n in enumerate(counts):
            k, v = (t[int(held[i]):int(held[i + 1])].repeat_interleave(self.hq // self.hk, 1) for t in (key, value))
            s = torch.einsum("qhd,khd->hqk", self.query[at:at + n], k) / math.sqrt(HEAD)
            future = torch.arange(lens[i], device="cuda") > torch.arange(lens[i] - n, lens[i], device="cuda")[:, None]
            out[at:at + n] = torch.einsum("hqk,khd->qhd", s.masked_fill(future, -torch.inf).softmax(-1), v)
            at += n
        return self.output(out, rows)

    def step(self, x, residual):
        """One token of every sequence."""
        seqs = x.shape[0]
        self.project(x, residual)
        self.pool.seq_append(seqs)
        self.store(seqs, seqs)
        out = torch.empty((seqs, self.hq, HEAD), device="cuda")
        self.pool.decode(0, seqs, self.hq, self.query, out)
        return self.output(out, seqs)

    def check(self):
        return self.pool.check() | self.qkv_product.check() | self.out_product.check()

    def close(self):
        self.pool.close()
        self.qkv_product.close()
        self.out_product.close()


def main():
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--codec", type=int, default=qb.CODEC_Q8_HEAD_F16, choices=[1, 2, 3, 4, 5])
    ap.add_argument("--steps", type=int, default=64)
    a = ap.parse_args()
    counts = [1000, 37, 512, 1]
    block = AttentionBlock(4096, 32, 8, len(counts), 2048, a.codec)
    g = torch.Generator("cuda").manual_seed(1)
    x = torch.randn((sum(counts), 4096), device="cuda", generator=g).bfloat16()
    out = block.prompt(x, torch.zeros_like(x), counts)
    print(f"prompts of {counts} tokens: output rms {float(out.float().square().mean().sqrt()):.4f}")
    x = out[torch.tensor(counts, device="cuda").cumsum(0) - 1].contiguous()
    residual = torch.zeros_like(x)
    begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    for i in range(a.steps):
        if i == min(8, a.steps - 1):
            begin.record()
        x = block.step(x, residual)
    end.record()
    assert block.check() == 0
    timed = a.steps - min(8, a.steps - 1)
    print(f"{a.steps} steps of {len(counts)} sequences: {begin.elapsed_time(end) / timed * 1e3:.1f} us a step, "
          f"output rms {float(x.float().square().mean().sqrt()):.4f}, {qb.launch_count()} launches")
    block.close()


if __name__ == "__main__":
    main()
