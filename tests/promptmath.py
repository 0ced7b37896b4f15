"""Attention of rows in 64 bits, with a bound on what the library's arithmetic may
be off by, for the tests of qwn_kv_chunk_attention and qwn_prompt_attention.

With p the probabilities, A = sum p |v| and u half a step of the 16-bit type:
  - a score is off by `es`: its products and their fp32 sum (128 terms and the
    tensor core's own additions), the rounding of the operands where they are
    rounded (`dk`), and of scale x log2 e and the exponent (2^-21 of its size);
    a probability and the sum of all by 2 es of their size;
  - P is rounded to 16 bits (u), or held in 24 (fp32 rows); f16 loses what is
    below 2^-25, where the largest is 2^7 at least: 2^-32 of the row's sum each;
  - the values may be rounded (`dv`); n terms are added in fp32; the output is
    rounded once.
"""
import math

import torch

HEAD = 128
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
TYPE_ID = {"f32": 1, "f16": 2, "bf16": 3}
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def seen(first, rows, tokens, causal, window, device="cuda"):
    pos = first + torch.arange(rows, device=device)[:, None]
    at = torch.arange(tokens, device=device)[None]
    m = torch.ones((rows, tokens), dtype=torch.bool, device=device)
    if causal:
        m = at <= pos
    if window:
        m = m & (at > pos - window)
    return m


def attend(q, k, v, mask, scale=0.0, kind="bf16", p_step=None, dk=None, dv=None):
    """q [rows, heads, 128], k and v [tokens, kv heads, 128] (any type), mask [rows, tokens].  Returns the
    output in 64 bits and the largest distance that an output of type `kind` may have from it."""
    rows, heads, kv = q.shape[0], q.shape[1], k.shape[1]
    scale = scale or 1 / math.sqrt(HEAD)
    u, tokens = HALF_STEP[kind], k.shape[0]
    p_step = {"f32": 2.0 ** -23}.get(kind, u) if p_step is None else p_step
    zero = torch.zeros((), dtype=torch.float64, device=q.device)
    # what is masked in every row must not matter
    used = mask.any(0)[:, None, None]
    k, v = (torch.where(used, x.double(), zero) for x in (k, v))
    dk = zero.expand_as(k) if dk is None else torch.where(used, dk.double(), zero)
    dv = zero.expand_as(v) if dv is None else torch.where(used, dv.double(), zero)
    out = torch.zeros((rows, heads, HEAD), dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    if rows == 0:
        return out, tol
    for h in range(heads):
        a, b = q[:, h].double(), k[:, h // (heads // kv)]
        s = (a @ b.T * scale).masked_fill(~mask, -math.inf)
        es = (a.abs() @ b.abs().T * ((128 + 64) * 2.0 ** -24) + a.abs() @ dk[:, h // (heads // kv)].T) * scale
        es = es + s.abs().masked_fill(~mask, 0) * 2.0 ** -21
        p = torch.softmax(s, -1).masked_fill(~mask, 0)
        x = v[:, h // (heads // kv)]
        out[:, h] = p @ x
        size = p @ x.abs()
        rel = p_step + 2 * es.masked_fill(~mask, 0).amax(-1, keepdim=True) + (tokens + 64) * 2.0 ** -23 + 2.0 ** -21
        # f16 has steps of 2^-24 below 2^-14, whose half is more than u of the value
        lost = tokens * 2.0 ** -32 * (x.abs() * mask.any(0)[:, None]).amax() if kind != "f32" else 0.0
        lost = lost + (2.0 ** -25 if kind == "f16" else 2.0 ** -30)
        tol[:, h] = rel * size + p @ dv[:, h // (heads // kv)] + u * out[:, h].abs() + lost
    return out, tol


def assert_near(got, want, tol, what=""):
    got = got.double()
    bad = ~((got - want).abs() <= tol)
    if bad.any():
        i = torch.nonzero(bad)[0].tolist()
        worst = ((got - want).abs() / tol).nan_to_num(math.inf).max().item()
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} values off, first at {i}: "
                             f"{got[tuple(i)].item()} for {want[tuple(i)].item()} +- {tol[tuple(i)].item()}; worst {worst:.3g} x")
