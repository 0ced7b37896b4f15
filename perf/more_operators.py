"""Cases of a prompt's operators: attention of a chunk of new tokens over the
paged cache, attention of packed prompts over their own rows, and the rotated
append with positions on several axes.

``own`` false: elementary torch operations.  ``own`` true: the library's calls.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
TYPE_ID = {"f32": 1, "f16": 2, "bf16": 3}
CODEC_ID = {"q8b64": 1, "q8head": 2, "tq35": 3, "q4": 4, "f16": 5}
KV_BYTES = {"q8b64": 272, "q8head": 260, "tq35": 128, "q4": 160, "f16": 512}  # K and V of one token and head
HEAD = 128
SCALE = 1.0 / math.sqrt(HEAD)


def listed():
    return [
        # the newest token of one sequence, 12 query heads on 2 (latency)
        {"name": "chunk one token", "op": "chunk", "seqs": 1, "rows": 1, "context": 2048, "kv_heads": 2, "group": 6,
         "codec": "q8head", "type": "bf16", "page": 16, "window": 0},
        # four drafted tokens of each of 32 sequences are verified in one call
        {"name": "chunk drafts", "op": "chunk", "seqs": 32, "rows": 128, "context": 8192, "kv_heads": 8, "group": 4,
         "codec": "q8head", "type": "bf16", "page": 16, "window": 0},
        # fp32 rows as the decode calls take them, ragged, an odd number
        {"name": "chunk ragged fp32", "op": "chunk", "seqs": 5, "rows": 517, "context": 4099, "kv_heads": 2, "group": 6,
         "codec": "q8b64", "type": "f32", "page": 16, "window": 0},
        # the next chunk of a long prompt over a 4-bit cache
        {"name": "chunk prompt", "op": "chunk", "seqs": 1, "rows": 2048, "context": 32768, "kv_heads": 8, "group": 4,
         "codec": "q4", "type": "bf16", "page": 16, "window": 0},
        # a question of 33 tokens on a very long document, 48 query heads on 8
        {"name": "chunk long", "op": "chunk", "seqs": 1, "rows": 33, "context": 131072, "kv_heads": 8, "group": 6,
         "codec": "q8head", "type": "f16", "page": 64, "window": 0},
        # one short prompt
        {"name": "prompt short", "op": "prompt", "seqs": 1, "rows": 37, "kv_heads": 2, "group": 6, "type": "f16",
         "causal": True, "window": 0},
        # 13 prompts packed into one batch of 16384 rows
        {"name": "prompt packed", "op": "prompt", "seqs": 13, "rows": 16384, "kv_heads": 8, "group": 4, "type": "bf16",
         "causal": True, "window": 0},
        # one long prompt: arithmetic is the cost
        {"name": "prompt long", "op": "prompt", "seqs": 1, "rows": 8192, "kv_heads": 8, "group": 4, "type": "bf16",
         "causal": True, "window": 0},
        # fp32 rows that see the last 1000 tokens only
        {"name": "prompt window fp32", "op": "prompt", "seqs": 3, "rows": 4099, "kv_heads": 2, "group": 6,
         "type": "f32", "causal": True, "window": 1000},
        # a decode step after images: one row of every sequence, its time, height and width positions
        {"name": "axes step", "op": "axes", "seqs": 32, "rows": 32, "context": 8192, "kv_heads": 8, "group": 4,
         "codec": "q8head", "type": "bf16", "neighbours": False, "page": 16, "sections": "16,24,24"},
        # prompts of text and images into a 4-bit cache
        {"name": "axes prompts", "op": "axes", "seqs": 13, "rows": 16384, "context": 16384, "kv_heads": 8, "group": 4,
         "codec": "q4", "type": "bf16", "neighbours": False, "page": 16, "sections": "16,24,24"},
    ]


def _span(rng, lo, hi):
    """A size of [lo, hi], even over its logarithm: odd, or a power of two, or five of them."""
    x = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    how = rng.randrange(3)
    if how:
        x = (1, 5)[how - 1] << max(0, int(math.log2(max(1, x / (1, 5)[how - 1]))))
    else:
        x |= 1
    return min(max(x, lo), hi)


MOST_SCORES = 2.1e9  # query heads x rows x tokens of a sequence: the plain form holds them in 32 bits
MOST_FLOPS = 1.0e12
MOST_BYTES = 5.4e8


def draw(rng):
    c = _drawn(rng)
    while c["rows"] > c["seqs"] and _too_much(c):
        c["rows"] = max(c["seqs"], c["rows"] // 2)
    while "context" in c and _too_much(c):
        c["context"] //= 2
    return c


def _too_much(c):
    w = work(c)
    heads = c["kv_heads"] * c["group"]
    scores = 0 if c["op"] == "axes" else max(heads * n * (f + n) for f, n in zip(*_runs(c)))
    return w["flops"] > MOST_FLOPS or w["bytes"] > MOST_BYTES or scores > MOST_SCORES


def _drawn(rng):
    op = rng.choice(("chunk", "chunk", "prompt", "prompt", "axes"))
    kind = rng.choice(("bf16", "bf16", "f16", "f32"))
    kv, group = rng.choice((1, 2, 4, 8)), rng.choice((1, 2, 4, 6, 8))
    if op == "prompt":
        seqs = _span(rng, 1, 32)
        causal = rng.random() < 0.8
        return {"op": op, "seqs": seqs, "rows": max(seqs, _span(rng, 1, 16384)), "kv_heads": kv, "group": group,
                "type": kind, "causal": causal, "window": _span(rng, 16, 4096) if causal and rng.random() < 0.25 else 0}
    codec, page = rng.choice(sorted(CODEC_ID)), rng.choice((16, 64))
    seqs = _span(rng, 1, 32)
    if op == "chunk":
        rows = seqs * _span(rng, 1, 16) if rng.random() < 0.5 else max(seqs, _span(rng, 1, 4096))
        context = _span(rng, 16, 131072 if seqs == 1 else 16384)
        return {"op": op, "seqs": seqs, "rows": rows, "context": context, "kv_heads": kv, "group": group,
                "codec": codec, "type": kind, "page": page,
                "window": _span(rng, 16, 4096) if rng.random() < 0.2 else 0}
    rows = seqs if rng.random() < 0.4 else max(seqs, _span(rng, 1, 16384))
    return {"op": op, "seqs": seqs, "rows": rows, "context": _span(rng, 16, 16384), "kv_heads": kv,
            "group": rng.choice((1, 2, 4, 6)), "codec": codec, "type": kind, "neighbours": rng.random() < 0.3,
            "page": page, "sections": rng.choice(("16,24,24", "24,20,20", "8,12,12", "32,32,0", "4,4,8"))}


def _runs(c):
    """Of each sequence the tokens it holds already, and its rows: unevenly, one row at least."""
    g = torch.Generator().manual_seed(c["rows"] * 131 + c["seqs"])
    seqs, rows = c["seqs"], c["rows"]
    share = torch.rand(seqs, generator=g) + 0.2
    if c["op"] == "chunk" and rows % seqs == 0:  # as many drafts of each
        n = torch.full((seqs,), rows // seqs)
    else:
        n = 1 + (share / share.sum() * (rows - seqs)).floor().long()
        n[0] += rows - int(n.sum())
    if c["op"] == "prompt":
        first = torch.zeros(seqs, dtype=torch.long)
    elif seqs == 1:
        first = torch.tensor([c["context"]])
    else:
        first = (torch.rand(seqs, generator=g) * c["context"]).long()
    return first.tolist(), n.tolist()


def work(case):
    c, es = case, SIZE[case["type"]]
    cached = c["rows"] * c["kv_heads"]
    q = cached * c["group"] * HEAD
    if c["op"] == "axes":
        # query in and out, new rows in, cache out and back, rows read back, three positions of each row
        return {"bytes": 2 * q * es + cached * (4 * HEAD * es + 2 * KV_BYTES[c["codec"]]) + 12 * c["rows"],
                "flops": 3 * q + 10 * cached * 2 * HEAD}
    pairs = tokens = 0
    for f, n in zip(*_runs(c)):
        w = c["window"] or f + n
        if c.get("causal", True):  # rows see f + 1 .. f + n tokens, the window's at most
            low = min(n, max(0, w - f))
            pairs += low * f + low * (low + 1) // 2 + (n - low) * w
            tokens += min(f + n, w + n - 1)
        else:
            pairs += n * n
            tokens += n
    kv_bytes = 2 * HEAD * es if c["op"] == "prompt" else KV_BYTES[c["codec"]]
    return {"bytes": 2 * q * es + tokens * c["kv_heads"] * kv_bytes,
            "flops": 4 * HEAD * c["kv_heads"] * c["group"] * pairs}


# ---- inputs -----------------------------------------------------------------

def _channels(width, g):
    """One channel in a hundred is eight times the others, as in a model's activations."""
    return torch.where(torch.rand(width, device=DEV, generator=g) < 0.01, 8.0, 1.0)


def prepare(case, seed):
    c, g = case, torch.Generator(DEV).manual_seed(seed)
    s = {"case": dict(c)}
    first, n = _runs(c)
    rows, seqs, kv, heads = c["rows"], c["seqs"], c["kv_heads"], c["kv_heads"] * c["group"]
    s["first"], s["counts"] = first, n
    begin = [0]
    for k in n:
        begin.append(begin[-1] + k)
    s["begin"] = torch.tensor(begin, dtype=torch.int32, device=DEV)
    kind = TYPES[c["type"]]
    if c["op"] == "prompt":
        # the projection's output after its rotation: query, key and value heads side by side in one row
        x = torch.randn((rows, heads + 2 * kv, HEAD), device=DEV, generator=g)
        x[:, :heads + kv] *= _channels(HEAD, g)
        s["qkv"] = x.to(kind).view(rows, -1)
        if own:
            s["out"] = torch.empty((rows, heads * HEAD), dtype=kind, device=DEV)
        return s
    lens = [f + k for f, k in zip(first, n)]
    pages = [-(-t // c["page"]) for t in lens]
    if c["op"] == "chunk":
        wide = _channels(HEAD, g)
        s["query"] = (torch.randn((rows, heads, HEAD), device=DEV, generator=g) * wide).to(kind)
        total = sum(lens)
        key = torch.randn((total, kv, HEAD), device=DEV, generator=g) * wide
        value = torch.randn((total, kv, HEAD), device=DEV, generator=g)
        _plain_cache(c, s, lens, pages, key, value, g)
    else:
        s["qkv"] = (torch.randn((rows, (c["group"] + 2) * kv * HEAD), device=DEV, generator=g)
                    * _channels((c["group"] + 2) * kv * HEAD, g)).to(kind)
        s["positions"] = _axis_positions(c, first, n, g)
        dims = 2 * sum(_sections(c))
        freq = 1.0 / (1e6 ** (torch.arange(0, dims, 2, device=DEV, dtype=torch.float64) / dims))
        s["max_position"] = c["context"] + rows
        angle = torch.arange(s["max_position"], device=DEV, dtype=torch.float64)[:, None] * freq
        s["rotations"] = torch.cat((angle.cos(), angle.sin()), 1).float()
    if own:
        import qwanto_b200 as qb
        pool = s["pool"] = qb.KvPool(CODEC_ID[c["codec"]], 1, kv, c["page"], sum(pages), seqs, max(pages),
                                     max_query_heads=heads, permutation_seed=seed + 1)
        pool.seq_append(seqs, counts=torch.tensor(lens, dtype=torch.int32, device=DEV))
        if c["op"] == "chunk":
            at = 0
            for i, t in enumerate(lens):
                pool.store_tokens(i, 0, 0, t, key[at:at + t], value[at:at + t])
                at += t
            s["out"] = torch.empty((rows, heads, HEAD), dtype=kind, device=DEV)
            s["workspace"] = torch.empty(pool.chunk_workspace(seqs, rows, heads), dtype=torch.uint8, device=DEV)
        else:
            s["query"] = torch.empty((rows, heads, HEAD), dtype=kind, device=DEV)
            s["key"] = torch.empty((rows, kv, HEAD), dtype=kind, device=DEV)
            s["value"] = torch.empty_like(s["key"])
        torch.cuda.synchronize()  # the pool's rows come from tensors that end here
    return s


def _plain_cache(c, s, lens, pages, key, value, g):
    """Codes and their parameters by page slot, the pages in any order; the slots of every sequence's tokens."""
    page = c["page"]
    order = torch.randperm(sum(pages), device=DEV, generator=g)
    at, slots = 0, []
    for t, m in zip(lens, pages):
        x = torch.arange(t, device=DEV)
        slots.append(order[at + x // page] * page + x % page)
        at += m
    s["slots"] = slots
    every, held = torch.cat(slots), sum(pages) * page
    s["cache"] = [tuple(torch.zeros((held, *e.shape[1:]), dtype=e.dtype, device=DEV).index_copy_(0, every, e)
                        for e in _encode(c["codec"], x)) for x in (key, value)]


def _sections(c):
    return [int(x) for x in c["sections"].split(",")]


def _axis_positions(c, first, n, g):
    """Time, height and width of every row: text counts all three up, an image (of up to 40 x 40 patches)
    keeps the time and walks its grid."""
    out = []
    for f, k in zip(first, n):
        x = torch.arange(k)
        side = min(40, max(1, math.isqrt(k) // 2))
        image = (x >= k // 4) & (x < k // 4 + side * side)
        y = (x - k // 4).clamp(min=0)
        base = f + k // 4
        after = torch.where(x >= k // 4 + side * side, x - side * side + side, x) + f
        out.append(torch.stack([torch.where(image, base, after), torch.where(image, base + y // side, after),
                                torch.where(image, base + y % side, after)]))
    return torch.cat(out, 1).int().to(DEV).contiguous()


# ---- the codecs in plain form ---------------------------------------------------

def _half_down(x):
    """fp16 with the excess bits cut off, as fp32."""
    a = x.abs()
    cut = (a.view(torch.int32) & ~0x1FFF).view(torch.float32)
    small = torch.floor(a * 2.0 ** 24) * 2.0 ** -24
    return torch.copysign(torch.where(a < 2.0 ** -14, small, torch.where(a >= 65536.0, torch.inf, cut)), x)


def _encode(codec, x):
    """Codes and parameters of fp32 rows [.., 128]."""
    if codec == "f16":
        return (x.half(),)
    if codec in ("q8head", "q8b64"):
        y = x.reshape(*x.shape[:-1], 1 if codec == "q8head" else 2, -1)
        top = y.abs().amax(-1, keepdim=True)
        scale = torch.where(top > 0, top / torch.full_like(top, 127.0), 1.0)
        if codec == "q8head":
            scale = scale.half().float().clamp(2.0 ** -24, 65504.0)
        code = (y / scale).round().clamp(-127, 127)
        return code.to(torch.int8), scale.half() if codec == "q8head" else scale
    y = x.reshape(*x.shape[:-1], -1, 32 if codec == "q4" else 64)
    low = y.amin(-1, keepdim=True)
    span = y.amax(-1, keepdim=True) - low
    norm = ((y - low) * torch.where(span > 1e-8, torch.ones_like(span) / span, 0.0)).clamp(0, 1) * _levels(codec, x)
    code = norm.floor() + (norm - norm.floor() >= 0.5)
    return code.to(torch.uint8), _half_down(span).half(), _half_down(low).half()


def _levels(codec, x):
    """Steps of a code: 15, and for TurboQuant 15 and 7 in turn."""
    n = torch.full((32 if codec == "q4" else 64,), 15.0, device=x.device, dtype=torch.float32)
    if codec == "tq35":
        n[1::2] = 7.0
    return n


def _decode(codec, enc):
    if codec == "f16":
        return enc[0].float()
    if codec in ("q8head", "q8b64"):
        return (enc[0].float() * enc[1].float()).flatten(-2)
    return (enc[0].float() * (enc[1].float() / _levels(codec, enc[0])) + enc[2].float()).flatten(-2)


# ---- one pass -------------------------------------------------------------------

def run(state):
    return (_run_own if own else _run_plain)(state)


def _attend(q, k, v, first, causal, window):
    """q [rows, heads, 128] at positions first.. over k, v [tokens, kv heads, 128], in fp32."""
    rows, heads, kv = q.shape[0], q.shape[1], k.shape[1]
    # the heads that share a kv head are rows of one product
    x = q.float().view(rows, kv, -1, HEAD).permute(1, 2, 0, 3).reshape(kv, -1, HEAD)
    scores = (x @ k.float().permute(1, 2, 0)).view(kv, -1, rows, k.shape[0]) * SCALE
    if causal:
        pos = first + torch.arange(rows, device=DEV)[:, None]
        at = torch.arange(k.shape[0], device=DEV)
        hidden = (at > pos) | (at <= pos - window) if window else at > pos
        scores.masked_fill_(hidden, -math.inf)
    p = (scores - scores.amax(-1, keepdim=True)).exp_()
    del scores
    total = p.sum(-1, keepdim=True)
    out = (p.view(kv, -1, k.shape[0]) @ v.float().transpose(0, 1)).view(kv, -1, rows, HEAD) / total
    return out.permute(2, 0, 1, 3).reshape(rows, heads, HEAD).to(q.dtype)


def _run_plain(s):
    c, kind = s["case"], TYPES[s["case"]["type"]]
    kv, heads = c["kv_heads"], c["kv_heads"] * c["group"]
    if c["op"] == "axes":
        x = s["qkv"].float().view(c["rows"], heads + 2 * kv, HEAD)
        turned = _rotate(x[:, :heads + kv], _row_angles(c, s), c["neighbours"])
        k, v = (_decode(c["codec"], _encode(c["codec"], y.contiguous())).to(kind)
                for y in (turned[:, heads:], x[:, heads + kv:]))
        return {"query": turned[:, :heads].to(kind), "key": k, "value": v}
    out, at = [], 0
    for i, (f, n) in enumerate(zip(s["first"], s["counts"])):
        if c["op"] == "prompt":
            x = s["qkv"][at:at + n].view(n, heads + 2 * kv, HEAD)
            q, k, v = x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:]
        else:
            q = s["query"][at:at + n]
            k, v = (_decode(c["codec"], [e[s["slots"][i]] for e in cache]) for cache in s["cache"])
        out.append(_attend(q, k, v, f, c.get("causal", True), c["window"]))
        at += n
    return {"out": torch.cat(out)}


def _row_angles(c, s):
    """Each row's cosines and sines: every frequency's from the position on its section's axis."""
    table = s["rotations"]
    axis = torch.repeat_interleave(torch.arange(3, device=DEV), torch.tensor(_sections(c), device=DEV)).repeat(2)
    rows = s["positions"].long()[axis].T  # [rows, rotary dims]
    return table.gather(0, rows)


def _rotate(x, cs, neighbours):
    """x [rows, heads, 128] with the first dims of each head rotated by the rows' angles."""
    r = cs.shape[-1]
    c, s = cs[:, None, :r // 2], cs[:, None, r // 2:]
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if neighbours else (x[..., :r // 2], x[..., r // 2:r])
    u, w = a * c - b * s, b * c + a * s
    y = torch.stack((u, w), -1).flatten(-2) if neighbours else torch.cat((u, w), -1)
    return torch.cat((y, x[..., r:]), -1)


def _run_own(s):
    import qwanto_b200 as qb
    c = s["case"]
    t, kv, heads = TYPE_ID[c["type"]], c["kv_heads"], c["kv_heads"] * c["group"]
    one = c["rows"] == c["seqs"]  # a decode step: the newest token of each sequence
    if c["op"] == "prompt":
        qkv = s["qkv"]
        wide = qkv.shape[1]
        qb.prompt_attention(qkv, qkv[:, heads * HEAD:], qkv[:, (heads + kv) * HEAD:], s["out"], c["rows"], t, heads, kv,
                            num_seqs=c["seqs"], row_begin=s["begin"], causal=c["causal"], window=c["window"],
                            query_stride=wide, key_stride=wide, value_stride=wide)
        return {"out": s["out"].view(c["rows"], heads, HEAD)}
    if c["op"] == "chunk":
        s["pool"].chunk_attention(0, c["seqs"], c["rows"], t, heads, s["query"], s["out"],
                                  row_begin=None if one else s["begin"], window=c["window"],
                                  workspace=s["workspace"], workspace_bytes=s["workspace"].numel())
        return {"out": s["out"]}
    qkv = s["qkv"]
    wide, sections = qkv.shape[1], _sections(c)
    s["pool"].append_rotary(0, c["seqs"], c["rows"], t, qkv[:, heads * HEAD:], qkv[:, (heads + kv) * HEAD:],
                            row_begin=None if one else s["begin"], query=qkv, query_heads=heads, query_out=s["query"],
                            query_out_dtype=t, rotations=s["rotations"], rotary_dim=2 * sum(sections),
                            max_position=s["max_position"], neighbours=c["neighbours"], query_stride=wide,
                            key_stride=wide, value_stride=wide, rotary_pos=s["positions"], rotary_sections=sections)
    s["pool"].load_tokens(0, c["seqs"], c["rows"], t, s["key"], s["value"], row_begin=None if one else s["begin"])
    return {"query": s["query"], "key": s["key"], "value": s["value"]}


# ---- 64 bits --------------------------------------------------------------------

def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    c = case
    kv, g = c["kv_heads"], c["group"]
    if c["op"] == "axes":
        return _exact_axes(c, s)
    out = torch.empty((c["rows"], kv * g, HEAD), dtype=torch.float64, device=DEV)
    start = 0
    for i, (f, n) in enumerate(zip(s["first"], s["counts"])):
        rows = slice(start, start + n)
        if c["op"] == "chunk":
            q = s["query"][rows]
            k, v = (_exact_values(c["codec"], [e.index_select(0, s["slots"][i]) for e in cache]) for cache in s["cache"])
        else:
            q, k, v = s["qkv"][rows].reshape(n, -1, HEAD).split((kv * g, kv, kv), 1)
        tokens = torch.arange(k.shape[0], device=DEV)[None]
        newest = torch.arange(f, f + n, device=DEV)[:, None]
        seen = torch.ones((n, k.shape[0]), dtype=torch.bool, device=DEV)
        if c.get("causal", True):
            seen = tokens <= newest
        if c["window"]:
            seen = seen & (newest - tokens < c["window"])
        for h in range(kv * g):
            kh, vh = k[:, h // g].double(), v[:, h // g].double()
            logits = torch.einsum("rd,td->rt", q[:, h].double(), kh) / math.sqrt(HEAD)
            out[rows, h] = torch.softmax(logits.where(seen, torch.full_like(logits, -math.inf)), -1) @ vh
        start += n
    return {"out": out}


def _exact_axes(c, s):
    kv, hq, half = c["kv_heads"], c["group"] * c["kv_heads"], sum(_sections(c))
    x = s["qkv"].double().reshape(c["rows"], -1, HEAD)
    q, k, v = x[:, :hq].clone(), x[:, hq:hq + kv].clone(), x[:, hq + kv:]
    bound, at = [], 0
    for size in _sections(c):  # the frequencies of an axis are a run of the table's columns
        where = s["positions"][len(bound)].long()
        part = s["rotations"].double().index_select(0, where)
        bound.append(torch.complex(part[:, at:at + size], part[:, half + at:half + at + size]))
        at += size
    turn = torch.cat(bound, 1)[:, None]
    i, j = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if c["neighbours"] else (slice(0, half), slice(half, 2 * half))
    for y in (q, k):  # a pair is a complex number, its rotation a product
        z = torch.complex(y[..., i], y[..., j]) * turn
        y[..., i], y[..., j] = z.real.clone(), z.imag.clone()
    return {"query": q, "key": _exact_cached(c["codec"], k), "value": _exact_cached(c["codec"], v)}


def _exact_values(codec, enc):
    if codec == "f16":
        return enc[0].double()
    code = enc[0].double()
    if len(enc) == 2:
        return (code * enc[1].double()).reshape(*code.shape[:-2], HEAD)
    odd = torch.arange(code.shape[-1], device=code.device) % 2 == 1
    step = torch.where(odd & (codec == "tq35"), 7.0, 15.0).double()
    return (enc[2].double() + code / step * enc[1].double()).reshape(*code.shape[:-2], HEAD)


def _exact_cached(codec, x):
    """The values that the cache holds for x: the codec's definition."""
    if codec == "f16":
        return x.half().double()
    y = x.reshape(*x.shape[:-1], {"q8head": 1, "q8b64": 2, "q4": 4, "tq35": 2}[codec], -1)
    if codec.startswith("q8"):
        step = y.abs().max(-1, keepdim=True).values / 127
        step = torch.where(step > 0, step, torch.ones_like(step))
        step = step.half().double().clamp_min(2.0 ** -24) if codec == "q8head" else step.float().double()
        return (torch.round(y / step).clamp(-127, 127) * step).reshape(x.shape)
    low, high = y.min(-1, keepdim=True).values, y.max(-1, keepdim=True).values
    odd = torch.arange(y.shape[-1], device=x.device) % 2 == 1
    top = torch.where(odd & (codec == "tq35"), 7.0, 15.0).double()
    code = torch.floor((y - low) / (high - low).clamp_min(1e-300) * top + 0.5)

    def down(z):  # towards zero in ten bits after the leading one
        e = torch.floor(torch.log2(z.abs().clamp_min(2.0 ** -14)))
        unit = torch.exp2(e - 10)
        return torch.trunc(z / unit) * unit
    return (down(low) + code / top * down(high - low)).reshape(x.shape)
