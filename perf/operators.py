"""Cases of the operators around the paged cache: the int8 norm, the int8
product, the rotated append and the read-back of cached rows.

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
MAX_POSITION = 131072  # rows of the rotation table
EPS = 1e-6


def listed():
    return [
        # one token of one sequence before the projections: 12 heads of 128, fp32 activations (latency)
        {"name": "norm one token", "op": "norm", "rows": 1, "width": 1536, "type": "f32", "residual": True},
        # a decode batch of 32 sequences, 32 heads of 128
        {"name": "norm batch", "op": "norm", "rows": 32, "width": 4096, "type": "bf16", "residual": True},
        # a long prompt, an odd number of tokens, 48 heads of 128
        {"name": "norm prompt", "op": "norm", "rows": 8191, "width": 6144, "type": "f16", "residual": True},
        # one token through the fused query/key/value projection of 12 + 2 + 2 heads
        {"name": "matmul one token", "op": "matmul", "rows": 1, "k": 1536, "n": 2048, "type": "f32", "bias": True},
        # a decode batch of 32 sequences through 32 + 8 + 8 heads: the weights are the traffic
        {"name": "matmul batch", "op": "matmul", "rows": 32, "k": 4096, "n": 6144, "type": "bf16", "bias": False},
        # a ragged chunk with sizes off every tile
        {"name": "matmul ragged", "op": "matmul", "rows": 257, "k": 4099, "n": 4095, "type": "f16", "bias": True},
        # a long prompt through 48 + 8 + 8 heads: arithmetic is the cost
        {"name": "matmul prompt", "op": "matmul", "rows": 8192, "k": 6144, "n": 8192, "type": "bf16", "bias": False},
        # one decode step of one sequence at 2048 tokens, 12 query heads on 2
        {"name": "append one token", "op": "append", "seqs": 1, "rows": 1, "context": 2048, "kv_heads": 2, "group": 6,
         "codec": "q8head", "type": "f32", "query_type": "f32", "rotary": 128, "neighbours": False, "page": 16},
        # one decode step of 32 sequences, 32 query heads on 8
        {"name": "append batch", "op": "append", "seqs": 32, "rows": 32, "context": 8192, "kv_heads": 8, "group": 4,
         "codec": "q8head", "type": "bf16", "query_type": "f32", "rotary": 128, "neighbours": False, "page": 16},
        # prompts of 13 sequences, ragged and off the page grid, into a 4-bit cache
        {"name": "append prompts", "op": "append", "seqs": 13, "rows": 16384, "context": 16384, "kv_heads": 8,
         "group": 4, "codec": "q4", "type": "bf16", "query_type": "bf16", "rotary": 128, "neighbours": False,
         "page": 16},
        # a short prefix read back for a prompt's next chunk
        {"name": "read short", "op": "read", "seqs": 1, "rows": 1001, "kv_heads": 2, "codec": "q8b64", "type": "f32",
         "page": 16},
        # the whole cache of one long sequence read back, pages of 64
        {"name": "read long", "op": "read", "seqs": 1, "rows": 131072, "kv_heads": 8, "codec": "q8head",
         "type": "bf16", "page": 64},
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


MOST_BYTES = 8.0e8  # of the largest listed case


def draw(rng):
    c = _drawn(rng)
    while work(c)["bytes"] > MOST_BYTES:
        c["rows"] = max(c.get("seqs", 1), c["rows"] // 2)
    return c


def _drawn(rng):
    op = rng.choice(("norm", "matmul", "append", "read"))
    kind = rng.choice(("f32", "f16", "bf16"))
    if op == "norm":
        return {"op": op, "rows": _span(rng, 1, 8192), "width": _span(rng, 256, 12288), "type": kind,
                "residual": rng.random() < 0.75}
    if op == "matmul":
        rows, k = _span(rng, 1, 8192), _span(rng, 64, 6144)
        return {"op": op, "rows": rows, "k": k, "n": _span(rng, 16, 8192 if rows > 256 else 16384), "type": kind,
                "bias": rng.random() < 0.5}
    kv, codec = rng.choice((1, 2, 4, 8)), rng.choice(sorted(CODEC_ID))
    page = rng.choice((16, 64))
    if op == "append":
        seqs = _span(rng, 1, 64)
        rows = seqs if rng.random() < 0.4 else max(seqs, _span(rng, 1, 16384))
        return {"op": op, "seqs": seqs, "rows": rows, "context": _span(rng, 16, 16384), "kv_heads": kv,
                "group": rng.choice((1, 2, 4, 6)), "codec": codec, "type": kind, "query_type": rng.choice((kind, "f32")),
                "rotary": rng.choice((32, 64, 96, 128, 128)), "neighbours": rng.random() < 0.3, "page": page}
    seqs = _span(rng, 1, 32)
    return {"op": op, "seqs": seqs, "rows": max(seqs, _span(rng, 1, 131072)), "kv_heads": kv, "codec": codec,
            "type": kind, "page": page}


def work(case):
    c, es = case, SIZE[case["type"]]
    if c["op"] == "norm":
        n = c["rows"] * c["width"]
        # x, residual in and out, codes, the rows in 16 bits, scales, weights
        return {"bytes": n * (es * (3 if c["residual"] else 1) + 1 + 2) + 4 * c["rows"] + es * c["width"],
                "flops": 8 * n}
    if c["op"] == "matmul":
        m, k, n = c["rows"], c["k"], c["n"]
        return {"bytes": m * k + n * k + m * n * es + 4 * (m + n) + (4 * n if c["bias"] else 0),
                "flops": 2 * m * k * n}
    cached = c["rows"] * c["kv_heads"]
    if c["op"] == "read":
        return {"bytes": cached * (KV_BYTES[c["codec"]] + 2 * HEAD * es), "flops": cached * 2 * HEAD * 2}
    q = cached * c["group"] * HEAD
    # query in and out, new rows in, cache out and back, rows read back, the positions' rotations
    return {"bytes": q * (es + SIZE[c["query_type"]]) + cached * (2 * HEAD * es + 2 * KV_BYTES[c["codec"]] + 2 * HEAD * es)
            + c["rows"] * c["rotary"] * 4, "flops": 3 * q + 10 * cached * 2 * HEAD}


# ---- inputs -----------------------------------------------------------------

def _normal(shape, g, kind="f32", scale=1.0):
    return (torch.randn(shape, device=DEV, generator=g) * scale).to(TYPES[kind])


def _channels(width, g):
    """One channel in a hundred is eight times the others, as in a model's activations."""
    return torch.where(torch.rand(width, device=DEV, generator=g) < 0.01, 8.0, 1.0)


def _lengths(total, seqs, seed):
    """`total` rows over the sequences, unevenly, one at least for each."""
    g = torch.Generator().manual_seed(seed)
    share = torch.rand(seqs, generator=g) + 0.2
    n = 1 + (share / share.sum() * (total - seqs)).floor().long()
    n[0] += total - int(n.sum())
    return n


def _rotations(dims):
    """The rotation table: of every position the cosines of the frequencies' angles, then their sines."""
    freq = 1.0 / (1e6 ** (torch.arange(0, dims, 2, device=DEV, dtype=torch.float64) / dims))
    angle = torch.arange(MAX_POSITION, device=DEV, dtype=torch.float64)[:, None] * freq
    return torch.cat((angle.cos(), angle.sin()), 1).float()


def prepare(case, seed):
    c, g = case, torch.Generator(DEV).manual_seed(seed)
    s = {"case": dict(c)}
    if c["op"] == "norm":
        t, w = c["rows"], c["width"]
        s["x"] = _normal((t, w), g, c["type"])
        s["weight"] = (1 + 0.1 * torch.randn(w, device=DEV, generator=g)).to(TYPES[c["type"]])
        if c["residual"]:
            s["residual"] = (torch.randn((t, w), device=DEV, generator=g) * _channels(w, g)).to(TYPES[c["type"]])
        if own:
            stride = -(-w // 16) * 16
            s["codes"] = torch.zeros((t, stride), dtype=torch.int8, device=DEV)
            s["scales"] = torch.empty(t, device=DEV)
            s["rows16"] = torch.empty((t, w), dtype=torch.bfloat16, device=DEV)
            s["sum"] = torch.empty_like(s["x"])
    elif c["op"] == "matmul":
        m, k, n = c["rows"], c["k"], c["n"]
        stride = -(-k // 16) * 16  # rows of codes start on 16 bytes
        full = torch.zeros((m, stride), dtype=torch.int8, device=DEV)
        full[:, :k] = (torch.randn((m, k), device=DEV, generator=g) * 34).round_().clamp_(-127, 127).to(torch.int8)
        s["codes"] = full[:, :k]
        s["scales"] = 0.01 + 0.03 * torch.rand(m, device=DEV, generator=g)
        s["weight"] = (torch.randn((n, k), device=DEV, generator=g) * 36).round_().clamp_(-127, 127).to(torch.int8)
        s["weight_scales"] = (0.5 + torch.rand(n, device=DEV, generator=g)) / (36 * math.sqrt(k))
        s["bias"] = torch.randn(n, device=DEV, generator=g) * 0.1 if c["bias"] else None
        if own:
            import qwanto_b200 as qb
            s["product"] = qb.MatmulQ8(s["weight"], n, k, s["weight_scales"], s["bias"])
            s["out"] = torch.empty((m, n), dtype=TYPES[c["type"]], device=DEV)
    else:
        k, v, lens, pages = _prepare_cache(c, seed, g, s)
        if own:
            import qwanto_b200 as qb
            rows, seqs, kv = c["rows"], c["seqs"], c["kv_heads"]
            s["pool"] = qb.KvPool(CODEC_ID[c["codec"]], 1, kv, c["page"], int(pages.sum()), seqs, int(pages.max()),
                                  permutation_seed=seed + 1)
            s["pool"].seq_append(seqs, counts=lens.int().to(DEV))
            if c["op"] == "append":
                s["query"] = torch.empty((rows, c["group"] * kv, HEAD), dtype=TYPES[c["query_type"]], device=DEV)
            else:
                for i, (a, b) in enumerate(zip(s["begin"].tolist(), s["begin"].tolist()[1:])):
                    s["pool"].store_tokens(i, 0, 0, b - a, k[a:b], v[a:b])
            s["key"] = torch.empty((rows, kv, HEAD), dtype=TYPES[c["type"]], device=DEV)
            s["value"] = torch.empty_like(s["key"])
            torch.cuda.synchronize()  # the pool's rows come from tensors that end here
    return s


def _prepare_cache(c, seed, g, s):
    seqs, rows, kv, page = c["seqs"], c["rows"], c["kv_heads"], c["page"]
    n = _lengths(rows, seqs, seed)
    if c["op"] == "append":  # the new rows follow on what each sequence holds already
        first = (torch.rand(seqs, generator=torch.Generator().manual_seed(seed + 1)) * c["context"]).long()
    else:
        first = torch.zeros(seqs, dtype=torch.long)
    s["first"] = first.int().to(DEV)
    s["begin"] = torch.cat((torch.zeros(1, dtype=torch.long), n.cumsum(0))).int().to(DEV)
    lens = first + n
    pages = (lens + page - 1) // page
    k = v = None
    if c["op"] == "append":
        where = [torch.arange(int(a), int(a + b)) for a, b in zip(first, n)]
        s["positions"] = torch.cat(where).int().to(DEV)
        width = (c["group"] + 2) * kv * HEAD
        # the projection's output: query, key and value heads side by side in one row
        s["qkv"] = (torch.randn((rows, width), device=DEV, generator=g) * _channels(width, g)).to(TYPES[c["type"]])
        s["rotations"] = _rotations(c["rotary"])
    else:
        k = torch.randn((rows, kv, HEAD), device=DEV, generator=g) * _channels(kv * HEAD, g).view(kv, HEAD)
        v = torch.randn((rows, kv, HEAD), device=DEV, generator=g)
        # the plain cache: codes and their parameters by page slot, the pages in any order
        order = torch.randperm(int(pages.sum()), device=DEV, generator=g)
        base = torch.cat((torch.zeros(1, dtype=torch.long), pages.cumsum(0)))
        at = torch.cat([torch.arange(int(m)) + int(b) * page for m, b in zip(n, base)]).to(DEV)
        s["slots"] = order[at // page] * page + at % page
        held = int(pages.sum()) * page
        s["cache"] = [tuple(torch.zeros((held, *e.shape[1:]), dtype=e.dtype, device=DEV).index_copy_(0, s["slots"], e)
                            for e in _encode(c["codec"], x)) for x in (k, v)]
    return k, v, lens, pages


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
        fine = y.isfinite()
        top = torch.where(fine, y.abs(), 0.0).amax(-1, keepdim=True)
        scale = torch.where(top > 0, top / torch.full_like(top, 127.0), 1.0)
        if codec == "q8head":
            scale = scale.half().float().clamp(2.0 ** -24, 65504.0)
        code = torch.where(fine, (y / scale).round().clamp(-127, 127), 0.0)
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


def _rotate(x, cs, neighbours):
    """x [rows, heads, 128] with the first dims of each head rotated by the rows' angles."""
    r = cs.shape[-1]
    c, s = cs[:, None, :r // 2], cs[:, None, r // 2:]
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if neighbours else (x[..., :r // 2], x[..., r // 2:r])
    u, w = a * c - b * s, b * c + a * s
    y = torch.stack((u, w), -1).flatten(-2) if neighbours else torch.cat((u, w), -1)
    return torch.cat((y, x[..., r:]), -1)


# ---- one pass -------------------------------------------------------------------

def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_plain(s):
    c, kind = s["case"], TYPES[s["case"]["type"]]
    if c["op"] == "norm":
        h = s["x"].float()
        if c["residual"]:
            h = h + s["residual"].float()
        y = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS) * s["weight"].float()
        top = y.abs().amax(-1, keepdim=True)
        scale = torch.where(top > 0, top / torch.full_like(top, 127.0), 1.0)
        rows = ((y / scale).round().clamp(-127, 127) * scale).bfloat16()
        return {"rows": rows, "scales": scale[:, 0], **({"sum": h.to(kind)} if c["residual"] else {})}
    if c["op"] == "matmul":
        y = (s["codes"].float() @ s["weight"].float().T) * s["scales"][:, None] * s["weight_scales"]
        return {"out": (y if s["bias"] is None else y + s["bias"]).to(kind)}
    if c["op"] == "read":
        k, v = (_decode(c["codec"], [e[s["slots"]] for e in cache]).to(kind) for cache in s["cache"])
        return {"key": k, "value": v}
    kv, hq = c["kv_heads"], c["group"] * c["kv_heads"]
    x = s["qkv"].float().view(c["rows"], hq + 2 * kv, HEAD)
    turned = _rotate(x[:, :hq + kv], s["rotations"][s["positions"]], c["neighbours"])
    k, v = (_decode(c["codec"], _encode(c["codec"], y.contiguous())).to(kind)
            for y in (turned[:, hq:], x[:, hq + kv:]))
    return {"query": turned[:, :hq].to(TYPES[c["query_type"]]), "key": k, "value": v}


def _run_own(s):
    import qwanto_b200 as qb
    c = s["case"]
    t = TYPE_ID[c["type"]]
    if c["op"] == "norm":
        qb.rmsnorm_q8(s["x"], c["rows"], c["width"], t, s["codes"], s["scales"], weight=s["weight"], eps=EPS,
                      residual=s.get("residual"), residual_out=s["sum"] if c["residual"] else None,
                      codes_stride=s["codes"].shape[1], rows_out=s["rows16"], rows_dtype=3)
        return {"rows": s["rows16"], "scales": s["scales"], **({"sum": s["sum"]} if c["residual"] else {})}
    if c["op"] == "matmul":
        s["product"](s["codes"], s["scales"], c["rows"], s["out"], t, codes_stride=s["codes"].stride(0))
        return {"out": s["out"]}
    if c["op"] == "append":
        kv, hq, qkv = c["kv_heads"], c["group"] * c["kv_heads"], s["qkv"]
        wide = qkv.shape[1]
        one = c["rows"] == c["seqs"]  # a decode step: the newest token of each sequence
        s["pool"].append_rotary(0, c["seqs"], c["rows"], t, qkv[:, hq * HEAD:], qkv[:, (hq + kv) * HEAD:],
                                row_begin=None if one else s["begin"], query=qkv, query_heads=hq,
                                query_out=s["query"], query_out_dtype=TYPE_ID[c["query_type"]],
                                rotations=s["rotations"], rotary_dim=c["rotary"], max_position=MAX_POSITION,
                                neighbours=c["neighbours"], query_stride=wide, key_stride=wide, value_stride=wide)
        s["pool"].load_tokens(0, c["seqs"], c["rows"], t, s["key"], s["value"], row_begin=None if one else s["begin"])
        return {"query": s["query"], "key": s["key"], "value": s["value"]}
    s["pool"].load_tokens(0, c["seqs"], c["rows"], t, s["key"], s["value"], row_begin=s["begin"])
    return {"key": s["key"], "value": s["value"]}


# ---- 64 bits --------------------------------------------------------------------

def exact(case, seed):
    c, s = case, _plain_state(case, seed)
    if c["op"] == "norm":
        h = s["x"].double() + (s["residual"].double() if c["residual"] else 0.0)
        y = h / (h.pow(2).sum(-1, keepdim=True) / c["width"] + EPS).sqrt() * s["weight"].double()
        step = y.abs().max(-1, keepdim=True).values / 127
        step[step == 0] = 1.0
        return {"rows": torch.round(y / step) * step, "scales": step.squeeze(-1), **({"sum": h} if c["residual"] else {})}
    if c["op"] == "matmul":
        y = torch.einsum("mk,nk->mn", s["codes"].double(), s["weight"].double())
        y = y * torch.outer(s["scales"].double(), s["weight_scales"].double())
        return {"out": y if s["bias"] is None else y + s["bias"].double()}
    if c["op"] == "read":
        return {name: _exact_values(c["codec"], [e.index_select(0, s["slots"]) for e in cache])
                for name, cache in zip(("key", "value"), s["cache"])}
    kv, hq, r = c["kv_heads"], c["group"] * c["kv_heads"], c["rotary"]
    x = s["qkv"].double().reshape(c["rows"], -1, HEAD)
    q, k, v = x[:, :hq].clone(), x[:, hq:hq + kv].clone(), x[:, hq + kv:]
    cs = s["rotations"].double()[s["positions"].long()]
    turn = torch.complex(cs[:, :r // 2], cs[:, r // 2:])[:, None]
    for y in (q, k):  # a pair is a complex number, its rotation a product
        i, j = (slice(0, r, 2), slice(1, r, 2)) if c["neighbours"] else (slice(0, r // 2), slice(r // 2, r))
        z = torch.complex(y[..., i], y[..., j]) * turn
        y[..., i], y[..., j] = z.real.clone(), z.imag.clone()
    return {"query": q, "key": _exact_cached(c["codec"], k), "value": _exact_cached(c["codec"], v)}


def _plain_state(case, seed):
    global own
    was, own = own, False
    try:
        return prepare(case, seed)
    finally:
        own = was


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
