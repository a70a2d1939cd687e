"""The token-serving operators of ``seldon_core_amd.ops`` as cases to measure.

Four operators that belong to one step of a served token model: low-rank
adapters added to a projection's output, the norm and rotation of the
projection's queries and keys, the paged key-value cache that keeps the keys
and values (in 16 or 8 bits), and the attention of one new token over it.

``run`` computes a case in plain torch operations, or with the framework's
kernels where ``own`` is true; ``exact`` gives the same outputs from the
definitions in 64 bits.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
E4M3_MAX = 448.0
DEVICE = "cuda"


# ------------------------------------------------------------------- cases
def listed():
    return [
        # one decode step of 16 requests: 32 query heads over 8 key heads, where the launch is what counts
        {"name": "rope step", "op": "rope", "dtype": "bf16", "tokens": 16, "q_heads": 32, "kv_heads": 8, "dim": 128,
         "rotary": 128, "interleaved": False, "far": 32768},
        # a long prompt's queries and keys, views of one fused projection
        {"name": "rope prompt", "op": "rope", "dtype": "bf16", "tokens": 8192, "q_heads": 32, "kv_heads": 8, "dim": 128,
         "rotary": 128, "interleaved": False, "far": 8192},
        # heads of 80 of which 32 dimensions turn in adjacent pairs, an uneven count of tokens and heads, far positions
        {"name": "rope partial", "op": "rope", "dtype": "fp16", "tokens": 1537, "q_heads": 25, "kv_heads": 5, "dim": 80,
         "rotary": 32, "interleaved": True, "far": 1000000},
        # a decode step's rows into a small 8-bit cache, and the cache read back
        {"name": "cache step", "op": "cache", "dtype": "bf16", "cache": "e4m3", "rows": 64, "pages": 64, "page": 16,
         "kv_heads": 8, "dim": 128},
        # a prompt's chunk quantised into the cache, then the context of all its chunks read back
        {"name": "cache prompt", "op": "cache", "dtype": "bf16", "cache": "int8", "rows": 8192, "pages": 1024, "page": 32,
         "kv_heads": 8, "dim": 128},
        # one request, alone, at an ordinary length
        {"name": "attend one", "op": "attend", "dtype": "bf16", "cache": "bf16", "batch": 1, "longest": 1000, "page": 16,
         "q_heads": 32, "kv_heads": 8, "dim": 128, "window": 0, "lse": False},
        # a full serving batch of uneven lengths, from none to 4096 tokens
        {"name": "attend batch", "op": "attend", "dtype": "bf16", "cache": "bf16", "batch": 64, "longest": 4096, "page": 16,
         "q_heads": 32, "kv_heads": 8, "dim": 128, "window": 0, "lse": False},
        # few requests over very long contexts in an 8-bit cache
        {"name": "attend long", "op": "attend", "dtype": "bf16", "cache": "e4m3", "batch": 4, "longest": 131072, "page": 64,
         "q_heads": 32, "kv_heads": 8, "dim": 128, "window": 0, "lse": True},
        # a head of its own for each query head, a sliding window, pages that no tile divides
        {"name": "attend window", "op": "attend", "dtype": "fp16", "cache": "int8", "batch": 17, "longest": 9001, "page": 24,
         "q_heads": 12, "kv_heads": 12, "dim": 64, "window": 1000, "lse": False},
        # a decode batch whose rows belong to 32 tenants in no order
        {"name": "adapters step", "op": "lora", "dtype": "bf16", "tokens": 64, "inner": 4096, "outer": 4096, "rank": 16,
         "adapters": 32, "runs": False, "none": 9},
        # prompts of 8 tenants, one after the other
        {"name": "adapters prompt", "op": "lora", "dtype": "bf16", "tokens": 8192, "inner": 4096, "outer": 4096, "rank": 64,
         "adapters": 8, "runs": True, "none": 0},
        # sizes that no tile divides
        {"name": "adapters odd", "op": "lora", "dtype": "fp16", "tokens": 333, "inner": 1001, "outer": 1503, "rank": 12,
         "adapters": 5, "runs": True, "none": 50},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["rope", "cache", "attend", "lora"])
    if op == "rope":
        dim = rng.choice([64, 72, 80, 96, 100, 128, 256])
        kv = rng.randint(1, 16)
        group = rng.randint(1, 8)
        tokens = min(_log(rng, 1, 8192), 60_000_000 // (kv * (group + 1) * dim))
        return {"op": op, "dtype": rng.choice(["bf16", "fp16", "fp32"]), "tokens": tokens, "q_heads": kv * group,
                "kv_heads": kv, "dim": dim, "rotary": rng.choice([dim, dim, dim // 2]),
                "interleaved": rng.random() < 0.4, "far": _log(rng, 100, 1000000)}
    if op == "cache":
        dim, kv = rng.choice([64, 80, 96, 128, 256]), rng.randint(1, 16)
        page = rng.choice([1, 16, 24, 32, 64])
        rows = min(_log(rng, 1, 8192), 60_000_000 // (kv * dim))
        pages = -(-rows // page) + _log(rng, 1, max(2, 24000 // page))
        return {"op": op, "dtype": rng.choice(["bf16", "fp16", "fp32"]), "cache": rng.choice(["e4m3", "int8", "same"]),
                "rows": rows, "pages": pages, "page": page, "kv_heads": kv, "dim": dim}
    if op == "attend":
        dim, kv = rng.choice([64, 80, 96, 128, 256]), rng.choice([1, 2, 3, 4, 8, 12])
        group = rng.choice([1, 2, 4, 5, 7, 8, 16])
        batch, longest = _log(rng, 1, 128), _log(rng, 1, 65536)
        longest = max(1, min(longest, 250_000_000 // (batch * kv * dim)))
        dtype = rng.choice(["bf16", "fp16"])
        return {"op": op, "dtype": dtype, "cache": rng.choice([dtype, "e4m3", "int8"]), "batch": batch, "longest": longest,
                "page": rng.choice([1, 16, 24, 32, 64]), "q_heads": kv * group, "kv_heads": kv, "dim": dim,
                "window": rng.choice([0, 0, _log(rng, 8, 8192)]), "lse": rng.random() < 0.5}
    tokens, rank = _log(rng, 1, 8192), rng.choice([4, 8, 12, 16, 24, 32, 64, 100])
    return {"op": op, "dtype": rng.choice(["bf16", "fp16", "fp32"]), "tokens": tokens, "inner": _log(rng, 200, 6000),
            "outer": _log(rng, 200, 6000), "rank": rank, "adapters": _log(rng, 1, 64), "runs": rng.random() < 0.5,
            "none": rng.choice([0, 0, tokens // 10, tokens])}


def _lengths(c):
    """Tokens that each request of an attention case has in the cache: spread evenly from none to the longest."""
    n, longest = c["batch"], c["longest"]
    return [longest] if n == 1 else [longest * i // (n - 1) for i in range(n)]


def _adapters(c):
    """Which adapter each row of a projection goes through; -1 for the first ``none`` rows of every run."""
    n, t = c["adapters"], c["tokens"]
    ids = [i * n // t if c["runs"] else (i * 7919 + i // 3) % n for i in range(t)]
    step = t // c["none"] if c["none"] else 0
    return [-1 if step and i % step == 0 else a for i, a in enumerate(ids)]


def _width(c, key="dtype"):
    return {"bf16": 2, "fp16": 2, "fp32": 4, "e4m3": 1, "int8": 1}[c["dtype"] if c[key] == "same" else c[key]]


def work(c):
    e = _width(c)
    if c["op"] == "rope":
        heads = c["q_heads"] + c["kv_heads"]
        n = c["tokens"] * heads * c["dim"]
        return {"bytes": 2 * n * e + 4 * c["tokens"] + 2 * c["dim"] * e + 4 * c["rotary"], "flops": 8 * n}
    if c["op"] == "cache":
        w = _width(c, "cache")
        scales = 4 if c["cache"] in ("e4m3", "int8") else 0
        slots = c["pages"] * c["page"]
        per_head = c["dim"] * (w + e) + scales
        return {"bytes": 2 * (c["rows"] + slots) * c["kv_heads"] * per_head + 8 * (c["rows"] + slots),
                "flops": 6 * (c["rows"] + slots) * c["kv_heads"] * c["dim"]}
    if c["op"] == "attend":
        seen = sum(min(n, c["window"]) if c["window"] else n for n in _lengths(c))
        per_head = 2 * (c["dim"] * _width(c, "cache") + (4 if c["cache"] in ("e4m3", "int8") else 0))
        rows = c["batch"] * c["q_heads"]
        return {"bytes": seen * c["kv_heads"] * per_head + 4 * (seen // c["page"]) + rows * (2 * c["dim"] * e + 4 * c["lse"]),
                "flops": 4 * seen * c["q_heads"] * c["dim"]}
    ids = _adapters(c)
    used, rows = len({a for a in ids if a >= 0}), sum(a >= 0 for a in ids)
    return {"bytes": e * (rows * c["inner"] + 2 * c["tokens"] * c["outer"] + used * c["rank"] * (c["inner"] + c["outer"])) + 4 * c["tokens"],
            "flops": 2 * rows * c["rank"] * (c["inner"] + c["outer"])}


# ------------------------------------------------------------------ inputs
def _quantise(x, kind):
    """Codes and scales, one for each row's head, of a cache kept in 8 bits.

    e4m3: the scale is the least power of two that brings the head's largest
    value to 448 or less, so dividing by it rounds nothing.  int8: the largest
    value over 127.  A head of zeros has a scale of 1."""
    x = x.float()
    top = x.abs().amax(-1)
    if kind == "e4m3":
        m, ex = torch.frexp(top)
        k = (ex - torch.where(m <= 0.875, 9, 8)).clamp(-120, 120).int()
        scale = torch.where(top > 0, ((k + 127) << 23).view(torch.float32), 1.0)
        return (x / scale[..., None]).to(torch.float8_e4m3fn), scale
    scale = torch.where(top > 0, (top * (1.0 / 127.0)).clamp_min(2.0 ** -120), 1.0)
    return (x / scale[..., None]).round().clamp(-127, 127).to(torch.int8), scale


def _pool(c, g):
    """A paged pool full of keys or values: [pages, page, heads, dim] and its scales."""
    x = torch.randn((c["pages"], c["page"], c["kv_heads"], c["dim"]), device=DEVICE, generator=g, dtype=torch.bfloat16)
    if c["cache"] in ("e4m3", "int8"):
        return _quantise(x, c["cache"])
    return x.to(DTYPES[c["dtype"]]), None


def prepare(c, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype = DTYPES[c["dtype"]]

    def randn(*shape, std=1.0):
        return (torch.randn(shape, device=DEVICE, generator=g) * std).to(dtype)

    if c["op"] == "rope":
        t, hq, hk, d = c["tokens"], c["q_heads"], c["kv_heads"], c["dim"]
        fused = randn(t, (hq + 2 * hk) * d, std=2.0)  # the projection's output: queries, keys, values side by side
        inv = 10000.0 ** (-torch.arange(0, c["rotary"], 2, device=DEVICE, dtype=torch.float64) / c["rotary"])
        return {"c": c, "q": fused[:, :hq * d].view(t, hq, d), "k": fused[:, hq * d:(hq + hk) * d].view(t, hk, d),
                "qw": (1 + 0.2 * torch.randn(d, device=DEVICE, generator=g)).to(dtype),
                "kw": (1 + 0.2 * torch.randn(d, device=DEVICE, generator=g)).to(dtype), "inv": inv.float(),
                "pos": torch.randint(0, c["far"], (t,), device=DEVICE, generator=g, dtype=torch.int32)}
    if c["op"] == "cache":
        (kc, ks), (vc, vs) = _pool(c, g), _pool(c, g)
        slots = torch.randperm(c["pages"] * c["page"], device=DEVICE, generator=g)
        sizes = (0.05 + 4 * torch.rand((c["rows"], c["kv_heads"], 1), device=DEVICE, generator=g))
        k = (torch.randn((c["rows"], c["kv_heads"], c["dim"]), device=DEVICE, generator=g) * sizes).to(dtype)
        pages = torch.randperm(c["pages"], device=DEVICE, generator=g)  # the context's pages, in no order
        order = (pages[:, None] * c["page"] + torch.arange(c["page"], device=DEVICE)).reshape(-1)
        return {"c": c, "kc": kc, "vc": vc, "ks": ks, "vs": vs, "k": k, "v": randn(*k.shape), "slots": slots[:c["rows"]],
                "order": order}
    if c["op"] == "attend":
        lens = _lengths(c)
        need = [-(-n // c["page"]) for n in lens]
        width = max(1, max(need))
        pages = max(1, sum(need))
        (kc, ks), (vc, vs) = _pool({**c, "pages": pages}, g), _pool({**c, "pages": pages}, g)
        # each request's pages lie anywhere in the pool; what its row of the table does not use is -1
        first = torch.tensor([sum(need[:i]) for i in range(len(need))], device=DEVICE)
        at = torch.arange(width, device=DEVICE)
        perm = torch.randperm(pages, device=DEVICE, generator=g)
        table = torch.where(at < torch.tensor(need, device=DEVICE)[:, None], perm[(first[:, None] + at).clamp_max(pages - 1)], -1)
        sharp = 0.5 + 2.5 * torch.rand((1, c["q_heads"], 1), device=DEVICE, generator=g)  # heads that look at few tokens and at many
        q = (torch.randn((c["batch"], c["q_heads"], c["dim"]), device=DEVICE, generator=g) * sharp).to(dtype)
        return {"c": c, "q": q, "kc": kc, "vc": vc, "ks": ks, "vs": vs, "table": table.int(),
                "lens": torch.tensor(lens, device=DEVICE, dtype=torch.int32)}
    n, r, ki, mo = c["adapters"], c["rank"], c["inner"], c["outer"]
    return {"c": c, "x": randn(c["tokens"], ki), "y": randn(c["tokens"], mo),
            "a": randn(n, r, ki, std=ki ** -0.5), "b": randn(n, mo, r, std=r ** -0.5),
            "ids": torch.tensor(_adapters(c), device=DEVICE, dtype=torch.int32),
            "scales": 0.5 + torch.rand(n, device=DEVICE, generator=g)}


# -------------------------------------------------------------- plain forms
def _rotated(x, w, cos, sin, c):
    x = x.float()
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w.float()
    r, h = c["rotary"], c["rotary"] // 2
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if c["interleaved"] else (x[..., :h], x[..., h:r])
    p, s = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack((p, s), -1).flatten(-2) if c["interleaved"] else torch.cat((p, s), -1)
    return torch.cat((turned, x[..., r:]), -1).to(DTYPES[c["dtype"]])


def _rope(s):
    c = s["c"]
    if own:
        from seldon_core_amd import ops

        return ops.qk_norm_rope(s["q"], s["k"], s["qw"], s["kw"], s["pos"], s["inv"], eps=1e-6, interleaved=c["interleaved"])
    angle = s["pos"].double()[:, None] * s["inv"].double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    return _rotated(s["q"], s["qw"], cos, sin, c), _rotated(s["k"], s["kw"], cos, sin, c)


def _write(cache, scales, x, slots, kind):
    flat = cache.view(-1, *cache.shape[2:])
    if scales is None:
        flat[slots] = x
        return
    codes, scale = _quantise(x, kind)
    flat.view(torch.uint8)[slots] = codes.view(torch.uint8)
    scales.view(-1, scales.shape[2])[slots] = scale


def _values(cache, scales, slots):
    """fp32 values that the cache's rows stand for."""
    flat = cache.view(-1, *cache.shape[2:])
    if scales is None:
        return flat[slots].float()
    codes = flat.view(torch.uint8)[slots].view(cache.dtype)
    return codes.float() * scales.view(-1, scales.shape[2])[slots][..., None]


def _cache(s):
    c = s["c"]
    if own:
        from seldon_core_amd import ops

        cache = ops.KVCache(s["kc"], s["vc"], s["ks"], s["vs"])
        ops.kv_cache_write(cache, s["k"], s["v"], s["slots"])
        return ops.kv_cache_read(cache, s["order"], dtype=DTYPES[c["dtype"]])
    _write(s["kc"], s["ks"], s["k"], s["slots"], c["cache"])
    _write(s["vc"], s["vs"], s["v"], s["slots"], c["cache"])
    return tuple(_values(*x, s["order"]).to(DTYPES[c["dtype"]]) for x in ((s["kc"], s["ks"]), (s["vc"], s["vs"])))


def _attend(s):
    c = s["c"]
    if own:
        from seldon_core_amd import ops

        cache = ops.KVCache(s["kc"], s["vc"], s["ks"], s["vs"])
        return ops.paged_attention(s["q"], cache, s["table"], s["lens"], window=c["window"], return_lse=c["lse"])
    span = min(c["longest"], c["window"] or c["longest"])  # the last tokens of each request, which are all that it sees
    t = s["lens"].long()[:, None] - span + torch.arange(span, device=s["q"].device)
    seen = t >= 0
    t = torch.where(seen, t, 0)
    slots = torch.where(seen, s["table"].long().gather(1, t // c["page"]) * c["page"] + t % c["page"], 0)
    mask = seen[:, :, None, None]
    k = torch.where(mask, _values(s["kc"], s["ks"], slots), 0.0).permute(0, 2, 1, 3)  # [batch, kv heads, tokens, dim]
    v = torch.where(mask, _values(s["vc"], s["vs"], slots), 0.0).permute(0, 2, 3, 1)
    q = s["q"].float().view(c["batch"], c["kv_heads"], -1, c["dim"]).transpose(2, 3) * c["dim"] ** -0.5
    scores = torch.where(seen[:, None, :, None], k @ q, -math.inf)  # [batch, kv heads, tokens, group]
    top = scores.amax(2, keepdim=True)
    p = torch.exp(scores - torch.where(top > -math.inf, top, 0.0))
    total = p.sum(2, keepdim=True)
    out = (v @ (p / torch.where(total > 0, total, 1.0))).transpose(2, 3)  # a request without tokens gets zeros
    out = out.reshape(s["q"].shape).to(s["q"].dtype)
    lse = (top + torch.log(total)).reshape(c["batch"], c["q_heads"])
    return (out, lse) if c["lse"] else out


def _lora(s):
    if own:
        from seldon_core_amd import ops

        return ops.lora_add(s["y"], s["x"], s["a"], s["b"], s["ids"], s["scales"])
    n, r, ki = s["a"].shape
    mine = (s["ids"][:, None] == torch.arange(n, device=s["ids"].device))  # [rows, adapters]
    h = (s["x"].float() @ s["a"].float().view(n * r, ki).T).view(-1, n, r) * s["scales"][:, None]
    h = torch.where(mine[:, :, None], h, 0.0)
    return (s["y"].float() + h.view(-1, n * r) @ s["b"].float().permute(0, 2, 1).reshape(n * r, -1)).to(s["y"].dtype)


def run(s):
    return {"rope": _rope, "cache": _cache, "attend": _attend, "lora": _lora}[s["c"]["op"]](s)


# -------------------------------------------------------------------- exact
def _exact_rope(s, c):
    half = c["rotary"] // 2
    turn = torch.outer(s["pos"].double(), s["inv"].double())
    z = torch.complex(turn.cos(), turn.sin()).unsqueeze(1)
    got = []
    for x, w in ((s["q"], s["qw"]), (s["k"], s["kw"])):
        y = x.double()
        y = y / (y.pow(2).sum(-1, keepdim=True) / c["dim"] + 1e-6).sqrt() * w.double()
        even = torch.arange(0, c["rotary"], 2, device=y.device) if c["interleaved"] else torch.arange(half, device=y.device)
        odd = even + 1 if c["interleaved"] else even + half
        pairs = torch.complex(y[..., even], y[..., odd]) * z
        y[..., even], y[..., odd] = pairs.real.clone(), pairs.imag.clone()
        got.append(y)
    return tuple(got)


def _exact_code(x, kind):
    """What x stands for after a round trip through 8 bits, in 64."""
    x = x.double()
    top = x.abs().amax(-1, keepdim=True)
    if kind == "int8":
        step = (top.float() * (1.0 / 127.0)).double()  # the scale is kept in 32 bits
        return torch.where(top > 0, (x / step).round() * step, 0.0)
    scale = torch.exp2(torch.ceil(torch.log2(top / E4M3_MAX)))
    y = torch.where(top > 0, x / scale, 0.0)
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)  # 3 bits behind the leading one, least exponent -6
    return torch.where(top > 0, torch.round(y / step) * step * scale, 0.0)


def _exact_cache(s, c):
    got = []
    for codes, scales, x in ((s["kc"], s["ks"], s["k"]), (s["vc"], s["vs"], s["v"])):
        now = codes.double() if scales is None else codes.float().double() * scales.double().unsqueeze(-1)
        now = now.reshape(-1, c["kv_heads"], c["dim"])
        now[s["slots"]] = x.double() if scales is None else _exact_code(x, c["cache"])
        got.append(now[s["order"]])
    return tuple(got)


def _exact_attend(s, c):
    group = c["q_heads"] // c["kv_heads"]
    out = torch.zeros(s["q"].shape, device=DEVICE, dtype=torch.float64)
    lse = torch.full((c["batch"], c["q_heads"]), -math.inf, device=DEVICE, dtype=torch.float64)
    for i, n in enumerate(s["lens"].tolist()):
        low = max(0, n - c["window"]) if c["window"] else 0
        if n == 0:
            continue
        pages = s["table"][i, low // c["page"]:-(-n // c["page"])].long()
        rows = slice(low % c["page"], low % c["page"] + n - low)
        k, v = ((x[pages].double() if y is None else x.view(torch.uint8)[pages].view(x.dtype).float().double() * y[pages].double()[..., None])
                .flatten(0, 1)[rows] for x, y in ((s["kc"], s["ks"]), (s["vc"], s["vs"])))
        for h in range(c["kv_heads"]):
            q = s["q"][i, h * group:(h + 1) * group].double() / math.sqrt(c["dim"])
            logits = q @ k[:, h].T.contiguous()
            lse[i, h * group:(h + 1) * group] = torch.logsumexp(logits, -1)
            out[i, h * group:(h + 1) * group] = torch.softmax(logits, -1) @ v[:, h].contiguous()
    return (out, lse) if c["lse"] else out


def _exact_lora(s, c):
    out = s["y"].double()
    for a in range(c["adapters"]):
        rows = (s["ids"] == a).nonzero()[:, 0]
        down = s["x"][rows].double() @ s["a"][a].double().T.contiguous()
        out[rows] += s["scales"][a].double() * (down @ s["b"][a].double().T.contiguous())
    return out


def exact(c, seed):
    s = prepare(c, seed)
    return {"rope": _exact_rope, "cache": _exact_cache, "attend": _exact_attend, "lora": _exact_lora}[c["op"]](s, c)
