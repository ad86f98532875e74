"""The operators of a paged 4-bit key/value cache, as measured: what a serving step does between its fused QKV
projection and its output projection.

* plan    -- block tables and slot maps of a step, built on the GPU from the requests' lengths
* rotary  -- rotary positions with several axes (time, height, width) on queries and keys
* append  -- queries and keys rotated, keys and values quantized to 4 bits (MLX affine, groups of 64) and stored in their
             slots; the stored values are read back, so that the pass answers with what the cache now holds
* attend  -- attention of one or more queries a request over its pages

`own` is false for the plain form (elementary torch operations in 32 bits, rounded once at the end) and true for the
calls a user makes of locals_b200.
"""

import math

import torch

own = False

GROUP = 64
_TYPE = {"bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # a decode step's bookkeeping: every running request gets one token, now and then a new page
        {"name": "plan decode", "op": "plan", "requests": 64, "page": 16, "cached": 32768, "new": 1},
        # admission of a batch of prompts, some of them continuing a cached prefix
        {"name": "plan prompts", "op": "plan", "requests": 200, "page": 16, "cached": 4096, "new": 512},
        # one text token of a model with (time, height, width) positions: pure latency
        {"name": "rotary token", "op": "rotary", "tokens": 1, "heads": 32, "kv_heads": 8, "dim": 128, "rot": 128,
         "axes": 3, "pairs": "halves", "dtype": "bf16"},
        # the patches of a few images in a vision tower: two axes, head dimension 80
        {"name": "rotary patches", "op": "rotary", "tokens": 16383, "heads": 16, "kv_heads": 16, "dim": 80, "rot": 80,
         "axes": 2, "pairs": "halves", "dtype": "f16"},
        # the cache write of a decode step
        {"name": "append decode", "op": "append", "tokens": 64, "heads": 32, "kv_heads": 4, "dim": 128, "rot": 128,
         "axes": 1, "pairs": "halves", "page": 16, "dtype": "bf16"},
        # the cache write of a prompt of text and images
        {"name": "append prompt", "op": "append", "tokens": 8191, "heads": 32, "kv_heads": 8, "dim": 128, "rot": 128,
         "axes": 3, "pairs": "halves", "page": 16, "dtype": "bf16"},
        # one user, one token, a short context: latency
        {"name": "attend one user", "op": "attend", "requests": 1, "cached": 1000, "new": 1, "ragged": False,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "window": 0, "sinks": False, "dtype": "bf16"},
        # a decode step of a full batch, requests of all ages, with sinks
        {"name": "attend decode batch", "op": "attend", "requests": 64, "cached": 8190, "new": 1, "ragged": True,
         "heads": 32, "kv_heads": 4, "dim": 128, "page": 16, "window": 0, "sinks": True, "dtype": "bf16"},
        # a few requests with very long contexts
        {"name": "attend long contexts", "op": "attend", "requests": 4, "cached": 131071, "new": 1, "ragged": False,
         "heads": 32, "kv_heads": 4, "dim": 128, "page": 64, "window": 0, "sinks": False, "dtype": "f16"},
        # the check of five drafted tokens a request
        {"name": "attend drafts", "op": "attend", "requests": 16, "cached": 4003, "new": 5, "ragged": True,
         "heads": 16, "kv_heads": 2, "dim": 256, "page": 32, "window": 0, "sinks": False, "dtype": "bf16"},
        # prompts and decoding requests in one batch
        {"name": "attend mixed batch", "op": "attend", "requests": 8, "cached": 2048, "new": 1024, "ragged": True,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "window": 0, "sinks": False, "dtype": "bf16"},
        # one piece of a long prompt against what is cached of it
        {"name": "attend prompt piece", "op": "attend", "requests": 1, "cached": 28672, "new": 4096, "ragged": False,
         "heads": 16, "kv_heads": 2, "dim": 128, "page": 16, "window": 0, "sinks": False, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["plan", "rotary", "append", "attend", "attend", "attend"])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    page = rng.choice([8, 16, 16, 32, 48, 64, 128])
    if op == "plan":
        return {"op": op, "requests": _log(rng, 1, 200), "page": page, "cached": _log(rng, 1, 32768),
                "new": rng.choice([1, 1, _log(rng, 2, 512)])}
    if op == "rotary":
        dim = rng.choice([64, 72, 80, 96, 128, 256])
        tokens, kv = _log(rng, 1, 8191), rng.choice([1, 2, 4, 8])
        return {"op": op, "tokens": tokens, "heads": kv * rng.choice([1, 2, 4]), "kv_heads": kv, "dim": dim,
                "rot": rng.choice([dim, dim, dim // 16 * 8]), "axes": rng.randint(1, 3),
                "pairs": rng.choice(["halves", "halves", "neighbours"]), "dtype": dtype}
    kv = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 3, 4, 5, 8, 16])
    dim = rng.choice([64, 128, 128, 128, 256])
    if op == "append":
        return {"op": op, "tokens": _log(rng, 1, 4096), "heads": kv * min(group, 8), "kv_heads": kv, "dim": dim,
                "rot": rng.choice([dim, dim, dim // 2, dim // 4]), "axes": rng.randint(1, 3),
                "pairs": rng.choice(["halves", "halves", "neighbours"]), "page": page, "dtype": dtype}
    # the score matrix of the plain form (requests x heads x new x keys) and the keys stay below the largest listed
    new = rng.choice([1, 1, 1, _log(rng, 2, 16), _log(rng, 17, 2048)])
    cached = _log(rng, 1, 65536)
    keys = cached + new
    most = min(64, (1 << 30) // (kv * group * new * keys), (1 << 27) // (kv * dim * keys))
    while most < 1:
        cached = max(1, cached // 2)
        keys = cached + new
        most = min(64, (1 << 30) // (kv * group * new * keys), (1 << 27) // (kv * dim * keys))
    return {"op": op, "requests": _log(rng, 1, most), "cached": cached, "new": new, "ragged": rng.random() < 0.7,
            "heads": kv * group, "kv_heads": kv, "dim": dim, "page": page,
            "window": rng.choice([0, 0, 0, 1 + rng.randrange(keys)]), "sinks": rng.random() < 0.4, "dtype": dtype}


# ---- inputs --------------------------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _ints(g, lo, hi, shape):
    return torch.randint(lo, hi + 1, shape, generator=g, device="cuda", dtype=torch.int32)


def _normal(g, shape, dtype):
    """Normal values, a few channels of which are several times as large, as keys have them."""
    x = torch.randn(shape, generator=g, device="cuda")
    big = 1 + 4 * (torch.rand(shape[-1], generator=g, device="cuda") < 0.04)
    return (x * big).to(dtype)


def _lengths(case, g):
    """Cached and new tokens a request. Ragged: of all ages (one of them the oldest), the new tokens spread over half
    to all of `new`, and of prompts every other request only decodes; in any order, but as many tokens in all."""
    B, cached, new = case["requests"], case["cached"], case["new"]
    if case.get("ragged", True):
        c = _ints(g, 0, cached, (B,))
        c[int(torch.randint(0, B, (1,), generator=g, device="cuda"))] = cached
        n = torch.linspace(new, max(1, new // 2), B, device="cuda", dtype=torch.float64).to(torch.int32)
        if new > 16:
            n[1::2] = 1
        n = n[torch.randperm(B, generator=g, device="cuda")]
    else:
        c, n = _ints(g, cached, cached, (B,)), _ints(g, new, new, (B,))
    return c, n


def _tables(rot, positions, dtype=torch.float64):
    """cos and sin of a position's angles, in 32 bits as servers keep them."""
    inv = 10000.0 ** (-torch.arange(0, rot, 2, device="cuda", dtype=dtype) / rot)
    a = torch.arange(positions, device="cuda", dtype=dtype)[:, None] * inv
    return a.cos().float(), a.sin().float()


def _axes(case):
    half, n = case["rot"] // 2, case["axes"]
    return (torch.arange(half, device="cuda") * n // half).to(torch.int32) if n > 1 else None


def _pool(case, pages, g):
    """Keys and values of a cache in use: normal values quantized to 4 bits."""
    dt, D = _TYPE[case["dtype"]], case["dim"]
    out = []
    for _ in range(2):
        x = _normal(g, (pages, case["kv_heads"], case["page"], D), torch.float32)
        q, s, b = _quantize(x)
        out.append((_pack(q), s.to(dt), b.to(dt)))
        del x, q, s, b
    return out


def prepare(case, seed):
    g, op = _gen(seed), case["op"]
    if op == "plan":
        cached, new = _lengths({**case, "ragged": True}, g)
        page = case["page"]
        have = (cached + page - 1) // page
        width = (case["cached"] + case["new"] + page - 1) // page + 1
        total = case["requests"] * width
        ids = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
        table = ids.view(case["requests"], width).clone()
        used = torch.arange(width, device="cuda")[None] < have[:, None]
        free = table[~used].contiguous()
        table[~used] = -1
        return {"case": case, "cached": cached, "new": new, "table": table, "free": free,
                "head": torch.zeros(1, dtype=torch.int32, device="cuda"), "tokens": int(new.sum())}
    dt, D = _TYPE[case["dtype"]], case["dim"]
    if op in ("rotary", "append"):
        N, far = case["tokens"], 4096
        cos, sin = _tables(case["rot"], far)
        s = {"case": case, "cos": cos, "sin": sin, "axes": _axes(case),
             "positions": _ints(g, 0, far - 1, (case["axes"], N)),
             "q": _normal(g, (N, case["heads"], D), dt), "k": _normal(g, (N, case["kv_heads"], D), dt)}
        if op == "append":
            pages = 2 * ((N + case["page"] - 1) // case["page"]) + 3
            s["v"] = _normal(g, (N, case["kv_heads"], D), dt)
            s["keys"], s["values"] = _pool(case, pages, g)
            s["slots"] = torch.randperm(pages * case["page"], generator=g, device="cuda")[:N].to(torch.int32)
        return s
    cached, new = _lengths(case, g)
    lens, page = cached + new, case["page"]
    width = (case["cached"] + case["new"] + page - 1) // page
    pages = case["requests"] * width
    keys, values = _pool(case, pages, g)
    table = torch.randperm(pages, generator=g, device="cuda").to(torch.int32).view(case["requests"], width)
    used = torch.arange(width, device="cuda")[None] < ((lens + page - 1) // page)[:, None]
    table = torch.where(used, table, -1).to(torch.int32).contiguous()
    start = torch.zeros(case["requests"] + 1, dtype=torch.int32, device="cuda")
    start[1:] = torch.cumsum(new, 0)
    N = int(start[-1])
    q = (1.5 * torch.randn((N, case["heads"], D), generator=g, device="cuda")).to(dt)
    sinks = 2 * torch.randn(case["heads"], generator=g, device="cuda") if case["sinks"] else None
    return {"case": case, "q": q, "keys": keys, "values": values, "table": table, "lens": lens.to(torch.int32),
            "start": start, "max_q": case["new"], "scale": D ** -0.5, "sinks": sinks}


# ---- one pass ------------------------------------------------------------------------------------

def run(state):
    return (_own if own else _plain)[state["case"]["op"]](state)


def _own_plan(s):
    from locals_b200 import paged

    p = paged.plan(s["cached"], s["new"], s["table"], s["free"], s["head"], s["case"]["page"], s["tokens"])
    return {"table": s["table"], "lens": p.lens, "start": p.q_start, "positions": p.positions, "slots": p.slots,
            "head": p.head}


def _own_rotary(s):
    from locals_b200 import rotary

    return rotary.rotate(s["q"], s["k"], s["positions"], s["cos"], s["sin"], s["axes"],
                         interleaved=s["case"]["pairs"] == "neighbours")


def _own_append(s):
    from locals_b200 import paged

    q = paged.append(s["q"], s["k"], s["v"], s["slots"], s["keys"], s["values"], s["positions"], s["cos"], s["sin"],
                     s["axes"], interleaved=s["case"]["pairs"] == "neighbours")
    return (q, *paged.read(s["keys"], s["values"], s["slots"]))


def _own_attend(s):
    from locals_b200 import paged

    return paged.attend(s["q"], s["keys"], s["values"], s["table"], s["lens"], s["scale"], q_start=s["start"],
                        max_q=s["max_q"], sinks=s["sinks"], window=s["case"]["window"])


_own = {"plan": _own_plan, "rotary": _own_rotary, "append": _own_append, "attend": _own_attend}


def _plain_plan(s):
    cached, new, table, free, page = s["cached"], s["new"], s["table"], s["free"], s["case"]["page"]
    lens = cached + new
    start = torch.zeros(len(new) + 1, dtype=torch.int32, device=new.device)
    start[1:] = torch.cumsum(new, 0)
    have, want = (cached + page - 1) // page, (lens + page - 1) // page
    need = want - have
    after = torch.cumsum(need, 0)
    column = torch.arange(table.shape[1], device=new.device)[None]
    fresh = (column >= have[:, None]) & (column < want[:, None])
    at = s["head"] + (after - need - have)[:, None] + column
    table.copy_(torch.where(fresh, free[at.clamp(0, len(free) - 1)], table))
    token = torch.arange(s["tokens"], device=new.device, dtype=torch.int32)
    row = torch.searchsorted(start[1:], token, right=True)
    positions = (cached[row] + token - start[row]).to(torch.int32)
    slots = (table[row, positions // page] * page + positions % page).to(torch.int32)
    return {"table": table, "lens": lens, "start": start, "positions": positions, "slots": slots,
            "head": (s["head"] + after[-1:]).to(torch.int32)}


def _rotate(x, s):
    """x (tokens, heads, dim) in 32 bits, its first `rot` dimensions rotated by the tables' rows of its positions."""
    case = s["case"]
    rot, half = case["rot"], case["rot"] // 2
    pair = torch.arange(half, device=x.device)
    at = s["positions"][s["axes"].long() if s["axes"] is not None else torch.zeros_like(pair)].T.long()  # (tokens, half)
    c, n = s["cos"][at, pair][:, None], s["sin"][at, pair][:, None]
    if case["pairs"] == "halves":
        a, b = x[..., :half], x[..., half:rot]
        return torch.cat([a * c - b * n, b * c + a * n, x[..., rot:]], -1)
    a, b = x[..., 0:rot:2], x[..., 1:rot:2]
    return torch.cat([torch.stack([a * c - b * n, b * c + a * n], -1).flatten(-2), x[..., rot:]], -1)


def _plain_rotary(s):
    dt = s["q"].dtype
    return _rotate(s["q"].float(), s).to(dt), _rotate(s["k"].float(), s).to(dt)


def _quantize(x):
    """Codes 0..15 and a scale and bias a group of 64: the larger edge of the group is met exactly, and the scale points
    away from it."""
    g = x.unflatten(-1, (-1, GROUP))
    lo, hi = g.amin(-1), g.amax(-1)
    neg = lo.abs() > hi.abs()
    fifteen = torch.full((), 15.0, device=x.device, dtype=x.dtype)
    scale = ((hi - lo) / fifteen.expand_as(hi)).clamp_min(1e-7)
    scale = torch.where(neg, scale, -scale)
    edge = torch.where(neg, lo, hi)
    q0 = torch.round(edge / scale)
    scale = torch.where(q0 != 0, edge / torch.where(q0 != 0, q0, torch.ones_like(q0)), scale)
    bias = torch.where(q0 != 0, edge, torch.zeros_like(edge))
    codes = torch.round((g - bias[..., None]) / scale[..., None]).clamp(0, 15)
    return codes.to(torch.int32).flatten(-2), scale, bias


def _pack(codes):
    w = codes.unflatten(-1, (-1, 8)) << (4 * torch.arange(8, device=codes.device, dtype=torch.int32))
    a = w[..., 0:4] | w[..., 4:8]
    a = a[..., 0:2] | a[..., 2:4]
    return (a[..., 0] | a[..., 1]).contiguous()


def _unpack(words, scales, biases):
    shift = 4 * torch.arange(8, device=words.device, dtype=torch.int32)
    q = ((words[..., None] >> shift) & 15).float().flatten(-2).unflatten(-1, (-1, GROUP))
    return (q * scales.float()[..., None] + biases.float()[..., None]).flatten(-2)


def _plain_append(s):
    dt, page = s["q"].dtype, s["case"]["page"]
    q = _rotate(s["q"].float(), s).to(dt)
    at = (s["slots"] // page).long(), (s["slots"] % page).long()
    for x, (words, scales, biases) in ((_rotate(s["k"].float(), s), s["keys"]), (s["v"].float(), s["values"])):
        codes, scale, bias = _quantize(x)
        words[at[0], :, at[1]] = _pack(codes)
        scales[at[0], :, at[1]] = scale.to(dt)
        biases[at[0], :, at[1]] = bias.to(dt)
    return (q, *(_unpack(*(a[at[0], :, at[1]] for a in t)).to(dt) for t in (s["keys"], s["values"])))


def _plain_attend(s):
    q, table, lens, start, case = s["q"], s["table"].long(), s["lens"], s["start"].long(), s["case"]
    N, H, D = q.shape
    B, KVH = len(lens), case["kv_heads"]
    G, dev = H // KVH, q.device
    k, v = (_unpack(*(a[table.clamp_min(0)].transpose(1, 2).flatten(2, 3) for a in t)) for t in (s["keys"], s["values"]))
    L = k.shape[2]  # (requests, kv heads, keys, dim)
    new = start[1:] - start[:-1]
    i = torch.arange(s["max_q"], device=dev)[None]
    token = (start[:-1, None] + i).clamp_max(N - 1)  # (requests, queries)
    x = q[token].float().view(B, -1, KVH, G, D).transpose(1, 2).flatten(2, 3) * s["scale"]
    score = (x @ k.transpose(-1, -2)).view(B, KVH, -1, G, L)
    at = (lens[:, None] - new[:, None] + i)[:, None, :, None, None]  # the query's own position
    key = torch.arange(L, device=dev)
    seen = (key <= at) & (i < new[:, None])[:, None, :, None, None]
    if case["window"]:
        seen &= key > at - case["window"]
    score.masked_fill_(~seen, -math.inf)
    top = score.amax(-1, keepdim=True)
    if s["sinks"] is not None:
        sink = s["sinks"].view(1, KVH, 1, G, 1)
        top = torch.maximum(top, sink)
    top = torch.where(top == -math.inf, 0.0, top)
    score.sub_(top).exp_()
    total = score.sum(-1, keepdim=True)
    if s["sinks"] is not None:
        total = total + (sink - top).exp()
    out = (score.flatten(2, 3) @ v).view(B, KVH, -1, G, D) / torch.where(total > 0, total, 1.0)
    out = out.permute(0, 2, 1, 3, 4).reshape(B, -1, H, D).to(q.dtype)
    return out[i.expand(B, -1) < new[:, None]]


_plain = {"plan": _plain_plan, "rotary": _plain_rotary, "append": _plain_append, "attend": _plain_attend}


# ---- what a pass cannot do without ----------------------------------------------------------------

def work(case):
    op = case["op"]
    if op == "plan":
        B, page = case["requests"], case["page"]
        new = case["new"] if case["new"] == 1 else 0.75 * case["new"] if case["new"] <= 16 else 0.375 * case["new"] + 0.5
        # lengths in and out, a position and a slot a token, and a page taken from the free list and entered for each
        # page of new tokens (the last page of a cached prefix is half full on average)
        return {"bytes": B * 4 * 4 + B * new * 8 + B * new / page * 8, "flops": B * new * 4}
    D, kv, H = case["dim"], case["kv_heads"], case["heads"]
    held = kv * (D // 2 + D // GROUP * 4)  # a token's keys (or values) in 4 bits, with scales and biases
    if op in ("rotary", "append"):
        N, rot, axes = case["tokens"], case["rot"], case["axes"]
        tables = min(N, 4096) * rot * 4 + N * axes * 4
        if op == "rotary":
            return {"bytes": N * (H + kv) * D * 4 + tables, "flops": N * (H + kv) * rot * 3}
        return {"bytes": N * (H * D * 4 + kv * D * 4 + 4 * held + 2 * kv * D * 2 + 8) + tables,
                "flops": N * ((H + kv) * rot * 3 + 2 * kv * D * 8)}
    # attend: the keys that some query sees, read once; each query's scores and sums
    B, c, n, w = case["requests"], case["cached"], case["new"], case["window"]
    some = [(c, n)] * B
    if case["ragged"]:
        some = [(c, n)] + [(c / 2, 1 if n > 16 and i % 2 else max(1, 0.75 * n)) for i in range(1, B)]
    keys = pairs = tokens = 0
    for cached, new in some:
        seen = cached + (new + 1) / 2
        keys += min(cached + new, w + new - 1) if w else cached + new
        pairs += new * (min(seen, w) if w else seen)
        tokens += new
    return {"bytes": keys * 2 * held + tokens * H * D * 4 + B * 8 + keys / case["page"] * 4, "flops": pairs * H * D * 4}


# ---- the definitions in 64 bits -------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"plan": _exact_plan, "rotary": _exact_rotary, "append": _exact_append, "attend": _exact_attend}[case["op"]](s)


def _exact_plan(s):
    return None  # whole numbers: held to equality


def _turned(x, s):
    """Each pair (a, b) of dimensions as a complex number a + ib, times cos + i sin."""
    case, half = s["case"], s["case"]["rot"] // 2
    y = x.double()
    for j in range(half):
        u, w = (j, j + half) if case["pairs"] == "halves" else (2 * j, 2 * j + 1)
        p = s["positions"][int(s["axes"][j]) if s["axes"] is not None else 0].long()
        z = torch.complex(s["cos"][p, j].double(), s["sin"][p, j].double())[:, None]
        z = torch.complex(x[..., u].double(), x[..., w].double()) * z
        y[..., u], y[..., w] = z.real, z.imag
    return y


def _exact_rotary(s):
    return _turned(s["q"], s), _turned(s["k"], s)


def _stands_for(x, dt):
    """What 4 bits a value, with a scale and bias in dt, make of x."""
    y = torch.empty_like(x)
    for g in range(x.shape[-1] // GROUP):
        v = x[..., g * GROUP:(g + 1) * GROUP]
        lo, hi = v.min(-1, keepdim=True).values, v.max(-1, keepdim=True).values
        edge = torch.where(-lo > hi.abs(), lo, torch.where(lo.abs() > hi.abs(), lo, hi))
        step = ((hi - lo) / 15).clamp(min=1e-7) * torch.where(lo.abs() > hi.abs(), 1.0, -1.0)
        n = (edge / step).round()
        some = n != 0
        step = torch.where(some, edge / n.where(some, torch.ones_like(n)), step)
        bias = edge * some
        code = ((v - bias) / step).round().clamp(0, 15)
        y[..., g * GROUP:(g + 1) * GROUP] = code * step.to(dt).double() + bias.to(dt).double()
    return y


def _exact_append(s):
    dt = s["q"].dtype
    return _turned(s["q"], s), _stands_for(_turned(s["k"], s), dt), _stands_for(s["v"].double(), dt)


def _exact_attend(s):
    q, case, page = s["q"], s["case"], s["case"]["page"]
    H, D, KVH = case["heads"], case["dim"], case["kv_heads"]
    G = H // KVH
    lens, start = s["lens"].tolist(), s["start"].tolist()
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    for b, n in enumerate(lens):
        ids = s["table"][b, :(n + page - 1) // page].long()
        first, new = start[b], start[b + 1] - start[b]
        for h in range(KVH):
            kv = []
            for words, scales, biases in (s["keys"], s["values"]):
                w = words[ids, h].reshape(-1, D // 8)[:n]
                x = torch.empty((n, D), dtype=torch.float64, device=q.device)
                for j in range(8):
                    x[:, j::8] = ((w >> (4 * j)) & 15).double()
                for g in range(D // GROUP):
                    at = slice(g * GROUP, (g + 1) * GROUP)
                    x[:, at] *= scales[ids, h].reshape(-1, D // GROUP)[:n, g:g + 1].double()
                    x[:, at] += biases[ids, h].reshape(-1, D // GROUP)[:n, g:g + 1].double()
                kv.append(x)
            for i in range(0, new, 1024):
                m = min(1024, new - i)
                x = q[first + i:first + i + m, h * G:(h + 1) * G].double()
                p = torch.einsum("mgd,nd->gmn", x, kv[0]) * s["scale"]
                at = (n - new + i + torch.arange(m, device=q.device))[:, None]
                key = torch.arange(n, device=q.device)[None]
                hidden = key > at
                if case["window"]:
                    hidden |= key <= at - case["window"]
                p[:, hidden] = -math.inf
                if s["sinks"] is not None:
                    sink = s["sinks"][h * G:(h + 1) * G].double()[:, None, None].expand(-1, m, 1)
                    p = torch.softmax(torch.cat([p, sink], -1), -1)[..., :n]
                else:
                    p = torch.softmax(p, -1)
                out[first + i:first + i + m, h * G:(h + 1) * G] = torch.einsum("gmn,nd->mgd", p, kv[1])
    return out
