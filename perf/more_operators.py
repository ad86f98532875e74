"""The operators of microscaled 4-bit floating point, as measured: values of 4 bits (sign, two bits of exponent, one of
mantissa: 0, 0.5, 1, 1.5, 2, 3, 4, 6) in groups along the input dimension that share a scale of 8 bits.

* quantize -- a matrix to 4 bits: "mxfp4", groups of 32 with a power of two each, or "nvfp4", groups of 16 with a scale of
              8-bit floating point (e4m3) each and, when "scaled", one 32-bit factor for the whole matrix; the stored
              values are read back, so that the pass answers with what they stand for
* product  -- x . w^T with both in 4 bits
* linear   -- x . w^T with x in 16 bits and w in mxfp4
* experts  -- a routed mixture of SwiGLU experts in mxfp4 on 16-bit tokens, with the tokens' weighted sum

`own` is false for the plain form (elementary torch operations in 32 bits, rounded once at the end) and true for the
calls a user makes of locals_b200.
"""

import math

import torch

own = False

_TYPE = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_GROUP = {"mxfp4": 32, "nvfp4": 16}


def listed():
    return [
        # one token's hidden state on its way into a 4-bit product: latency
        {"name": "quantize token", "op": "quantize", "rows": 1, "cols": 4096, "format": "nvfp4", "scaled": True,
         "dtype": "bf16"},
        # a prompt's hidden states
        {"name": "quantize prompt", "op": "quantize", "rows": 8191, "cols": 4096, "format": "mxfp4", "scaled": False,
         "dtype": "bf16"},
        # a 32-bit checkpoint's matrix converted
        {"name": "quantize weights", "op": "quantize", "rows": 14336, "cols": 4096, "format": "nvfp4", "scaled": True,
         "dtype": "f32"},
        # one token through a wide projection: the weights are read once
        {"name": "product token", "op": "product", "tokens": 1, "out": 14336, "in": 4096, "format": "nvfp4",
         "scaled": True, "dtype": "bf16"},
        # a batch of decoding requests through a down projection, an odd number of them
        {"name": "product batch", "op": "product", "tokens": 77, "out": 2560, "in": 9728, "format": "mxfp4",
         "scaled": False, "dtype": "f16"},
        # a prompt
        {"name": "product prompt", "op": "product", "tokens": 4096, "out": 14336, "in": 4096, "format": "nvfp4",
         "scaled": True, "dtype": "bf16"},
        # one token through a fused query, key and value projection
        {"name": "linear token", "op": "linear", "tokens": 1, "out": 6144, "in": 2560, "dtype": "bf16"},
        # a few requests, or one request's drafted tokens, through a square projection
        {"name": "linear batch", "op": "linear", "tokens": 8, "out": 4096, "in": 4096, "dtype": "f16"},
        # a prompt
        {"name": "linear prompt", "op": "linear", "tokens": 2048, "out": 14336, "in": 4096, "dtype": "bf16"},
        # one token through its four experts
        {"name": "experts token", "op": "experts", "tokens": 1, "experts": 64, "top": 4, "dim": 2048, "hidden": 768,
         "dtype": "bf16"},
        # a decode step of a full batch: a few tokens an expert
        {"name": "experts batch", "op": "experts", "tokens": 64, "experts": 64, "top": 4, "dim": 2048, "hidden": 768,
         "dtype": "bf16"},
        # a prompt of ragged length
        {"name": "experts prompt", "op": "experts", "tokens": 4001, "experts": 64, "top": 4, "dim": 2048,
         "hidden": 768, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["quantize", "product", "product", "linear", "linear", "experts", "experts"])
    if op == "quantize":
        fmt = rng.choice(["mxfp4", "nvfp4"])
        cols = _log(rng, 2, 256) * 32 if rng.random() < 0.7 else _log(rng, 16, 8192)  # any number of columns
        return {"op": op, "rows": _log(rng, 1, min(16384, (14336 * 4096) // cols)), "cols": cols, "format": fmt,
                "scaled": fmt == "nvfp4" and rng.random() < 0.5, "dtype": rng.choice(["bf16", "bf16", "f16", "f32"])}
    if op in ("product", "linear"):
        tokens = rng.choice([1, _log(rng, 1, 64), _log(rng, 65, 4096)])
        out = _log(rng, 1, 128) * 128 if rng.random() < 0.6 else _log(rng, 8, 16384)
        n = _log(rng, 2, 128) * 64 if rng.random() < 0.6 else _log(rng, 1, 256) * 32
        if op == "linear":
            tokens = min(tokens, max(1, (2048 * 14336 * 4096) // (out * n)))
            return {"op": op, "tokens": tokens, "out": out, "in": n, "dtype": rng.choice(["bf16", "bf16", "f16"])}
        fmt = rng.choice(["mxfp4", "nvfp4"])
        tokens = min(tokens, max(1, (4096 * 14336 * 4096) // (out * n)))
        return {"op": op, "tokens": tokens, "out": out, "in": n, "format": fmt,
                "scaled": fmt == "nvfp4" and rng.random() < 0.7, "dtype": rng.choice(["bf16", "bf16", "f16", "f32"])}
    experts = rng.choice([4, 8, 16, 32, 60, 64, 128])
    top = rng.choice([1, 2, 4, 4, 6, 8])
    dim, hidden = _log(rng, 4, 128) * 32, _log(rng, 2, 64) * 32
    while experts * dim * hidden > 64 * 2048 * 1536:
        dim, hidden = max(128, dim // 64 * 32), max(64, hidden // 64 * 32)
    # the plain form takes every token through every expert: it stays below the largest listed case's
    most = max(1, min(4001, (4001 * 64 * 768) // (experts * hidden), (4001 * 64 * 2048 * 768) // (experts * dim * hidden)))
    return {"op": op, "tokens": min(most, rng.choice([1, _log(rng, 2, 64), _log(rng, 65, 4001)])), "experts": experts,
            "top": min(top, experts), "dim": dim, "hidden": hidden, "dtype": rng.choice(["bf16", "bf16", "f16"])}


# ---- the format ----------------------------------------------------------------------------------

def _codes(q):
    """Codes of 4 bits for magnitudes and signs of q: the nearest value, ties to the even code, 6 beyond."""
    a = q.abs()
    m = ((a > 0.25).to(torch.int32) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    return m + 8 * (q < 0).to(torch.int32)


def _e4m3(t):
    """The byte of the e4m3 value nearest to t >= 0 (ties to even), at most 448."""
    t = t.clamp(max=448.0)
    e = torch.frexp(t).exponent - 1
    step = torch.ldexp(torch.ones_like(t), e.clamp(min=-6) - 3)
    n = torch.round(t / step).to(torch.int32)  # 8 .. 16 eighths of 2^e, or below 8 where t < 2^-6
    return ((e.clamp(min=-6) + 6) * 8 + n).to(torch.int32)


def _quantize(x, fmt, factor):
    """(codes, scale bytes), (..., groups * group) and (..., groups), of x in 64 bits; a last group short of values is
    filled with zeros."""
    group = _GROUP[fmt]
    g = torch.nn.functional.pad(x.double(), (0, -x.shape[-1] % group)).unflatten(-1, (-1, group))
    top = g.abs().amax(-1)
    if fmt == "mxfp4":
        byte = (torch.frexp(top).exponent - 1 - 2).clamp(min=-127) + 127
        byte = torch.where(top > 0, byte, 0)
        scale = torch.ldexp(torch.ones_like(top), byte - 127)
    else:
        f = factor.double() if factor is not None else 1.0
        byte = _e4m3(top / (6.0 * f))
        scale = _scales(byte, fmt).double() * f
    q = torch.where(scale[..., None] > 0, g / torch.where(scale > 0, scale, 1.0)[..., None], 0.0)
    return _codes(q).flatten(-2), byte.to(torch.uint8)


def _scales(byte, fmt):
    """What scale bytes stand for, in 32 bits."""
    b = byte.to(torch.int32)
    if fmt == "mxfp4":
        return torch.ldexp(torch.ones(b.shape, device=b.device), b - 127)
    e, m = (b >> 3) & 15, b & 7
    return torch.where(e > 0, torch.ldexp(1 + m / 8, e - 7), torch.ldexp(m / 8, torch.full_like(e, -6)))


def _values(codes):
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], device=codes.device)
    return torch.cat([table, -table])[codes.long()]


def _dequantize(a, fmt, factor=None):
    """The values of an operand {"codes", "bytes"}, in 32 bits, as many columns as its groups hold."""
    group = _GROUP[fmt]
    shift = 4 * torch.arange(8, device=a["codes"].device, dtype=torch.int32)
    codes = ((a["codes"][..., None] >> shift) & 15).flatten(-2)
    v = _values(codes[..., :a["bytes"].shape[-1] * group]).unflatten(-1, (-1, group))
    v = (v * _scales(a["bytes"], fmt)[..., None]).flatten(-2)
    return v if factor is None else v * factor


def _operand(x, fmt, factor=None):
    """x as a program holds it in 4 bits: words of eight codes, lowest bits first, rows filled with zeros to a multiple
    of 128 codes; scale bytes by row; and the same bytes in tiles of 128 rows and four groups, the order that the tensor
    cores read them in (byte 16 (r % 32) + 4 (r / 32) + g % 4 of the 512 of rows r and groups g)."""
    codes, byte = _quantize(x, fmt, factor)
    wide = -(-codes.shape[-1] // 128) * 128
    codes = torch.nn.functional.pad(codes, (0, wide - codes.shape[-1]))
    w = codes.unflatten(-1, (-1, 8)) << (4 * torch.arange(8, device=codes.device, dtype=torch.int32))
    w = w[..., 0:4] | w[..., 4:8]
    w = w[..., 0:2] | w[..., 2:4]
    words = (w[..., 0] | w[..., 1]).contiguous()
    groups = wide // _GROUP[fmt]
    t = torch.nn.functional.pad(byte, (0, groups - byte.shape[-1], 0, -byte.shape[-2] % 128))
    t = t.unflatten(-1, (-1, 4)).unflatten(-3, (-1, 4, 32))  # (..., tile, r / 32, r % 32, g / 4, g % 4)
    return {"codes": words, "bytes": byte, "tiles": t.movedim(-2, -4).movedim(-3, -2).flatten(-3).contiguous()}


# ---- inputs --------------------------------------------------------------------------------------

def _normal(g, shape):
    return torch.randn(shape, generator=g, device="cuda")


def _activations(g, shape):
    """Normal values, a few channels of which are many times as large, as hidden states have them."""
    big = 1 + 14 * (torch.rand(shape[-1], generator=g, device="cuda") < 0.01)
    return _normal(g, shape) * big


def _factor(x):
    """The 32-bit factor of a matrix: its largest magnitude over the largest that codes and scales hold."""
    return (x.abs().amax() / (6.0 * 448.0)).float().reshape(1)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    op, dt = case["op"], _TYPE[case["dtype"]]
    s = {"case": case}
    if op == "quantize":
        shape = (case["rows"], case["cols"])
        s["x"] = (_activations(g, shape) if case["dtype"] != "f32" else 0.02 * _normal(g, shape)).to(dt)
        s["factor"] = _factor(s["x"]) if case["scaled"] else None
        return s
    if op in ("product", "linear"):
        x, w = _activations(g, (case["tokens"], case["in"])), 0.02 * _normal(g, (case["out"], case["in"]))
        if op == "linear":
            return {**s, "x": x.to(dt), "w": _operand(w, "mxfp4")}
        fx, fw = (_factor(x), _factor(w)) if case["scaled"] else (None, None)
        return {**s, "fx": fx, "fw": fw, "x": _operand(x, case["format"], fx), "w": _operand(w, case["format"], fw)}
    E, D, I, T = case["experts"], case["dim"], case["hidden"], case["tokens"]
    s["x"] = _normal(g, (T, D)).to(dt)
    score = _normal(g, (T, E)) + 0.5 * _normal(g, (1, E))  # some experts are asked more often than others
    top = score.topk(case["top"], dim=-1)
    s["inds"], s["weights"] = top.indices.to(torch.int32), torch.softmax(top.values, -1)
    s["gate_up"] = _operand(0.02 * _normal(g, (E, 2 * I, D)), "mxfp4")  # rows: gate 0, up 0, gate 1, up 1, ...
    s["down"] = _operand(0.02 * _normal(g, (E, D, I)), "mxfp4")
    return s


# ---- a pass --------------------------------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    if own:
        return _own[op](state)
    return _plain[op](state)


def _own_quantize(s):
    from locals_b200 import fp4

    a = fp4.quantize(s["x"], s["case"]["format"], scale=s["factor"])
    return fp4.dequantize(a, s["x"].dtype)


def _own_operand(a, fmt, columns, factor=None):
    from locals_b200 import fp4

    return fp4.Fp4(a["codes"], a["tiles"], fmt, columns, factor)


def _own_product(s):
    from locals_b200 import fp4

    c = s["case"]
    x, w = (_own_operand(s[m], c["format"], c["in"], s["f" + m]) for m in "xw")
    return fp4.matmul(x, w, dtype=_TYPE[c["dtype"]])


def _own_linear(s):
    from locals_b200 import fp4

    return fp4.matmul(s["x"], _own_operand(s["w"], "mxfp4", s["case"]["in"]))


def _own_experts(s):
    from locals_b200 import fp4

    c = s["case"]
    return fp4.experts(s["x"], s["inds"], s["weights"], _own_operand(s["gate_up"], "mxfp4", c["dim"]),
                       _own_operand(s["down"], "mxfp4", c["hidden"]))


_own = {"quantize": _own_quantize, "product": _own_product, "linear": _own_linear, "experts": _own_experts}


def _plain_quantize(s):
    x, fmt, factor = s["x"], s["case"]["format"], s["factor"]
    codes, byte = _quantize(x, fmt, factor)
    group = _GROUP[fmt]
    v = (_values(codes).unflatten(-1, (-1, group)) * _scales(byte, fmt)[..., None]).flatten(-2)[..., :x.shape[-1]]
    return (v if factor is None else v * factor).to(x.dtype)


def _plain_product(s):
    c = s["case"]
    x, w = (_dequantize(s[m], c["format"], s["f" + m]) for m in "xw")
    return (x @ w.T).to(_TYPE[c["dtype"]])


def _plain_linear(s):
    return (s["x"].float() @ _dequantize(s["w"], "mxfp4").T).to(s["x"].dtype)


def _plain_experts(s):
    """Every token through every expert, those that it is not routed to with weight 0."""
    x, c = s["x"].float(), s["case"]
    T, E, I = c["tokens"], c["experts"], c["hidden"]
    gu = (x @ _dequantize(s["gate_up"], "mxfp4").flatten(0, 1).T).view(T, E, I, 2)
    h = gu[..., 0] / (1 + torch.exp(-gu[..., 0])) * gu[..., 1]
    weight = torch.zeros((T, E), device=x.device).scatter_(1, s["inds"].long(), s["weights"])
    h *= weight[..., None]
    down = _dequantize(s["down"], "mxfp4").permute(1, 0, 2).flatten(1)  # (D, E * I)
    return (h.flatten(1) @ down.T).to(s["x"].dtype)


_plain = {"quantize": _plain_quantize, "product": _plain_product, "linear": _plain_linear, "experts": _plain_experts}


# ---- what a pass cannot do without ----------------------------------------------------------------

def work(case):
    op = case["op"]
    if op == "quantize":
        n = case["rows"] * case["cols"]
        size = 4 if case["dtype"] == "f32" else 2
        held = n / 2 + n / _GROUP[case["format"]]
        return {"bytes": n * size + held + held + n * size, "flops": n * 6}  # written, and read back
    if op in ("product", "linear"):
        T, N, K = case["tokens"], case["out"], case["in"]
        size = 4 if case["dtype"] == "f32" else 2
        held = 0.5 + 1 / _GROUP[case.get("format", "mxfp4")]
        x = T * K * (held if op == "product" else 2)
        return {"bytes": x + N * K * held + T * N * size, "flops": 2 * T * N * K}
    T, E, k, D, I = (case[n] for n in ("tokens", "experts", "top", "dim", "hidden"))
    used = E * (1 - (1 - k / E) ** T)  # experts that some token is routed to, on average
    return {"bytes": used * 3 * D * I * (0.5 + 1 / 32) + T * D * 4 + T * k * 8, "flops": 2 * T * k * 3 * D * I}


# ---- the definitions in 64 bits -------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"quantize": _exact_quantize, "product": _exact_product, "linear": _exact_linear,
            "experts": _exact_experts}[case["op"]](s)


_GRID = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _two_to(e):
    return ((e + 1023) << 52).view(torch.float64)


def _nearest(v, grid):
    """The value of the grid nearest to v >= 0; halfway, the one with the even place."""
    grid = torch.tensor(grid, dtype=torch.float64, device=v.device)
    middle = (grid[1:] + grid[:-1]) / 2
    at = torch.searchsorted(middle, v.contiguous())  # places below v; a tie stays with the lower value
    tie = (at < len(middle)) & (middle[at.clamp(max=len(middle) - 1)] == v) & (at % 2 == 1)
    return grid[at + tie]


def _exact_quantize(s):
    x, case = s["x"].double(), s["case"]
    group = _GROUP[case["format"]]
    f = s["factor"].double() if s["factor"] is not None else 1.0
    minifloats = [m / 8 * 2.0 ** -6 for m in range(8)] + [(1 + m / 8) * 2.0 ** e for e in range(-6, 9) for m in range(8)][:-1]
    out = torch.zeros_like(x)
    pieces = [(x[:, :x.shape[1] // group * group].unflatten(1, (-1, group)), slice(0, x.shape[1] // group * group))]
    if x.shape[1] % group:
        pieces.append((x[:, x.shape[1] // group * group:][:, None], slice(x.shape[1] // group * group, x.shape[1])))
    for v, at in pieces:
        if v.numel() == 0:
            continue
        most = v.abs().max(-1, keepdim=True).values
        if case["format"] == "mxfp4":
            scale = _two_to(((most.view(torch.int64) >> 52) - 1023 - 2).clamp(min=-127))  # the exponent's bits
        else:
            scale = _nearest(most / 6 / f, minifloats) * f
        r = _nearest((v.abs() / scale).nan_to_num(0.0, posinf=0.0), _GRID)
        out[:, at] = (torch.sign(v) * r * scale).flatten(1)
    return out


def _stands_for(a, fmt, factor, columns):
    """The matrix (or stack) that an operand holds, in 64 bits."""
    words, byte = a["codes"], a["bytes"].double()
    if fmt == "mxfp4":
        scale = _two_to(byte.long() - 127)
    else:
        e = torch.floor(byte / 8)
        scale = torch.where(e > 0, (1 + (byte - 8 * e) / 8) * _two_to(e.long() - 7), byte / 8 * 2.0 ** -6)
    grid = torch.tensor(_GRID + [-v for v in _GRID], dtype=torch.float64, device=words.device)
    out = torch.empty((*words.shape[:-1], words.shape[-1] * 8), dtype=torch.float64, device=words.device)
    for j in range(8):
        out[..., j::8] = grid[((words >> (4 * j)) & 15).long()]
    out = out[..., :columns]
    out *= scale.repeat_interleave(_GROUP[fmt], dim=-1)[..., :columns]
    return out if factor is None else out * factor.double()


def _exact_product(s):
    c = s["case"]
    return torch.einsum("tk,nk->tn", _stands_for(s["x"], c["format"], s["fx"], c["in"]),
                        _stands_for(s["w"], c["format"], s["fw"], c["in"]))


def _exact_linear(s):
    return torch.einsum("tk,nk->tn", s["x"].double(), _stands_for(s["w"], "mxfp4", None, s["case"]["in"]))


def _exact_experts(s):
    c, x = s["case"], s["x"].double()
    y = torch.zeros_like(x)
    for e in range(c["experts"]):
        token, slot = torch.where(s["inds"] == e)
        if len(token) == 0:
            continue
        part = {n: {k: v[e] for k, v in s[n].items()} for n in ("gate_up", "down")}
        gu = x[token] @ _stands_for(part["gate_up"], "mxfp4", None, c["dim"]).T
        h = torch.nn.functional.silu(gu[:, 0::2]) * gu[:, 1::2]
        y.index_add_(0, token, (h @ _stands_for(part["down"], "mxfp4", None, c["hidden"]).T) * s["weights"][token, slot, None].double())
    return y
