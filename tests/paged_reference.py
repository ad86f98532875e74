"""Plain statements of the paged 4-bit cache's operators, in 64 bits or in whole numbers, for the tests."""

import math

import torch

GROUP = 64
#: unit roundoff of the activation dtypes
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def plan(cached, new, table, free, head, page, tokens):
    """(table, lens, q_start, positions, slots, head) as Python lists."""
    table = [list(r) for r in table]
    lens, q_start, positions, slots = [], [0], [], []
    for b, (c, n) in enumerate(zip(cached, new)):
        c, n = max(c, 0), max(n, 0)
        for col in range(-(-c // page), -(-(c + n) // page)):
            if col < len(table[b]):
                table[b][col] = free[head] if head < len(free) else -1
            head += 1
        for p in range(c, c + n):
            col = p // page
            ident = table[b][col] if col < len(table[b]) else -1
            positions.append(p)
            slots.append(ident * page + p % page if ident >= 0 else -1)
        lens.append(c + n)
        q_start.append(q_start[-1] + n)
    positions += [0] * (tokens - len(positions))
    slots += [-1] * (tokens - len(slots))
    return table, lens, q_start, positions[:tokens], slots[:tokens], head


def rotated(x, positions, cos, sin, axes, interleaved):
    """x (N, heads, D) rotated in 64 bits; and what its 32-bit products may be off by, a value."""
    N, _, D = x.shape
    half = cos.shape[1]
    pos = positions if positions.dim() == 2 else positions[None]
    ax = axes.long() if axes is not None else torch.zeros(half, dtype=torch.long, device=x.device)
    at = pos.long()[ax].T.clamp(0, cos.shape[0] - 1)  # (N, half)
    j = torch.arange(half, device=x.device)
    c, s = cos.double()[at, j][:, None], sin.double()[at, j][:, None]
    a_ix, b_ix = (2 * j, 2 * j + 1) if interleaved else (j, j + half)
    y, slack = x.double().clone(), torch.zeros_like(x, dtype=torch.float64)
    a, b = x.double()[..., a_ix], x.double()[..., b_ix]
    y[..., a_ix], y[..., b_ix] = a * c - b * s, b * c + a * s
    slack[..., a_ix] = slack[..., b_ix] = 2.0 ** -22 * (a.abs() + b.abs())
    return y, slack


def rotated32(x, positions, cos, sin, axes, interleaved):
    """The rotation in 32 bits, each product, difference and sum rounded by itself."""
    half = cos.shape[1]
    pos = positions if positions.dim() == 2 else positions[None]
    ax = axes.long() if axes is not None else torch.zeros(half, dtype=torch.long, device=x.device)
    at = pos.long()[ax].T
    j = torch.arange(half, device=x.device)
    c, s = cos[at, j][:, None], sin[at, j][:, None]
    a_ix, b_ix = (2 * j, 2 * j + 1) if interleaved else (j, j + half)
    y = x.float().clone()
    a, b = x.float()[..., a_ix], x.float()[..., b_ix]
    y[..., a_ix] = a * c - b * s
    y[..., b_ix] = b * c + a * s
    return y


def unpacked(triple):
    """(pages, KVH, page, D) in 64 bits of a 4-bit triple."""
    w, s, b = triple
    x = torch.stack([(w >> (4 * i)) & 15 for i in range(8)], -1).flatten(-2).double()
    return x * s.double().repeat_interleave(GROUP, -1) + b.double().repeat_interleave(GROUP, -1)


def attended(q, keys, values, table, lens, scale, q_start, sinks, window):
    """(out, bound) in 64 bits: attention of each query by itself, and how far a result in q's dtype may be off -- the
    output's rounding, u |out|; probabilities and values that are each rounded to 11 bits, 2 * 2^-11 of A = sum p |v| /
    sum p; keys rounded to 11 bits, which move a score by at most 2^-11 scale sum |q k| and so every p by that share (in
    the sum and in its divisor: twice); and 2^-14 of A for 32-bit arithmetic."""
    N, H, D = q.shape
    k, v = unpacked(keys), unpacked(values)
    KVH, page = k.shape[1], k.shape[2]
    G = H // KVH
    out = torch.zeros((N, H, D), dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    lens = lens.tolist()
    start = q_start.tolist() if q_start is not None else list(range(len(lens) + 1))
    for b, n in enumerate(lens):
        new = start[b + 1] - start[b]
        if new == 0 or n == 0:
            continue
        ids = table[b, :-(-n // page)].long()
        kb = k[ids].transpose(0, 1).flatten(1, 2)[:, :n]  # (KVH, n, D)
        vb = v[ids].transpose(0, 1).flatten(1, 2)[:, :n]
        x = q[start[b]:start[b + 1]].double().view(new, KVH, G, D)
        s = scale * torch.einsum("ihgd,hjd->hgij", x, kb)
        at = (n - new + torch.arange(new, device=q.device))[:, None]
        j = torch.arange(n, device=q.device)[None]
        seen = (j <= at) & ((j > at - window) if window else torch.ones_like(j, dtype=torch.bool))
        s = s.masked_fill(~seen, -math.inf)
        m = s.amax(-1, keepdim=True)
        if sinks is not None:
            sk = sinks.double().view(KVH, G, 1, 1)
            m = torch.maximum(m, sk)
        m = torch.where(m == -math.inf, 0.0, m)
        p = (s - m).exp()
        tot = p.sum(-1, keepdim=True)
        if sinks is not None:
            tot = tot + (sk - m).exp()
        p = p / torch.where(tot > 0, tot, 1.0)
        o = torch.einsum("hgij,hjd->ihgd", p, vb)
        A = torch.einsum("hgij,hjd->ihgd", p, vb.abs())
        qk = abs(scale) * torch.einsum("ihgd,hjd->hgij", x.abs(), kb.abs()).masked_fill(~seen, 0.0).amax(-1)
        moved = 2 * 2.0 ** -11 * qk.permute(2, 0, 1)[..., None]
        out[start[b]:start[b + 1]] = o.reshape(new, H, D)
        bound[start[b]:start[b + 1]] = (U[q.dtype] * o.abs() + A * (2.0 ** -10 + 2.0 ** -14 + moved)).reshape(new, H, D)
    return out, bound + 2.0 ** -24  # (the least values of the dtypes)
