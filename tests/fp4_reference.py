"""Microscaled 4-bit floating point in 64 bits, stated plainly: what quantize makes of a matrix, what an operand stands for,
and products and experts with a bound on what 32-bit sums may lose."""

import torch

GRID = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
GROUP = {"mxfp4": 32, "nvfp4": 16}
# one e4m3 number a byte 0 .. 126
E4M3 = [m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7) for e in range(16) for m in range(8)][:127]


def nearest(v, grid):
    """Places in the grid nearest to v >= 0; halfway, the even place; beyond the last, the last."""
    g = torch.tensor(grid, dtype=torch.float64, device=v.device)
    middle = (g[1:] + g[:-1]) / 2
    at = torch.searchsorted(middle, v.contiguous())
    tie = (at < len(middle)) & (middle[at.clamp(max=len(middle) - 1)] == v) & (at % 2 == 1)
    return at + tie


def scale_values(byte, mode):
    if mode == "mxfp4":
        v = torch.exp2(byte.double().cpu() - 127).to(byte.device)
        return torch.where(byte == 255, torch.nan, v)
    table = torch.tensor(E4M3 + [float("nan")], dtype=torch.float64, device=byte.device)
    return table[byte.long()]


def quantize(x, mode, factor=None):
    """(codes (rows, groups * group), scale bytes (rows, groups)) of x (rows, K), as whole numbers."""
    group = GROUP[mode]
    f = 1.0 if factor is None else factor.double().item()
    g = torch.nn.functional.pad(x.double(), (0, -x.shape[1] % group)).unflatten(1, (-1, group))
    top = g.abs().amax(-1)
    odd = ~torch.isfinite(g).all(-1)
    if mode == "mxfp4":
        t = torch.where(odd | (top == 0), 1.0, top)
        byte = ((t.view(torch.int64) >> 52) - 1023 - 2).clamp(min=-127) + 127
        byte = torch.where(top == 0, 0, byte)
        byte = torch.where(odd, 255, byte)
    else:
        byte = torch.where(odd, 127, nearest(torch.where(odd, 0.0, top) / (6.0 * f), E4M3))
    s = scale_values(byte, mode) * f
    q = torch.where((s > 0)[..., None], g.abs() / torch.where(s > 0, s, 1.0)[..., None], 0.0)
    codes = nearest(q.nan_to_num(0.0), GRID) + 8 * (torch.signbit(g) & (s > 0)[..., None]).long()
    return codes.flatten(1), byte


def unpack_words(words, columns):
    shift = 4 * torch.arange(8, device=words.device, dtype=torch.int32)
    return ((words.view(torch.int32)[..., None] >> shift) & 15).flatten(-2)[..., :columns]


def values(codes, byte, mode, columns, factor=None):
    """What codes (..., n) and bytes (..., groups) stand for, (..., columns) in 64 bits."""
    grid = torch.tensor(GRID + [-v for v in GRID], dtype=torch.float64, device=codes.device)
    v = grid[codes.long()[..., :columns]] * scale_values(byte, mode).repeat_interleave(GROUP[mode], -1)[..., :columns]
    return v if factor is None else v * factor.double()


def tile(byte):
    """Scale bytes by row (..., rows, groups) in tiles of 128 rows and four groups, by the definition of a byte's place."""
    rows, groups = byte.shape[-2:]
    R, G = -(-rows // 128), -(-groups // 4)
    out = torch.zeros((*byte.shape[:-2], R, G, 512), dtype=torch.uint8)
    for r in range(rows):
        for g in range(groups):
            out[..., r // 128, g // 4, 16 * (r % 32) + 4 * (r % 128 // 32) + g % 4] = byte[..., r, g]
    return out


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def lost(K, a, b, steps=1):
    """What 32-bit sums of a . b^T may lose: a MMA adds 32 values or more to a sum and keeps at least 22 bits below the
    largest term, `steps` MMAs a 32 values; eight shares of a split sum are joined. a, b in 64 bits."""
    return (steps * -(-K // 32) + 8) * 2.0 ** -22 * (a.abs() @ b.abs().transpose(-1, -2))


def split_lost(x, w):
    """What the pieces of 16-bit x may miss: 2^-21 (bf16) or 2^-25 (fp16) of a group of 32's largest magnitude."""
    g = torch.nn.functional.pad(x.double().abs(), (0, -x.shape[-1] % 32)).unflatten(-1, (-1, 32)).amax(-1)
    most = g.repeat_interleave(32, -1)[..., :x.shape[-1]]
    return (2.0 ** -21 if x.dtype == torch.bfloat16 else 2.0 ** -25) * (most @ w.abs().transpose(-1, -2))


def linear(x, w, dtype):
    """(x . w^T, how far a product may be off) for x in 64 bits or 16, w in 64 bits."""
    y = x.double() @ w.transpose(-1, -2)
    bound = lost(x.shape[-1], x.double(), w, 3)
    if x.dtype in (torch.float16, torch.bfloat16):
        bound = bound + split_lost(x, w)
    return y, bound + half_step(dtype) * y.abs() + torch.finfo(dtype).tiny


def glu(x, gate, up, dtype):
    """silu(x . gate^T) * (x . up^T): the derivative of silu is below 1.1, its 32-bit form is off by less than 2^-19."""
    g, eg = linear(x, gate, torch.float32)
    u, eu = linear(x, up, torch.float32)
    s = torch.nn.functional.silu(g)
    h = s * u
    return h, 1.1 * eg * u.abs() + (s.abs() + 1.1 * eg) * eu + (2.0 ** -19 + half_step(dtype)) * h.abs() + torch.finfo(dtype).tiny


def experts(x, inds, weights, gate, up, down, dtype):
    """(y, bound) of the routed experts; gate, up (E, I, D) and down (E, D, I) in 64 bits. h and each expert's output are
    rounded to dtype, the weighted sum is taken in 32 bits and rounded."""
    y = torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    bound = torch.zeros_like(y)
    for e in range(gate.shape[0]):
        t, slot = torch.where(inds == e)
        if len(t) == 0:
            continue
        h, eh = glu(x[t], gate[e], up[e], dtype)
        hr = h.to(dtype)  # (for the bound on its pieces)
        d = h @ down[e].T
        ed = eh @ down[e].abs().T + lost(h.shape[1], h.abs() + eh, down[e], 3) + 2 * split_lost(hr, down[e])
        ed = ed + half_step(dtype) * (d.abs() + ed) + torch.finfo(dtype).tiny
        w = weights[t, slot, None].double()
        y.index_add_(0, t, w * d)
        bound.index_add_(0, t, w.abs() * (ed + 2.0 ** -22 * d.abs()))
    return y, bound + half_step(dtype) * (y.abs() + bound) + torch.finfo(dtype).tiny
