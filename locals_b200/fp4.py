"""Microscaled 4-bit floating point: weights and activations of 4 bits (e2m1: 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their
negatives) in groups along the input dimension that share a scale of 8 bits, multiplied by the block-scaled tensor cores.

    w = pack(codes, scales)                       # a checkpoint's mxfp4 matrix (MLX's layout), once
    y = matmul(x, w)                              # x in 16 bits, or
    y = matmul(quantize(x, "nvfp4", s), w)        # both in 4 bits
    y = experts(x, inds, weights, gate_up, down)  # routed SwiGLU experts (the reference's mxfp4 experts,
                                                  # locals/moe_kernel.py:68-155,230-239)

* "mxfp4": groups of 32, scale 2^(byte - 127); * "nvfp4": groups of 16, scale an e4m3 number, and a float32 factor for the
whole matrix (``scale``). An operand (``Fp4``) holds words of eight codes, rows filled with zero codes to a multiple of 128, and
the scale bytes in the tiles of 128 rows x 4 groups that the tensor cores read; ``pack`` and ``unpack`` go between it and
MLX's layout (words (..., N, K/8), scale bytes (..., N, K/group)). 16-bit activations are multiplied with "mxfp4" weights
only: the tensor cores take an e4m3 scale with 4 bits on both sides only.
"""

from __future__ import annotations

from typing import NamedTuple, Optional, Sequence, Tuple

import torch

from . import _lib, moe
from ._lib import call
from .kernels import _ptr, _stream, dtype_code

GROUP = {"mxfp4": 32, "nvfp4": 16}
_MODE = {"mxfp4": _lib.MXFP4, "nvfp4": _lib.NVFP4}
PAD = 128  # codes a row is filled to a multiple of


class Fp4(NamedTuple):
    """A matrix (N, K), or a stack (E, N, K) of them, in 4 bits: ``codes`` int32 (..., N, Kp / 8) with Kp = K rounded up to a
    multiple of 128; ``tiles`` uint8 (..., ceil(N / 128), Kp / (4 * group), 512); the format; K; the matrix' float32
    factor (one element, "nvfp4" only) or None."""

    codes: torch.Tensor
    tiles: torch.Tensor
    mode: str
    K: int
    scale: Optional[torch.Tensor] = None

    @property
    def rows(self) -> int:
        return self.codes.shape[-2]


def _mode(mode: str) -> int:
    try:
        return _MODE[mode]
    except KeyError:
        raise ValueError(f"a 4-bit format is one of {', '.join(_MODE)}, not {mode!r}") from None


def _padded(K: int) -> int:
    return -(-K // PAD) * PAD


def _check_scale(scale: Optional[torch.Tensor], mode: str, device) -> None:
    if scale is None:
        return
    if mode != "nvfp4":
        raise ValueError("only nvfp4 has a factor for the whole matrix")
    if scale.dtype != torch.float32 or scale.numel() != 1 or scale.device != device:
        raise ValueError("scale is one float32 element on the matrix' device")


def _check(a: Fp4, what: str, dims: Sequence[int] = (2,)) -> None:
    """An operand's tensors fit one another: the kernels read them through raw pointers."""
    code = _mode(a.mode)
    if not a.codes.is_cuda or a.tiles.device != a.codes.device:
        raise ValueError(f"{what}: codes and tiles are CUDA tensors of one device")
    if a.codes.dtype not in (torch.int32, torch.uint32) or a.tiles.dtype != torch.uint8:
        raise TypeError(f"{what}: codes are 32-bit words and tiles uint8")
    if a.codes.dim() not in dims:
        raise ValueError(f"{what}: codes have {' or '.join(map(str, dims))} dimensions, not {a.codes.dim()}")
    if a.K < 1:
        raise ValueError(f"{what}: K={a.K}")
    N, Kp = a.codes.shape[-2], _padded(a.K)
    want = (*a.codes.shape[:-2], -(-N // 128), Kp // (4 * GROUP[a.mode]), 512)
    if a.codes.shape[-1] != Kp // 8 or tuple(a.tiles.shape) != want:
        raise ValueError(f"{what}: codes {tuple(a.codes.shape)} / tiles {tuple(a.tiles.shape)} do not hold {N} rows of "
                         f"K={a.K} in {a.mode} (tiles {want})")
    if not a.codes.is_contiguous() or not a.tiles.is_contiguous():
        raise ValueError(f"{what}: codes and tiles are contiguous")
    _check_scale(a.scale, a.mode, a.codes.device)
    return code


class _on:
    """The device of a call's tensors made current where it is not."""

    def __init__(self, device: torch.device):
        i = device.index
        self.guard = None if i is None or i == torch._C._cuda_getDevice() else torch.cuda.device(i)

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()

    def __exit__(self, *a):
        if self.guard is not None:
            self.guard.__exit__(*a)


def _rows(x: torch.Tensor) -> torch.Tensor:
    """x (..., K) as rows: a view where the rows lie at one distance and a row's values next to one another."""
    if x.dim() == 0:
        raise ValueError("a matrix of rows is wanted")
    x2 = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    if x2.shape[1] > 1 and x2.stride(1) != 1 or x2.shape[0] > 1 and x2.stride(0) < x2.shape[1]:
        x2 = x2.contiguous()
    return x2


def _row_stride(x2: torch.Tensor) -> int:
    return x2.stride(0) if x2.shape[0] > 1 else x2.shape[1]


# ---- the format ----------------------------------------------------------------------------------

def pack(codes: torch.Tensor, scales: torch.Tensor, mode: str = "mxfp4", scale: Optional[torch.Tensor] = None) -> Fp4:
    """An operand of a matrix or stack in MLX's layout: ``codes`` (..., N, K/8) 32-bit words of eight codes, lowest bits
    first, ``scales`` uint8 (..., N, K/group). Done once: the scales are laid out in tiles (and codes copied where K is no
    multiple of 128)."""
    _mode(mode)
    group = GROUP[mode]
    if codes.dtype not in (torch.int32, torch.uint32) or scales.dtype != torch.uint8:
        raise TypeError("codes are 32-bit words and scales uint8")
    K = codes.shape[-1] * 8
    if codes.dim() not in (2, 3) or K % group or tuple(scales.shape) != (*codes.shape[:-1], K // group):
        raise ValueError(f"codes {tuple(codes.shape)} and scales {tuple(scales.shape)} are no {mode} matrix or stack")
    _check_scale(scale, mode, codes.device)
    codes = codes.view(torch.int32)
    Kp, N = _padded(K), codes.shape[-2]
    if Kp != K:
        codes = torch.nn.functional.pad(codes, (0, (Kp - K) // 8))
    t = torch.nn.functional.pad(scales, (0, (Kp - K) // group, 0, -N % 128))
    t = t.unflatten(-1, (-1, 4)).unflatten(-3, (-1, 4, 32))  # (..., tile, r / 32, r % 32, g / 4, g % 4)
    tiles = t.movedim(-2, -4).movedim(-3, -2).flatten(-3).contiguous()
    return Fp4(codes.contiguous(), tiles, mode, K, scale)


def unpack(a: Fp4) -> Tuple[torch.Tensor, torch.Tensor]:
    """(codes, scales) of an operand in MLX's layout; a K that its groups do not divide is filled up with zero codes."""
    group = GROUP[a.mode]
    groups = -(-a.K // group)
    t = a.tiles.unflatten(-1, (32, 4, 4)).movedim(-2, -3)  # (..., tile, k tile, r / 32, r % 32, g % 4)
    s = t.movedim(-4, -2).flatten(-2).flatten(-4, -2)  # (..., rows, groups)
    return a.codes[..., :groups * group // 8].contiguous(), s[..., :a.codes.shape[-2], :groups].contiguous()


def interleave(gate: Tuple[torch.Tensor, torch.Tensor], up: Tuple[torch.Tensor, torch.Tensor],
               mode: str = "mxfp4") -> Fp4:
    """One operand of gate and up projections (MLX's layout, (codes, scales) each) with their rows in turn: gate 0, up 0,
    gate 1, ... -- what ``matmul(..., glu=True)`` and the experts take."""
    if any(g.shape != u.shape for g, u in zip(gate, up)):
        raise ValueError("gate and up differ in shape")
    return pack(*(torch.stack((g.view(torch.int32) if i == 0 else g, u.view(torch.int32) if i == 0 else u), -2).flatten(-3, -2)
                  for i, (g, u) in enumerate(zip(gate, up))), mode)


def quantize(x: torch.Tensor, mode: str = "mxfp4", scale: Optional[torch.Tensor] = None) -> Fp4:
    """x (..., K) in fp16, bf16 or fp32 to 4 bits, its leading dimensions flattened to rows. mxfp4: a group's scale is
    2^(floor(log2 of its largest magnitude) - 2). nvfp4: the e4m3 number nearest to that magnitude / (6 scale), where ``scale``
    (one float32 element > 0; None: 1) is the matrix' factor, such as its largest magnitude / 2688. Codes are the nearest to
    x / (their scales), ties to the even code, and 6 beyond it. A group with an infinity or no number in it has the scale that is
    not a number."""
    code = _mode(mode)
    dt = dtype_code(x.dtype)
    if not x.is_cuda:
        raise ValueError("locals_b200 kernels take CUDA tensors")
    _check_scale(scale, mode, x.device)
    x2 = _rows(x)
    R, K = x2.shape
    if K < 1:
        raise ValueError("rows of no values")
    Kp = _padded(K)
    codes = torch.empty((R, Kp // 8), dtype=torch.int32, device=x.device)
    tiles = torch.empty((-(-R // 128), Kp // (4 * GROUP[mode]), 512), dtype=torch.uint8, device=x.device)
    if R:
        with _on(x.device):
            call("lq_fp4_quantize", x2.data_ptr(), dt, _row_stride(x2), R, K, code, _ptr(scale), codes.data_ptr(),
                 tiles.data_ptr(), _stream())
    return Fp4(codes, tiles, mode, K, scale)


def dequantize(a: Fp4, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values of an operand, (N, K) or (E, N, K), rounded once to ``dtype``."""
    code = _check(a, "dequantize", (2, 3))
    dt = dtype_code(dtype)
    out = torch.empty((*a.codes.shape[:-1], a.K), dtype=dtype, device=a.codes.device)
    if out.numel():
        with _on(out.device):
            call("lq_fp4_dequantize", a.codes.data_ptr(), a.tiles.data_ptr(), a.codes.shape[0] if a.codes.dim() == 3 else 1,
                 a.rows, a.K, code, _ptr(a.scale), dt, out.data_ptr(), _stream())
    return out


# ---- products ------------------------------------------------------------------------------------

def matmul(x, w: Fp4, dtype: Optional[torch.dtype] = None, glu: bool = False) -> torch.Tensor:
    """y = x . w^T with 32-bit sums, rounded once. ``x`` an ``Fp4`` matrix of w's format: y (M, N) in ``dtype`` (default
    bf16; fp16, fp32). ``x`` a tensor (..., K) in fp16 or bf16 and w in mxfp4: y (..., N) in x's dtype; x is exact down to
    2^-13 of a group of 32's largest magnitude, below that off by at most 2^-21 of it, and a row with an infinity or no number in
    it gives no numbers. ``glu``: w holds gate and up rows in turn (``interleave``) and y (..., N / 2) is silu(gate) * up."""
    code = _check(w, "w")
    N = w.rows
    if glu and N % 2:
        raise ValueError(f"{N} rows are no pairs of gate and up")
    width = N // 2 if glu else N
    if isinstance(x, Fp4):
        _check(x, "x")
        if x.mode != w.mode or x.K != w.K:
            raise ValueError(f"x ({x.mode}, K={x.K}) and w ({w.mode}, K={w.K}) do not multiply")
        if x.codes.device != w.codes.device:
            raise ValueError("x and w are on different devices")
        dtype = dtype or torch.bfloat16
        y = torch.empty((x.rows, width), dtype=dtype, device=w.codes.device)
        dt = dtype_code(dtype)
        if y.numel():
            with _on(y.device):
                call("lq_fp4_qmm", x.codes.data_ptr(), x.tiles.data_ptr(), _ptr(x.scale), w.codes.data_ptr(),
                     w.tiles.data_ptr(), _ptr(w.scale), x.rows, N, w.K, code, int(glu), dt, y.data_ptr(), _stream())
        return y
    _check_16(x, w)
    if dtype is not None and dtype != x.dtype:
        raise TypeError("a product of 16-bit activations has their dtype")
    x2 = _rows(x)
    M, dt = x2.shape[0], dtype_code(x.dtype)
    y = torch.empty((M, width), dtype=x.dtype, device=x.device)
    if y.numel():
        with _on(y.device):
            n = int(_lib.lib().lq_fp4_linear_workspace(M, w.K, dt))
            ws = torch.empty(n, dtype=torch.uint8, device=x.device)
            call("lq_fp4_linear", x2.data_ptr(), _row_stride(x2), w.codes.data_ptr(), w.tiles.data_ptr(), M, N, w.K, int(glu),
                 dt, y.data_ptr(), ws.data_ptr(), n, _stream())
    return y.reshape(*x.shape[:-1], width)


def _check_16(x: torch.Tensor, w: Fp4) -> None:
    if x.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError(f"activations are fp16, bf16 or Fp4, not {x.dtype}")
    if w.mode != "mxfp4":
        raise ValueError(f"16-bit activations are multiplied with mxfp4 weights, not {w.mode}: quantize them for it")
    if x.device != w.codes.device:
        raise ValueError("x and w are on different devices")
    if x.dim() < 1 or x.shape[-1] != w.K:
        raise ValueError(f"x {tuple(x.shape)} does not match K={w.K}")


# ---- routed experts --------------------------------------------------------------------------------

def grouped(xs: torch.Tensor, grouping, w: Fp4, max_rows: int, glu: bool = False, gather_k: int = 0) -> torch.Tensor:
    """``moe.experts`` for a stack ``w`` (E, N, K) in mxfp4: the rows of each segment of ``grouping`` (moe.group) times its
    expert's matrix, (P, N), or (P, N / 2) with ``glu``. With gather_k, xs is the token matrix and row j of the pairs reads
    token order[j] // gather_k; otherwise xs holds one row a pair, in expert order."""
    _check(w, "experts", (3,))
    _check_16(xs, w)
    order, starts, experts_, nseg, _ = grouping
    E, N, P = w.codes.shape[0], w.rows, order.numel()
    if xs.dim() != 2 or not xs.is_contiguous():
        raise ValueError("xs is a contiguous matrix of rows")
    if glu and N % 2:
        raise ValueError(f"{N} rows are no pairs of gate and up")
    if not gather_k and xs.shape[0] < P:
        raise ValueError(f"{xs.shape[0]} rows for {P} pairs")
    out = torch.empty((P, N // 2 if glu else N), dtype=xs.dtype, device=xs.device)
    if out.numel():
        dt = dtype_code(xs.dtype)
        with _on(out.device):
            n = int(_lib.lib().lq_fp4_experts_workspace(P, max_rows, E, w.K, dt))
            ws = torch.empty(n, dtype=torch.uint8, device=xs.device)
            call("lq_fp4_experts", xs.data_ptr(), xs.shape[0], order.data_ptr() if gather_k else None, gather_k,
                 starts.data_ptr(), experts_.data_ptr(), nseg.data_ptr(), P, max_rows, int(glu), w.codes.data_ptr(),
                 w.tiles.data_ptr(), out.data_ptr(), E, N, w.K, dt, ws.data_ptr(), n, _stream())
    return out


def _check_experts(x: torch.Tensor, inds: torch.Tensor, gate_up: Fp4, down: Fp4) -> None:
    _check(gate_up, "gate_up", (3,))
    _check(down, "down", (3,))
    if x.dim() != 2 or inds.dim() != 2 or inds.shape[0] != x.shape[0] or inds.dtype not in (torch.int32, torch.uint32):
        raise ValueError(f"x (T, D) and inds int32 (T, k) are wanted, not {tuple(x.shape)} and {tuple(inds.shape)}")
    if inds.device != x.device:
        raise ValueError("x and inds are on different devices")
    E, rows, D = gate_up.codes.shape[0], gate_up.rows, gate_up.K
    if rows % 2 or down.codes.shape[0] != E or down.K != rows // 2 or down.rows != D:
        raise ValueError(f"gate_up ({E}, {rows}, {D}) and down ({down.codes.shape[0]}, {down.rows}, {down.K}) are no experts")


def _pairs(x: torch.Tensor, inds: torch.Tensor, gate_up: Fp4, down: Fp4, grouping) -> torch.Tensor:
    M, k = inds.shape
    h = grouped(x.contiguous(), grouping, gate_up, M, glu=True, gather_k=k)
    return grouped(h, grouping, down, M)


def _grouping(inds: torch.Tensor, E: int):
    return moe.direct_grouping(inds) if inds.shape[0] <= moe.DIRECT_MAX_TOKENS else moe.group(inds, E)


def switch_glu(x: torch.Tensor, inds: torch.Tensor, gate_up: Fp4, down: Fp4, grouping=None) -> torch.Tensor:
    """``moe.switch_glu`` for mxfp4 experts: x (M, D), expert ids inds (M, k), gate_up (E, 2 I, D) with gate and up rows in
    turn (``interleave``), down (E, D, I): (M, k, D), slot r of token t in row (t, r)."""
    _check_experts(x, inds, gate_up, down)
    M, k = inds.shape
    if M == 0 or k == 0:
        return x.new_empty((M, k, x.shape[1]))
    with _on(x.device):
        g = grouping if grouping is not None else _grouping(inds, gate_up.codes.shape[0])
        ys = _pairs(x, inds, gate_up, down, g)
        if g[4] is not None:
            ys = moe.gather(ys, g[4], 1)
    return ys.reshape(M, k, -1)


def experts(x: torch.Tensor, inds: torch.Tensor, weights: torch.Tensor, gate_up: Fp4, down: Fp4) -> torch.Tensor:
    """The routed experts of a step: sum over slots r of weights[t, r] * expert inds[t, r] of x[t], (T, D) in x's dtype
    (``switch_glu``, then ``moe.combine``). weights float32 (T, k). A token names an expert at most once."""
    _check_experts(x, inds, gate_up, down)
    if weights.shape != inds.shape or weights.dtype != torch.float32 or weights.device != x.device:
        raise ValueError("weights are float32, one an expert id")
    if inds.numel() == 0:
        return torch.zeros_like(x)
    with _on(x.device):
        g = _grouping(inds, gate_up.codes.shape[0])
        return moe.combine(_pairs(x, inds, gate_up, down, g), weights.contiguous(), g[4])


class MoELayer:
    """``moe.MoELayer`` over mxfp4 experts: router, top-k, experts, weighted sum."""

    def __init__(self, router_w: torch.Tensor, gate_up: Fp4, down: Fp4, top_k: int, mode: int = moe.SOFTMAX):
        self.router_w, self.gate_up, self.down, self.top_k, self.mode = router_w, gate_up, down, top_k, mode

    def __call__(self, x: torch.Tensor) -> torch.Tensor:
        x2 = x.reshape(-1, x.shape[-1]).contiguous()
        inds, weights = moe.route(x2, self.router_w, self.top_k, self.mode)
        return experts(x2, inds, weights, self.gate_up, self.down).reshape(x.shape)


class Linear:
    """A linear layer with an mxfp4 matrix: ``y = matmul(x, weight) (+ bias)``."""

    def __init__(self, weight: Fp4, bias: Optional[torch.Tensor] = None):
        self.weight, self.bias = weight, bias

    def __call__(self, x: torch.Tensor) -> torch.Tensor:
        y = matmul(x, self.weight)
        return y if self.bias is None else y + self.bias
