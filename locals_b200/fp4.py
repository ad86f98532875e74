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

from typing import NamedTuple, Optional, Tuple

import torch

from . import moe
from ._lib import ext

GROUP = {"mxfp4": 32, "nvfp4": 16}
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


def _group(mode: str) -> int:
    try:
        return GROUP[mode]
    except KeyError:
        raise ValueError(f"a 4-bit format is one of {', '.join(GROUP)}, not {mode!r}") from None


def _padded(K: int) -> int:
    return -(-K // PAD) * PAD


def _check_scale(scale: Optional[torch.Tensor], mode: str, device) -> None:
    if scale is None:
        return
    if mode != "nvfp4":
        raise ValueError("only nvfp4 has a factor for the whole matrix")
    if scale.dtype != torch.float32 or scale.numel() != 1 or scale.device != device:
        raise ValueError("scale is one float32 element on the matrix' device")


# ---- the format ----------------------------------------------------------------------------------

def pack(codes: torch.Tensor, scales: torch.Tensor, mode: str = "mxfp4", scale: Optional[torch.Tensor] = None) -> Fp4:
    """An operand of a matrix or stack in MLX's layout: ``codes`` (..., N, K/8) 32-bit words of eight codes, lowest bits
    first, ``scales`` uint8 (..., N, K/group). Done once: the scales are laid out in tiles (and codes copied where K is no
    multiple of 128)."""
    group = _group(mode)
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
    (one float32 element > 0; None: 1) is the matrix' factor, such as its largest magnitude / 2688 (0 for a matrix of zeros). Codes are the nearest to
    x / (their scales), ties to the even code, and 6 beyond it. A group with an infinity or no number in it has the scale that is
    not a number."""
    return Fp4(*ext().fp4_quantize(x, mode, scale), mode, x.shape[-1], scale)


def dequantize(a: Fp4, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values of an operand, (N, K) or (E, N, K), rounded once to ``dtype`` (with a factor and 16 bits, to 32 bits first)."""
    return ext().fp4_dequantize(a, dtype)


# ---- products ------------------------------------------------------------------------------------

def matmul(x, w: Fp4, dtype: Optional[torch.dtype] = None, glu: bool = False) -> torch.Tensor:
    """y = x . w^T with 32-bit sums, rounded once. ``x`` an ``Fp4`` matrix of w's format: y (M, N) in ``dtype`` (default
    bf16; fp16, fp32). ``x`` a tensor (..., K) in fp16 or bf16 and w in mxfp4: y (..., N) in x's dtype; x is exact down to
    2^-14 of a group of 32's largest magnitude, below that off by at most 2^-21 of it, and a row with an infinity or no number in
    it gives no numbers. ``glu``: w holds gate and up rows in turn (``interleave``) and y (..., N / 2) is silu(gate) * up."""
    if isinstance(x, Fp4):
        return ext().fp4_product(x, w, dtype or torch.bfloat16, glu)
    if dtype is not None and dtype != x.dtype:
        raise TypeError("a product of 16-bit activations has their dtype")
    return ext().fp4_linear(x, w, glu)


# ---- routed experts --------------------------------------------------------------------------------

def grouped(xs: torch.Tensor, grouping, w: Fp4, max_rows: int, glu: bool = False, gather_k: int = 0) -> torch.Tensor:
    """``moe.experts`` for a stack ``w`` (E, N, K) in mxfp4: the rows of each segment of ``grouping`` (moe.group) times its
    expert's matrix, (P, N), or (P, N / 2) with ``glu``. With gather_k, xs is the token matrix and row j of the pairs reads
    token order[j] // gather_k; otherwise xs holds one row a pair, in expert order."""
    order, starts, experts_, nseg, _ = grouping
    return ext().fp4_grouped(xs, order, starts, experts_, nseg, w, max_rows, glu, gather_k)


def switch_glu(x: torch.Tensor, inds: torch.Tensor, gate_up: Fp4, down: Fp4, grouping=None) -> torch.Tensor:
    """``moe.switch_glu`` for mxfp4 experts: x (M, D), expert ids inds (M, k), gate_up (E, 2 I, D) with gate and up rows in
    turn (``interleave``), down (E, D, I): (M, k, D), slot r of token t in row (t, r)."""
    M, k = inds.shape
    if x.dim() != 2 or x.shape[0] != M:
        raise ValueError(f"x (M, D) and inds (M, k) are wanted, not {tuple(x.shape)} and {tuple(inds.shape)}")
    if gate_up.rows != 2 * down.K or down.rows != gate_up.K or gate_up.codes.shape[0] != down.codes.shape[0]:
        raise ValueError("gate_up (E, 2 I, D) and down (E, D, I) do not fit one another")
    if M == 0 or k == 0:
        return x.new_empty((M, k, down.rows))
    with torch.cuda.device(x.device):
        g = grouping if grouping is not None else moe.group(inds, gate_up.codes.shape[0])
        h = grouped(x.contiguous(), g, gate_up, M, glu=True, gather_k=k)
        ys = grouped(h, g, down, M)
        if g[4] is not None:
            if ys.shape[1] % 8 == 0:
                ys = moe.gather(ys, g[4], 1)
            else:  # (gather copies 16 bytes at a time)
                ys = ys.index_select(0, g[4].clamp(min=0)).masked_fill_((g[4] < 0)[:, None], 0)
    return ys.reshape(M, k, -1)


def experts(x: torch.Tensor, inds: torch.Tensor, weights: torch.Tensor, gate_up: Fp4, down: Fp4) -> torch.Tensor:
    """The routed experts of a step: sum over slots r of weights[t, r] * expert inds[t, r] of x[t], (T, D) in x's dtype
    (grouping, gate and up, down, weighted sum). silu(gate) * up and the experts' outputs stay in 32 bits, so that y is rounded
    once; ``switch_glu`` gives both in x's dtype. inds int32 and weights float32 (T, k), as moe.route gives them; an id that is no
    expert's adds nothing and is recorded (``kernels.device_status``)."""
    return ext().fp4_experts(x, inds, weights, gate_up, down)


class MoELayer:
    """``moe.MoELayer`` over mxfp4 experts: router, top-k, experts, weighted sum."""

    def __init__(self, router_w: torch.Tensor, gate_up: Fp4, down: Fp4, top_k: int, mode: int = moe.SOFTMAX):
        self.router_w, self.gate_up, self.down, self.top_k, self.mode = router_w, gate_up, down, top_k, mode

    def __call__(self, x: torch.Tensor) -> torch.Tensor:
        x2 = x.reshape(-1, x.shape[-1]).contiguous()
        with torch.cuda.device(x.device):
            inds, weights = moe.route(x2, self.router_w, self.top_k, self.mode)
        return experts(x2, inds, weights, self.gate_up, self.down).reshape(x.shape)


class Linear:
    """A linear layer with an mxfp4 matrix: ``y = matmul(x, weight) (+ bias)``."""

    def __init__(self, weight: Fp4, bias: Optional[torch.Tensor] = None):
        self.weight, self.bias = weight, bias

    def __call__(self, x: torch.Tensor) -> torch.Tensor:
        y = matmul(x, self.weight)
        return y if self.bias is None else y + self.bias
