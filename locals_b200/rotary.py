"""Rotary positions with one or several axes (text: one; images: height and width; video: time, height and width).

``rotate(q, k, positions, cos, sin, axes)`` turns each pair of a head's first ``rot`` dimensions by the angle of its
token's position on the pair's axis, in one sm_100a kernel (``lq_rotary``) for queries and keys: 32-bit arithmetic,
rounded once. ``tables`` makes the cos and sin tables, ``sections`` the axis of each pair.
"""

from __future__ import annotations

from typing import Optional, Sequence, Tuple

import torch

from ._lib import call
from .kernels import _stream, dtype_code


def tables(positions: int, rot: int, base: float = 10000.0, device="cuda") -> Tuple[torch.Tensor, torch.Tensor]:
    """cos and sin (positions, rot / 2) float32 of position * base^(-2 j / rot), computed in 64 bits."""
    inv = base ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * inv
    return angle.cos().float().to(device), angle.sin().float().to(device)


def sections(counts: Sequence[int], device="cuda") -> torch.Tensor:
    """The axis of each pair, (sum(counts),) int32: the first counts[0] pairs on axis 0, the next on axis 1, ..."""
    return torch.tensor([a for a, n in enumerate(counts) for _ in range(n)], dtype=torch.int32, device=device)


def _rows(x: torch.Tensor, name: str) -> Tuple[torch.Tensor, int]:
    """x (N, heads, D) with a token's heads contiguous (a slice of a fused projection is fine), and the elements from
    one token to the next."""
    if x.dim() != 3:
        raise ValueError(f"{name}: (tokens, heads, head_dim) expected, got {tuple(x.shape)}")
    if not x.is_cuda or x.get_device() != torch._C._cuda_getDevice():
        raise ValueError("locals_b200 kernels take CUDA tensors of the current device")
    N, H, D = x.shape
    if x.is_contiguous():
        return x, H * D
    sn, sh, sd = x.stride()
    if (sd != 1 and D > 1) or (sh != D and H > 1) or (N > 1 and sn < H * D):
        return x.contiguous(), H * D
    return x, (sn if N > 1 else H * D)


def _like(x: torch.Tensor) -> torch.Tensor:
    """A contiguous tensor of x's shape, dtype and device."""
    return torch.empty_like(x) if x.is_contiguous() else torch.empty_like(x, memory_format=torch.contiguous_format)


def _angles(positions, cos, sin, axes, N: int, D: int) -> Tuple[int, int]:
    """(rot, number of axes) of checked angle arguments."""
    ps, cs = positions.shape, cos.shape
    if positions.dtype != torch.int32 or len(ps) not in (1, 2) or ps[-1] != N:
        raise ValueError(f"positions: int32 ({N},) or (axes, {N}) expected")
    if cos.dtype != torch.float32 or sin.dtype != torch.float32 or len(cs) != 2 or cs != sin.shape:
        raise ValueError("cos and sin: float32 (positions, rot / 2) tables expected")
    rot, naxes = 2 * cs[1], 1 if len(ps) == 1 else ps[0]
    if rot < 2 or rot > D or cs[0] < 1 or naxes < 1:
        raise ValueError(f"{rot} rotated dimensions do not fit head_dim {D}")
    if axes is not None and (axes.dtype != torch.int32 or tuple(axes.shape) != (rot // 2,)):
        raise ValueError(f"axes: int32 ({rot // 2},) expected")
    d = torch._C._cuda_getDevice()
    for t in (positions, cos, sin, axes):
        if t is not None and (t.get_device() != d or not t.is_contiguous()):
            raise ValueError("positions, cos, sin and axes must be contiguous tensors on the queries' device")
    return rot, naxes


def rotate(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
           axes: Optional[torch.Tensor] = None, interleaved: bool = False):
    """``q`` (N, H, D) and ``k`` (N, KVH, D) (or None) rotated: (q', k'). ``positions`` (N,) or (naxes, N) int32; ``cos``,
    ``sin`` (max positions, rot / 2) float32; ``axes`` (rot / 2,) int32 names each pair's axis (None: axis 0). Pairs are
    (j, j + rot / 2), or (2 j, 2 j + 1) when ``interleaved``; dimensions from rot on are copied. A position outside the
    tables takes the nearest row and sets LQ_DEV_BOUNDS in the device status."""
    q, q_row = _rows(q, "q")
    N, H, D = q.shape
    KVH, k_row = 0, 0
    if k is not None:
        k, k_row = _rows(k, "k")
        KVH = k.shape[1]
        if k.shape[0] != N or k.shape[2] != D or k.dtype != q.dtype:
            raise ValueError("q and k must have the same tokens, head_dim and dtype")
    rot, naxes = _angles(positions, cos, sin, axes, N, D)
    qo = _like(q)
    ko = None if k is None else _like(k)
    if N:
        call("lq_rotary", q.data_ptr(), q_row, qo.data_ptr(), H, None if k is None else k.data_ptr(), k_row,
             None if k is None else ko.data_ptr(), KVH, N, D, rot, positions.data_ptr(), cos.data_ptr(), sin.data_ptr(),
             cos.shape[0], None if axes is None else axes.data_ptr(), naxes, int(interleaved), dtype_code(q.dtype),
             _stream())
    return qo, ko
