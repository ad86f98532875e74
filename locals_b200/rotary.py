"""Rotary positions with one or several axes (text: one; images: height and width; video: time, height and width).

``rotate(q, k, positions, cos, sin, axes)`` turns each pair of a head's first ``rot`` dimensions by the angle of its
token's position on the pair's axis, in one sm_100a kernel (``lq_rotary``) for queries and keys: 32-bit arithmetic,
rounded once. ``tables`` makes the cos and sin tables, ``sections`` the axis of each pair.
"""

from __future__ import annotations

from typing import Optional, Sequence, Tuple

import torch

from ._lib import ext


def tables(positions: int, rot: int, base: float = 10000.0, device="cuda") -> Tuple[torch.Tensor, torch.Tensor]:
    """cos and sin (positions, rot / 2) float32 of position * base^(-2 j / rot), computed in 64 bits: one run of frequencies
    over all pairs, whatever their axes. Where an axis' pairs start the run anew, join the axes' own tables along the pairs
    (``torch.cat([tables(n, 2 * pairs_of_axis)[0], ...], 1)``)."""
    inv = base ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * inv
    return angle.cos().float().to(device), angle.sin().float().to(device)


def sections(counts: Sequence[int], device="cuda") -> torch.Tensor:
    """The axis of each pair, (sum(counts),) int32: the first counts[0] pairs on axis 0, the next on axis 1, ..."""
    return torch.tensor([a for a, n in enumerate(counts) for _ in range(n)], dtype=torch.int32, device=device)


def rotate(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
           axes: Optional[torch.Tensor] = None, interleaved: bool = False):
    """``q`` (N, H, D) and ``k`` (N, KVH, D) (or None) rotated: (q', k'). ``positions`` (N,) or (naxes, N) int32; ``cos``,
    ``sin`` (max positions, rot / 2) float32; ``axes`` (rot / 2,) int32 names each pair's axis (None: axis 0). Pairs are
    (j, j + rot / 2), or (2 j, 2 j + 1) when ``interleaved``; dimensions from rot on are copied. A position outside the
    tables takes the nearest row and sets LQ_DEV_BOUNDS in the device status."""
    return ext().rotate(q, k, positions, cos, sin, axes, interleaved)
