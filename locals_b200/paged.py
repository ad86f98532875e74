"""A paged key/value cache in 4 bits: what a serving step does between its fused QKV projection and its output
projection, for a batch of requests of different lengths.

    p = plan(cached, new, table, free, head, page_size, tokens)        # block tables and slot maps, on the GPU
    q = append(q, k, v, p.slots, keys, values, p.positions, cos, sin)  # a layer: rotate, quantize, store
    o = attend(q, keys, values, table, p.lens, scale, q_start=p.q_start, max_q=...)

``keys`` and ``values`` are triples (words int32 (pages, KVH, page_size, D / 8), scales, biases (pages, KVH, page_size,
D / 64)) of MLX affine 4-bit groups of 64, as ``kernels.quantize`` writes them (the 8-bit cache of qkv.py has the same
layout with one page a row). ``pool`` makes an empty one; ``read`` gives back the values at given slots. Head dimensions
64, 128 and 256; pages of a multiple of 8 tokens; fp16 and bf16.

What the kernels find out of range in device memory (page ids, slots, positions, lengths beyond the table) they leave
out, and set LQ_DEV_BOUNDS in the device status (``kernels.device_status``).
"""

from __future__ import annotations

from typing import NamedTuple, Optional, Sequence, Tuple

import torch

from ._lib import ext

BITS, GROUP = 4, 64
HEAD_DIMS = (64, 128, 256)

Triple = Tuple[torch.Tensor, torch.Tensor, torch.Tensor]


class Plan(NamedTuple):
    """A step's lengths and places: ``lens`` (B,) tokens a request after the step; ``q_start`` (B + 1,) where its new
    tokens start; ``positions`` and ``slots`` (tokens,) of each new token (padding: 0 and -1); ``head`` (1,) the next
    free entry of the free list. All int32."""

    lens: torch.Tensor
    q_start: torch.Tensor
    positions: torch.Tensor
    slots: torch.Tensor
    head: torch.Tensor


def pool(pages: int, KVH: int, page_size: int, head_dim: int, dtype: torch.dtype = torch.bfloat16,
         device="cuda") -> Tuple[Triple, Triple]:
    """Empty keys and values of a cache of ``pages`` pages."""
    if head_dim not in HEAD_DIMS or page_size < 8 or page_size % 8:
        raise ValueError(f"a 4-bit cache has head_dim 64, 128 or 256 and pages of a multiple of 8 tokens, not "
                         f"{head_dim} and {page_size}")

    def one() -> Triple:
        return (torch.zeros((pages, KVH, page_size, head_dim // 8), dtype=torch.int32, device=device),
                torch.zeros((pages, KVH, page_size, head_dim // GROUP), dtype=dtype, device=device),
                torch.zeros((pages, KVH, page_size, head_dim // GROUP), dtype=dtype, device=device))

    return one(), one()


def plan(cached: torch.Tensor, new: torch.Tensor, block_table: torch.Tensor, free: torch.Tensor, head: torch.Tensor,
         page_size: int, tokens: int) -> Plan:
    """The block tables and slot maps of a step, built on the GPU in one launch: request b holds ``cached[b]`` tokens, in
    the pages that the first entries of ``block_table[b]`` name, and brings ``new[b]``; the pages it needs beyond those
    come from ``free[head]``, ``free[head + 1]``, ... and are entered into ``block_table`` in place. ``tokens`` is the
    step's number of token rows (the sum of ``new``, or more where a batch is padded). ``free`` and ``head`` are not
    changed: pass ``Plan.head`` on to the next step. A token that finds no page, or no column in its table row, gets slot
    -1 (and LQ_DEV_BOUNDS)."""
    return Plan(*ext().plan(cached, new, block_table, free, head, page_size, tokens))


def append(q: Optional[torch.Tensor], k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor,
           keys: Sequence[torch.Tensor], values: Sequence[torch.Tensor], positions: Optional[torch.Tensor] = None,
           cos: Optional[torch.Tensor] = None, sin: Optional[torch.Tensor] = None, axes: Optional[torch.Tensor] = None,
           interleaved: bool = False) -> Optional[torch.Tensor]:
    """Store a step's ``k`` and ``v`` (N, KVH, D) at ``slots`` (N,) int32 (negative: nothing is stored), in 4 bits, and
    return ``q`` (N, H, D) rotated; ``q`` and ``k`` are rotated as by ``rotary.rotate`` where ``positions`` are given, the
    keys quantized from their rotated 32-bit values. One launch; the cache is changed in place."""
    return ext().append(q, k, v, slots, keys, values, positions, cos, sin, axes, interleaved)


def read(keys: Sequence[torch.Tensor], values: Sequence[torch.Tensor],
         slots: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """The keys and values that the cache holds at ``slots`` (N,), (N, KVH, D) each in the scales' dtype (zeros for a
    negative slot): what ``kernels.dequantize`` makes of those rows."""
    return ext().read(keys, values, slots)


def attend(q: torch.Tensor, keys: Sequence[torch.Tensor], values: Sequence[torch.Tensor], block_table: torch.Tensor,
           lens: torch.Tensor, scale: float, q_start: Optional[torch.Tensor] = None, max_q: int = 1,
           sinks: Optional[torch.Tensor] = None, window: int = 0) -> torch.Tensor:
    """Attention of a step's queries over the pages: ``q`` (N, H, D), request b's queries being rows ``q_start[b]`` to
    ``q_start[b + 1]`` - 1 (None: row b, one each), at most ``max_q`` of them (of more, the first ``max_q`` are answered, and
    LQ_DEV_BOUNDS is set); they are the last of its ``lens[b]`` tokens, whose keys and values are already in the cache, in the pages of ``block_table[b]``. A query sees the keys up to its
    own position, the last ``window`` of them when that is not 0. ``sinks`` (H,) float32 logits join the softmax's sum.
    Returns (N, H, D) in q's dtype: 0 where a query sees nothing, and in rows that are no answered query's."""
    return ext().attend(q, keys, values, block_table, lens, scale, q_start, max_q, sinks, window)
