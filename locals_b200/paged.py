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

import functools
from typing import NamedTuple, Optional, Sequence, Tuple

import torch

from . import rotary
from ._lib import call, lib
from .kernels import _stream, dtype_code

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


def _ints(*ts: torch.Tensor) -> None:
    for t in ts:
        if t.dtype != torch.int32 or not t.is_contiguous() or not t.is_cuda or \
                t.get_device() != torch._C._cuda_getDevice():
            raise ValueError("lengths, tables, page lists and slots are contiguous int32 tensors of the current GPU")


def _pool(keys: Sequence[torch.Tensor], values: Sequence[torch.Tensor], dtype: torch.dtype):
    """(pages, KVH, page_size, head_dim) of a checked pool on the current device, and its six addresses."""
    kq, ks, kb = keys
    vq, vs, vb = values
    shape, small = kq.shape, ks.shape
    if len(shape) != 4 or kq.dtype != torch.int32 or vq.dtype != torch.int32:
        raise ValueError("words: int32 (pages, KVH, page_size, head_dim / 8) expected")
    pages, KVH, page, words = shape
    if vq.shape != shape or small != (pages, KVH, page, words * 8 // GROUP) or kb.shape != small or \
            vs.shape != small or vb.shape != small:
        raise ValueError(f"keys and values are not 4-bit triples of one pool: words {tuple(shape)}, scales "
                         f"{tuple(small)}")
    if not (ks.dtype == kb.dtype == vs.dtype == vb.dtype == dtype):
        raise TypeError("scales and biases must have the queries' dtype")
    d = torch._C._cuda_getDevice()
    if not (kq.get_device() == ks.get_device() == kb.get_device() == vq.get_device() == vs.get_device()
            == vb.get_device() == d):
        raise ValueError("the cache must be on the queries' device, the current one")
    if not (kq.is_contiguous() and ks.is_contiguous() and kb.is_contiguous() and vq.is_contiguous()
            and vs.is_contiguous() and vb.is_contiguous()):
        raise ValueError("the cache must be contiguous")
    return pages, KVH, page, words * 8, (kq.data_ptr(), ks.data_ptr(), kb.data_ptr(), vq.data_ptr(), vs.data_ptr(),
                                         vb.data_ptr())


@functools.lru_cache(maxsize=1024)
def _attend_workspace(device: int, B: int, max_q: int, H: int, KVH: int, D: int, width: int, page: int) -> int:
    return int(lib().lq_kv4_attend_workspace(B, max_q, H, KVH, D, width, page))


def plan(cached: torch.Tensor, new: torch.Tensor, block_table: torch.Tensor, free: torch.Tensor, head: torch.Tensor,
         page_size: int, tokens: int) -> Plan:
    """The block tables and slot maps of a step, built on the GPU in one launch: request b holds ``cached[b]`` tokens, in
    the pages that the first entries of ``block_table[b]`` name, and brings ``new[b]``; the pages it needs beyond those
    come from ``free[head]``, ``free[head + 1]``, ... and are entered into ``block_table`` in place. ``tokens`` is the
    step's number of token rows (the sum of ``new``, or more where a batch is padded). ``free`` and ``head`` are not
    changed: pass ``Plan.head`` on to the next step. A token that finds no page, or no column in its table row, gets slot
    -1 (and LQ_DEV_BOUNDS)."""
    _ints(cached, new, block_table, free, head)
    B = cached.shape[0]
    if cached.shape != new.shape or cached.dim() != 1 or block_table.dim() != 2 or block_table.shape[0] != B:
        raise ValueError("plan: cached (B,), new (B,), block_table (B, width)")
    n, B1 = int(tokens), B + 1
    if n < 0:
        raise ValueError("plan: tokens must not be negative")
    buf = cached.new_empty(B + B1 + 2 * n + 1)
    p = buf.data_ptr()
    call("lq_page_plan", cached.data_ptr(), new.data_ptr(), B, block_table.data_ptr(), block_table.shape[1],
         free.data_ptr(), free.shape[0], head.data_ptr(), int(page_size), n, p, p + 4 * B, p + 4 * (B + B1),
         p + 4 * (B + B1 + n), p + 4 * (B + B1 + 2 * n), _stream())
    return Plan(*buf.split_with_sizes((B, B1, n, n, 1)))


def append(q: Optional[torch.Tensor], k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor,
           keys: Sequence[torch.Tensor], values: Sequence[torch.Tensor], positions: Optional[torch.Tensor] = None,
           cos: Optional[torch.Tensor] = None, sin: Optional[torch.Tensor] = None, axes: Optional[torch.Tensor] = None,
           interleaved: bool = False) -> Optional[torch.Tensor]:
    """Store a step's ``k`` and ``v`` (N, KVH, D) at ``slots`` (N,) int32 (negative: nothing is stored), in 4 bits, and
    return ``q`` (N, H, D) rotated; ``q`` and ``k`` are rotated as by ``rotary.rotate`` where ``positions`` are given, the
    keys quantized from their rotated 32-bit values. One launch; the cache is changed in place."""
    k, k_row = rotary._rows(k, "k")
    v, v_row = rotary._rows(v, "v")
    N, KVH, D = k.shape
    pages, pool_kvh, page, pool_d, ptrs = _pool(keys, values, k.dtype)
    if v.shape != k.shape or v.dtype != k.dtype or (KVH, D) != (pool_kvh, pool_d):
        raise ValueError(f"append: k {tuple(k.shape)}, v {tuple(v.shape)} do not fit a cache of {pool_kvh} heads of "
                         f"{pool_d}")
    _ints(slots)
    if slots.shape != (N,):
        raise ValueError(f"append: slots ({N},) expected")
    H, q_row, qo = 0, 0, None
    if q is not None:
        q, q_row = rotary._rows(q, "q")
        H = q.shape[1]
        if q.shape[0] != N or q.shape[2] != D or q.dtype != k.dtype:
            raise ValueError("append: q and k must have the same tokens, head_dim and dtype")
        qo = rotary._like(q)
    rot, naxes, max_pos = 0, 1, 1
    if positions is not None:
        if cos is None or sin is None:
            raise ValueError("append: positions without cos and sin tables")
        rot, naxes = rotary._angles(positions, cos, sin, axes, N, D)
        max_pos = cos.shape[0]
    if N:
        call("lq_kv4_append", None if q is None else q.data_ptr(), q_row, None if q is None else qo.data_ptr(), H,
             k.data_ptr(), k_row, v.data_ptr(), v_row, KVH, N, D, rot,
             None if positions is None else positions.data_ptr(), None if positions is None else cos.data_ptr(),
             None if positions is None else sin.data_ptr(), max_pos, None if axes is None else axes.data_ptr(), naxes,
             int(interleaved), slots.data_ptr(), *ptrs, pages, page, dtype_code(k.dtype), _stream())
    return qo


def read(keys: Sequence[torch.Tensor], values: Sequence[torch.Tensor],
         slots: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """The keys and values that the cache holds at ``slots`` (N,), (N, KVH, D) each in the scales' dtype (zeros for a
    negative slot): what ``kernels.dequantize`` makes of those rows."""
    _ints(slots)
    dtype = keys[1].dtype
    pages, KVH, page, D, ptrs = _pool(keys, values, dtype)
    if slots.dim() != 1:
        raise ValueError("read: slots (N,) expected")
    N = slots.shape[0]
    ko = keys[1].new_empty((N, KVH, D))
    vo = torch.empty_like(ko)
    if N:
        call("lq_kv4_read", *ptrs, pages, page, KVH, D, slots.data_ptr(), N, ko.data_ptr(), vo.data_ptr(),
             dtype_code(dtype), _stream())
    return ko, vo


def attend(q: torch.Tensor, keys: Sequence[torch.Tensor], values: Sequence[torch.Tensor], block_table: torch.Tensor,
           lens: torch.Tensor, scale: float, q_start: Optional[torch.Tensor] = None, max_q: int = 1,
           sinks: Optional[torch.Tensor] = None, window: int = 0) -> torch.Tensor:
    """Attention of a step's queries over the pages: ``q`` (N, H, D), request b's queries being rows ``q_start[b]`` to
    ``q_start[b + 1]`` - 1 (None: row b, one each), at most ``max_q`` of them; they are the last of its ``lens[b]`` tokens,
    whose keys and values are already in the cache, in the pages of ``block_table[b]``. A query sees the keys up to its
    own position, the last ``window`` of them when that is not 0. ``sinks`` (H,) float32 logits join the softmax's sum.
    Returns (N, H, D) in q's dtype: 0 where a query sees nothing, and in rows past ``q_start[-1]``."""
    q, q_row = rotary._rows(q, "q")
    N, H, D = q.shape
    if q_row != H * D:
        q = q.contiguous()
    pages, KVH, page, pool_d, ptrs = _pool(keys, values, q.dtype)
    _ints(block_table, lens)
    B, table = lens.shape[0], block_table.shape
    if D != pool_d or H % KVH:
        raise ValueError(f"attend: {H} heads of {D} against a cache of {KVH} heads of {pool_d}")
    if lens.dim() != 1 or len(table) != 2 or table[0] != B:
        raise ValueError("attend: lens (B,), block_table (B, width)")
    max_q = int(max_q)
    if q_start is None:
        if N != B or max_q != 1:
            raise ValueError("attend: without q_start there is one query a request")
    else:
        _ints(q_start)
        if q_start.shape != (B + 1,):
            raise ValueError(f"attend: q_start ({B + 1},) expected")
    if sinks is not None:
        if sinks.dtype != torch.float32 or sinks.get_device() != q.get_device() or not sinks.is_contiguous():
            sinks = sinks.to(device=q.device, dtype=torch.float32).contiguous()
        if sinks.shape != (H,):
            raise ValueError(f"attend: sinks ({H},) expected")
    out = torch.empty_like(q)
    if N == 0:
        return out
    nbytes = _attend_workspace(q.get_device(), B, max_q, H, KVH, D, table[1], page)
    ws = q.new_empty(nbytes // 2) if nbytes else None
    call("lq_kv4_attend", q.data_ptr(), N, None if q_start is None else q_start.data_ptr(), max_q, *ptrs, pages, page,
         block_table.data_ptr(), table[1], lens.data_ptr(), B, None if sinks is None else sinks.data_ptr(), float(scale),
         int(window), H, KVH, D, dtype_code(q.dtype), None if ws is None else ws.data_ptr(), nbytes, out.data_ptr(),
         _stream())
    return out
