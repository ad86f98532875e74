"""Microscaled 4-bit floating point on the CPU: the layout of operands, and what is refused before any launch."""

import ctypes

import pytest
import torch

from locals_b200 import _lib, fp4
from tests import fp4_reference as R


def _mlx(rows, K, mode, stack=None, seed=0):
    g = torch.Generator().manual_seed(seed)
    lead = () if stack is None else (stack,)
    codes = torch.randint(-2 ** 31, 2 ** 31, (*lead, rows, K // 8), generator=g, dtype=torch.int64).to(torch.int32)
    scales = torch.randint(0, 127, (*lead, rows, K // R.GROUP[mode]), generator=g).to(torch.uint8)
    return codes, scales


@pytest.mark.parametrize("mode", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("rows,K,stack", [(1, 32, None), (128, 128, None), (130, 96, None), (257, 2880, None), (5, 160, 3), (129, 64, 2)])
def test_pack_lays_out_tiles_and_unpack_takes_them_back(mode, rows, K, stack):
    codes, scales = _mlx(rows, K, mode, stack)
    a = fp4.pack(codes, scales, mode)
    Kp = -(-K // 128) * 128
    assert a.K == K and a.rows == rows and a.codes.shape[-1] == Kp // 8
    assert torch.equal(a.codes[..., :K // 8], codes) and not a.codes[..., K // 8:].any()
    want = R.tile(scales)
    assert a.tiles.shape[-2] == Kp // (4 * R.GROUP[mode])
    assert torch.equal(a.tiles[..., :want.shape[-2], :], want) and not a.tiles[..., want.shape[-2]:, :].any()
    back = fp4.unpack(a)
    assert torch.equal(back[0], codes) and torch.equal(back[1], scales)


def test_interleave_puts_gate_and_up_rows_in_turn():
    gate, up = _mlx(70, 96, "mxfp4", 2, 1), _mlx(70, 96, "mxfp4", 2, 2)
    codes, scales = fp4.unpack(fp4.interleave(gate, up))
    for got, g, u in ((codes, gate[0], up[0]), (scales, gate[1], up[1])):
        assert torch.equal(got[:, 0::2], g) and torch.equal(got[:, 1::2], u)


@pytest.mark.parametrize("call", [
    lambda c, s: fp4.pack(c, s[:, :-1]),                                   # scales that do not fit
    lambda c, s: fp4.pack(c[:, :-1], s),                                   # no whole groups
    lambda c, s: fp4.pack(c, s, "int4"),                                   # another format
    lambda c, s: fp4.pack(c, s, "nvfp4"),                                  # groups of another size
    lambda c, s: fp4.pack(c, s, "mxfp4", torch.ones(1)),                   # mxfp4 has no factor
    lambda c, s: fp4.interleave((c, s), (c[:1], s[:1])),                   # gate and up differ
    lambda c, s: fp4.quantize(torch.zeros(4, 64), "mxfp4"),                # not on a GPU
    lambda c, s: fp4.quantize(torch.zeros(4, 64), "fp4"),
    lambda c, s: fp4.dequantize(fp4.pack(c, s)),
    lambda c, s: fp4.matmul(torch.zeros(4, 64, dtype=torch.float16), fp4.pack(c, s)),
    lambda c, s: fp4.matmul(fp4.pack(c, s), fp4.pack(c, s)),
    lambda c, s: fp4.experts(torch.zeros(4, 64, dtype=torch.float16), torch.zeros(4, 2, dtype=torch.int32), torch.ones(4, 2),
                             fp4.pack(c[None], s[None]), fp4.pack(c[None], s[None])),
])
def test_refusals_of_values(call):
    with pytest.raises(ValueError):
        call(*_mlx(8, 64, "mxfp4"))


@pytest.mark.parametrize("call", [
    lambda c, s: fp4.pack(c.float(), s),
    lambda c, s: fp4.pack(c, s.int()),
    lambda c, s: fp4.quantize(torch.zeros(4, 64, dtype=torch.float64), "mxfp4"),
    lambda c, s: fp4.matmul(torch.zeros(4, 64, dtype=torch.float16), fp4.pack(c, s), dtype=torch.float32),
])
def test_refusals_of_types(call):
    with pytest.raises(TypeError):
        call(*_mlx(8, 64, "mxfp4"))


OK, BAD = ctypes.c_void_p(4096), ctypes.c_void_p(4098)  # never dereferenced: argument checks come first


def test_abi_refusals():
    L = _lib.lib()
    E = _lib
    q = lambda x=OK, dt=E.BF16, row=64, rows=4, K=64, mode=E.MXFP4, f=None, c=OK, t=OK: L.lq_fp4_quantize(x, dt, row, rows, K, mode, f, c, t, None)  # noqa: E731
    assert q(x=None) == E.LQ_E_ARG and q(c=None) == E.LQ_E_ARG and q(dt=7) == E.LQ_E_ARG and q(f=OK) == E.LQ_E_ARG
    assert q(mode=2) == E.LQ_E_UNSUPPORTED
    assert q(rows=0) == E.LQ_E_SHAPE and q(K=0) == E.LQ_E_SHAPE and q(row=63) == E.LQ_E_SHAPE and q(rows=(1 << 29) + 1) == E.LQ_E_SHAPE
    assert q(c=BAD) == E.LQ_E_ALIGN and q(t=BAD) == E.LQ_E_ALIGN and q(dt=E.F32, x=BAD) == E.LQ_E_ALIGN
    d = lambda stack=1, rows=4, K=64, mode=E.MXFP4, dt=E.F32, c=OK: L.lq_fp4_dequantize(c, OK, stack, rows, K, mode, None, dt, OK, None)  # noqa: E731
    assert d(c=None) == E.LQ_E_ARG and d(stack=0) == E.LQ_E_SHAPE and d(mode=5) == E.LQ_E_UNSUPPORTED and d(c=BAD) == E.LQ_E_ALIGN
    m = lambda x=OK, M=4, N=6, K=64, mode=E.NVFP4, glu=0, dt=E.BF16, y=OK: L.lq_fp4_qmm(x, OK, None, OK, OK, None, M, N, K, mode, glu, dt, y, None)  # noqa: E731
    assert m(x=None) == E.LQ_E_ARG and m(dt=9) == E.LQ_E_ARG and m(M=0) == E.LQ_E_SHAPE and m(N=0) == E.LQ_E_SHAPE
    assert m(N=7, glu=1) == E.LQ_E_SHAPE and m(mode=-1) == E.LQ_E_UNSUPPORTED and m(x=BAD) == E.LQ_E_ALIGN
    n = L.lq_fp4_linear_workspace(100, 6, 64, E.BF16)
    assert n > 0 and L.lq_fp4_linear_workspace(4, 6, 64, E.BF16) == 0 and L.lq_fp4_linear_workspace(100, 6, 64, E.F32) == 0 and L.lq_fp4_linear_workspace(0, 6, 64, E.BF16) == 0
    li = lambda x=OK, row=64, M=100, dt=E.BF16, ws=OK, b=n: L.lq_fp4_linear(x, row, OK, OK, M, 6, 64, 0, dt, OK, ws, b, None)  # noqa: E731
    assert li(x=None) == E.LQ_E_ARG and li(dt=E.F32) == E.LQ_E_ARG and li(ws=None) == E.LQ_E_ARG
    assert li(b=n - 1) == E.LQ_E_SHAPE and li(row=60) == E.LQ_E_SHAPE and li(ws=BAD) == E.LQ_E_ALIGN
    n = L.lq_fp4_experts_workspace(800, 400, 8, 6, 64, E.BF16)
    assert n > 0 and L.lq_fp4_experts_workspace(8, 4, 16, 6, 64, E.BF16) == 0
    ex = lambda order=None, k=0, rows=800, st=OK, ns=OK, P=800, E_=8, b=n: L.lq_fp4_experts(OK, rows, order, k, st, OK, ns, P, 400, 0, OK, OK, OK, E_, 6, 64, E.BF16, OK, b, None)  # noqa: E731
    assert ex(order=OK) == E.LQ_E_ARG and ex(k=-1) == E.LQ_E_ARG and ex(st=None) == E.LQ_E_ARG
    assert ex(rows=799) == E.LQ_E_SHAPE and ex(k=2, rows=399) == E.LQ_E_SHAPE and ex(b=n - 1) == E.LQ_E_SHAPE and ex(E_=0) == E.LQ_E_SHAPE
    assert ex(P=4096, E_=2000, rows=4096, b=1 << 40) == E.LQ_E_SHAPE  # more than 1024 segments
