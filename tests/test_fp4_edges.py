"""Microscaled 4-bit floating point on the CPU: what the calls of lq_fp4_moe refuse before any launch."""

import ctypes

from locals_b200 import _lib

OK, BAD = ctypes.c_void_p(4096), ctypes.c_void_p(4098)  # never dereferenced: argument checks come first


def test_moe_refusals():
    L, E = _lib.lib(), _lib
    n = L.lq_fp4_moe_workspace(5, 2, 4, 64, 96, E.BF16)
    # hidden rows and outputs in 32 bits, at least
    assert n >= 5 * 2 * (64 + 96) * 4
    for bad in ((0, 2, 4, 64, 96, E.BF16), (5, 0, 4, 64, 96, E.BF16), (5, 2, 0, 64, 96, E.BF16), (5, 2, 4, 0, 96, E.BF16),
                (5, 2, 4, 64, 0, E.BF16), (5, 2, 4, 64, 96, E.F32), (1, 1025, 4, 64, 96, E.BF16), (600, 2, 1025, 64, 96, E.BF16),
                (1 << 20, 1 << 10, 4, 64, 96, E.BF16)):
        assert L.lq_fp4_moe_workspace(*bad) == 0, bad
    for good in ((1, 1024, 4, 64, 96, E.BF16), (600, 2, 1024, 64, 96, E.F16), (2, 2, 5000, 64, 96, E.BF16)):
        assert L.lq_fp4_moe_workspace(*good) > 0, good

    def moe(x=OK, inds=OK, w=OK, c=OK, t=OK, y=OK, T=5, k=2, e=4, dt=E.BF16, ws=OK, b=n):
        return L.lq_fp4_moe(x, inds, w, c, t, OK, OK, y, T, k, e, 64, 96, dt, ws, b, None)

    for a in ({"x": None}, {"inds": None}, {"w": None}, {"c": None}, {"t": None}, {"y": None}, {"ws": None}, {"dt": E.F32}):
        assert moe(**a) == E.LQ_E_ARG, a
    for a in ({"T": 0}, {"k": 0}, {"e": 0}, {"b": n - 1}, {"T": 600, "e": 2000, "b": 1 << 40}):
        assert moe(**a) == E.LQ_E_SHAPE, a
    for a in ({"c": BAD}, {"t": BAD}, {"ws": BAD}, {"inds": BAD}, {"w": BAD}, {"x": ctypes.c_void_p(4097)}, {"y": ctypes.c_void_p(4097)}):
        assert moe(**a) == E.LQ_E_ALIGN, a
