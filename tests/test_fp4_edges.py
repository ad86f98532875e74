"""Microscaled 4-bit floating point on the CPU: what the calls of lq_fp4_moe refuse before any launch, and models of what the kernels
write."""

import ctypes
import random

import pytest

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


@pytest.mark.parametrize("P,E,ctas", [(1, 1, 1), (5, 3, 1), (40, 8, 1), (300, 7, 1), (1000, 1, 1), (2049, 5, 8), (2500, 70, 8)])
def test_every_place_that_a_combine_may_read_is_written(P, E, ctas):
    """The grouping's writes, restated: shares of CTAs and warps, ranks in pair order; ids outside [0, E) have pos -1, and order
    ends with -1. Every entry of both is written, once, and a pos is -1 or a row of a segment."""
    rng = random.Random(P)
    ids = [rng.choice([-1, E, -2 ** 31, 2 ** 31 - 1] + list(range(E)) * 2) for _ in range(P)]
    order, pos = {}, {}
    count = [sum(i == e for i in ids) for e in range(E)]
    run = [sum(count[:e]) for e in range(E)]
    share = -(-P // ctas)
    for rank in range(ctas):
        s0 = min(rank * share, P)
        s1 = min(s0 + share, P)
        ch = -(-(s1 - s0) // 32)
        for warp in range(32):
            p0 = min(s0 + warp * ch, s1)
            for p in range(p0, min(p0 + ch, s1)):
                valid = 0 <= ids[p] < E
                j = run[ids[p]] if valid else -1
                if valid:
                    run[ids[p]] += 1
                    assert j not in order
                    order[j] = p
                assert p not in pos
                pos[p] = j
    for j in range(sum(count), P):
        assert j not in order
        order[j] = -1
    assert sorted(order) == list(range(P)) and sorted(pos) == list(range(P))
    assert all(order[j] == p for p, j in pos.items() if j >= 0)
    assert all((j == -1) == (not 0 <= ids[p] < E) for p, j in pos.items())
