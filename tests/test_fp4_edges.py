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


def _clusters(needs, frees_before_join, seed):
    """Two clusters of two CTAs, one a SM of 512 columns of tensor memory: each takes `needs` columns of its SM (and waits until it
    has them), works, and waits for the other of its cluster. "ok", or "deadlock", of a random schedule."""
    rng = random.Random(seed)
    free = [512, 512]
    state = {(c, sm): "start" for c in range(2) for sm in range(2)}
    while any(v != "done" for v in state.values()):
        moves = []
        for (c, sm), v in state.items():
            if v == "start" and free[sm] >= needs[c]:
                moves.append((c, sm, "has"))
            elif v == "has":
                moves.append((c, sm, "join"))
            elif v == "join" and state[(c, 1 - sm)] in ("join", "done"):
                moves.append((c, sm, "done"))
        if not moves:
            return "deadlock"
        c, sm, to = rng.choice(moves)
        state[(c, sm)] = to
        if to == "has":
            free[sm] -= needs[c]
        if to == ("join" if frees_before_join[c] else "done"):
            free[sm] += needs[c]
    return "ok"


@pytest.mark.parametrize("needs", [(256, 512), (512, 512), (256, 256), (64, 512)])
@pytest.mark.parametrize("other", [True, False])
def test_tensor_memory_given_back_before_the_join_holds_no_cluster_up(needs, other):
    """The product's clusters (the first), beside a kernel that does the same or holds its own across its join."""
    assert {_clusters(needs, (True, other), s) for s in range(300)} == {"ok"}


def test_tensor_memory_held_across_both_joins_would():
    assert "deadlock" in {_clusters((256, 512), (False, False), s) for s in range(300)}
