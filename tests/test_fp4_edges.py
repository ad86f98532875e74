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
                (1 << 20, 1 << 10, 4, 64, 96, E.BF16), (2, 2, 8193, 64, 96, E.BF16)):
        assert L.lq_fp4_moe_workspace(*bad) == 0, bad
    for good in ((1, 1024, 4, 64, 96, E.BF16), (2, 2, 8192, 64, 96, E.BF16), (1, 2, 9000, 64, 96, E.BF16), (600, 2, 1024, 64, 96, E.F16), (2, 2, 5000, 64, 96, E.BF16)):
        assert L.lq_fp4_moe_workspace(*good) > 0, good

    def moe(x=OK, inds=OK, w=OK, c=OK, t=OK, y=OK, T=5, k=2, e=4, dt=E.BF16, ws=OK, b=n):
        return L.lq_fp4_moe(x, inds, w, c, t, OK, OK, y, T, k, e, 64, 96, dt, ws, b, None)

    for a in ({"x": None}, {"inds": None}, {"w": None}, {"c": None}, {"t": None}, {"y": None}, {"ws": None}, {"dt": E.F32}):
        assert moe(**a) == E.LQ_E_ARG, a
    for a in ({"T": 0}, {"k": 0}, {"e": 0}, {"b": n - 1}, {"T": 600, "e": 2000, "b": 1 << 40}, {"T": 2, "e": 9000, "b": 1 << 40}):
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


class _Barrier:
    """An mbarrier: arrivals and bytes outstanding; a phase is over when both are none."""

    def __init__(self, count):
        self.count, self.pending, self.tx, self.phase = count, count, 0, 0

    def arrive(self, expect=0):
        self.tx += expect
        self.pending -= 1
        self._over()

    def bytes(self, n):
        self.tx -= n
        self._over()

    def _over(self):
        assert self.pending >= 0
        if self.pending == 0 and self.tx == 0:
            self.phase += 1
            self.pending = self.count

    def passes(self, parity):  # a parity wait: the phase of that parity is the last one that is over
        return self.phase % 2 != parity


def _ring(ctas, places, stages, seed):
    """The wide products' ring of stages: in each CTA a warp for codes and one for scales load a stage's bytes once its place is
    free there, all of a pair's on the lower rank's barrier, for which one thread says what arrives; the issuer takes a stage when it
    is full, and its commit frees the place in each CTA. Loads land and commits arrive at any time. "ok", or what went wrong."""
    rng = random.Random(seed)
    full = [_Barrier(1) for _ in range(places)]
    empty = [[_Barrier(1) for _ in range(places)] for _ in range(ctas)]
    following = {(c, what): 0 for c in range(ctas) for what in ("codes", "scales")}
    flying, held, commits, used = [], {}, [], 0
    while used < stages or commits:
        moves = [("land", i) for i in range(len(flying))]
        if commits:
            moves.append(("commit", 0))
        for key, x in following.items():
            place, turn = x % places, x // places
            if x < stages and (turn == 0 or empty[key[0]][place].passes((turn - 1) % 2)):
                moves.append(("load", key))
        # (the scales' two places of tensor memory: the stage before last is done)
        done = used < 2 or empty[0][(used - 2) % places].passes((used - 2) // places % 2)
        if used < stages and done and full[used % places].passes(used // places % 2):
            moves.append(("issue", 0))
        if not moves:
            return "deadlock"
        kind, at = rng.choice(moves)
        if kind == "load":
            x = following[at]
            following[at] += 1
            if at == (0, "codes"):  # what arrives in all CTAs, of both warps
                full[x % places].arrive(expect=2 * ctas)
            flying.append((at, x))
        elif kind == "land":
            key, x = flying.pop(at)
            if held.get((key, x % places), -1) >= 0:
                return "overrun"
            held[(key, x % places)] = x
            full[x % places].bytes(1)
        elif kind == "issue":
            for key in following:
                if held.get((key, used % places), -1) != used:
                    return "not there"
            commits.append(used)
            used += 1
        else:  # commits arrive in order
            x = commits.pop(0)
            for key in following:
                held[(key, x % places)] = -1
            for c in range(ctas):
                empty[c][x % places].arrive()
    return "ok"


@pytest.mark.parametrize("ctas", [1, 2])
@pytest.mark.parametrize("places", [2, 3, 4, 5])
def test_the_ring_of_a_pair_never_overruns(ctas, places):
    assert {_ring(ctas, places, 30, s) for s in range(150)} == {"ok"}


def _accumulators(columns, warps, tiles, seed, first_half=True):
    """Two accumulators of `columns`: of 256 they share 128, which the writing-out warps read first, and free for the next tile; of 128
    or less they lie side by side, each freed when it is read. The issuer writes a tile's columns, warps read them."""
    rng = random.Random(seed)
    shared = columns == 256
    step = 128 if shared else columns
    full, empty = [_Barrier(1) for _ in range(2)], [_Barrier(warps) for _ in range(2)]
    owner, read = {}, {}  # a column's tile; how often a tile's column was read
    issued, at = 0, [(0, 0)] * warps  # a warp's tile and half
    while any(j < tiles for j, _ in at):
        moves = []
        j = issued
        if shared:
            ready = j < 1 or empty[0].passes((j - 1) % 2)
        else:
            ready = j < 2 or empty[j % 2].passes((j // 2 - 1) % 2)
        if j < tiles and ready:
            moves.append(None)
        moves += [w for w, (k, half) in enumerate(at) if k < tiles and (half or full[k % 2].passes(k // 2 % 2))]
        if not moves:
            return "deadlock"
        w = rng.choice(moves)
        if w is None:
            for c in range(j % 2 * step, j % 2 * step + columns):
                if c in owner and read.get((owner[c], c), 0) < warps:
                    return "overwritten"
                owner[c] = j
            full[j % 2].arrive()
            issued += 1
        else:
            k, half = at[w]
            n = columns // 2
            lo = k % 2 * step + n * ((half + k % 2 + first_half) % 2 if shared else half)
            for c in range(lo, lo + n):
                if owner[c] != k:
                    return "stale"
                read[(k, c)] = read.get((k, c), 0) + 1
            if half == (0 if shared else 1):
                empty[0 if shared else k % 2].arrive()
            at[w] = (k + half, 1 - half)
    return "ok"


@pytest.mark.parametrize("columns", [256, 128])
@pytest.mark.parametrize("warps", [2, 8, 16])
def test_an_accumulator_is_read_before_the_next_tile_writes_it(columns, warps):
    assert {_accumulators(columns, warps, 12, s) for s in range(60)} == {"ok"}


def test_the_other_half_first_would_be_overwritten():
    assert {"overwritten", "stale"} & {_accumulators(256, 8, 12, s, first_half=False) for s in range(60)}


def _product_bytes(rows, N, K, pieces, segments, max_rows):
    """What a grouped product with pieces takes, by its rules for tiles."""
    average = rows // segments
    want = min(2 * average, max_rows)
    if want <= 128:
        tokens = next(t for t in (16, 32, 64, 128) if want <= t)
    else:
        narrow, wide = -(-want // 128) * 128, -(-want // 256) * 256
        tokens = 256 if wide * 8 <= narrow * 9 and average >= 1024 else 128
    tiles, Kp = rows // tokens + segments, -(-K // 128) * 128
    if tokens <= 32 and tiles * -(-N // 128) <= 2 * 148:
        return 0
    blocks = 1 if tokens <= 32 else pieces * -(-tokens // 128)
    return -(-pieces * rows * Kp // 512) * 512 + tiles * (Kp // 128) * blocks * 512


def test_the_workspace_of_routed_experts_holds_what_its_products_take():
    """Their tiles go by the number of segments: sized for one more than they run with (17 rows a segment or 13), they wrote past its
    end."""
    L, rng = _lib.lib(), random.Random(0)
    cases = [(34, 2, 4, 256, 96), (17, 1, 1, 128, 64), (2, 17, 2, 128, 64)]
    cases += [(rng.choice([1, 2, 3, rng.randint(2, 60), rng.randint(2, 3000)]), rng.randint(1, 9), rng.choice([1, 2, 3, 4, 8, 60, 64, 128, 1000]),
               rng.randint(1, 3000), rng.randint(1, 1500)) for _ in range(4000)]
    for T, k, E, D, I in cases:
        P = T * k
        segments = min(E, P) if T > 1 else P
        for dtype, pieces in ((_lib.BF16, 2), (_lib.F16, 3)):
            n = L.lq_fp4_moe_workspace(T, k, E, D, I, dtype)
            if segments > 1024:
                assert n == 0
                continue
            ints = (2 * P + 2 * segments + 2) * 4 if T > 1 else 0
            product = max(_product_bytes(P, 2 * I, D, pieces, segments, T), _product_bytes(P, D, I, 3, segments, T))
            assert n >= 4 * P * (D + I) + ints + product, (T, k, E, D, I)
