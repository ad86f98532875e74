"""The ring of a product that makes its activations' pieces itself (fp4_gemm.cu), modelled on the CPU: converter warps take
stages in turn and wait, by parity, for a stage's place to be free. A parity wait also passes two rounds early, so no warp may
come to its next stage before the place of the stage two rounds back was handed over."""

import random

import pytest


def _run(places, turns, stages, seed):
    """One random schedule of `turns` warps and the MMA issuer: "ok", or what went wrong."""
    rng = random.Random(seed)
    freed = [0] * places  # completed phases of each place's barrier
    following = list(range(turns))  # each warp's next stage
    made, used = set(), 0
    while used < stages:
        moves = []
        for w, x in enumerate(following):
            if x < stages:
                place, turn = x % places, x // places
                if turn == 0 or freed[place] % 2 != (turn - 1) % 2:  # the wait for phase turn - 1 passes
                    moves.append((w, x, place, turn))
        if used in made:
            moves.append(None)
        if not moves:
            return "deadlock"
        m = rng.choice(moves)
        if m is None:
            freed[used % places] += 1
            used += 1
        else:
            w, x, place, turn = m
            if freed[place] < turn:
                return "overrun"
            made.add(x)
            following[w] = x + turns
    return "ok"


@pytest.mark.parametrize("places", [2, 3, 4, 5, 7, 10])
def test_no_more_warps_than_places_never_overrun(places):
    turns = min(4, places)  # as the kernel has it
    assert {_run(places, turns, 50, s) for s in range(400)} == {"ok"}


def test_more_warps_than_places_would(places=3):
    assert "overrun" in {_run(places, 4, 50, s) for s in range(400)}
