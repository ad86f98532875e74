"""How the many-row attention kernel ends after a wait that gave up: a model of its roles' waits and barriers, on the CPU.

Each role is a coroutine that yields the condition it stands at. A wait on an mbarrier may give up, at any place, and sets
`abort`; from then on no wait is taken, and every role has to come to its end. A barrier that counts warps has no limit: a
role that leaves while another goes on to the barrier hangs the kernel. The model follows locals_b200/csrc/kv4_prefill.cu:
the page warp (a step's runs into one of four slots), the unpacking warps (a step's loads one step ahead, their largest
values put together at a barrier, tiles into one of two buffers) and a consumer that frees the buffers.
"""

import random

import pytest

WARPS, SLOTS = 8, 4


class Kernel:
    def __init__(self, steps, rng, give_up, agree):
        self.steps, self.rng, self.give_up, self.agree = steps, rng, give_up, agree
        self.abort = False
        self.left = [None] * SLOTS
        self.top = [[0] * WARPS for _ in range(2)]
        self.told, self.taken, self.full, self.freed = 0, [0] * WARPS, [0] * WARPS, 0
        self.arrived, self.passed = 0, 0

    def wait(self, ready):
        """A bounded wait: nothing once abort is set; it may run out before what it waits for has come."""
        while not self.abort and not ready():
            if self.rng.random() < self.give_up:
                self.abort = True
                return
            yield lambda: self.abort or ready() or self.give_up > 0

    def barrier(self):
        """A barrier of the unpacking warps: no limit."""
        turn = self.passed
        self.arrived += 1
        if self.arrived == WARPS:
            self.arrived, self.passed = 0, turn + 1
        yield lambda: self.passed > turn

    def page(self):
        it = 0
        for it in range(self.steps):
            yield from self.wait(lambda: min(self.taken) >= it - SLOTS + 1)
            self.left[it % SLOTS] = 1
            self.told = it + 1
            yield None
            if self.abort and self.agree and self.rng.random() < 0.1:  # (at an item's start)
                break
        yield from self.wait(lambda: min(self.taken) >= self.steps - SLOTS + 1)
        self.left[self.steps % SLOTS] = 0
        self.told = self.steps + 1

    def fetch(self, asked):
        yield from self.wait(lambda: self.told > asked)
        return not (self.left[asked % SLOTS] == 0 or self.abort)

    def unpack(self, w):
        if self.agree:
            have, asked, it = (yield from self.fetch(0)), 1, 0
            while True:
                ahead = have and (yield from self.fetch(asked))
                asked += ahead
                self.top[it & 1][w] = 1 if have else -1
                yield from self.barrier()
                yield None
                if min(self.top[it & 1]) < 0:
                    return
                yield from self.tiles(w, it)
                have, it = ahead, it + 1
        have, asked, it = (yield from self.fetch(0)), 1, 0  # each warp by what it saw itself
        while have:
            ahead = yield from self.fetch(asked)
            asked += ahead
            yield from self.barrier()
            yield from self.tiles(w, it)
            have, it = ahead, it + 1

    def tiles(self, w, it):
        self.taken[w] = it + 1
        yield from self.wait(lambda: self.freed >= it - 1)
        yield None
        self.full[w] = it + 1

    def consume(self):
        for it in range(self.steps):
            yield from self.wait(lambda: min(self.full) > it)
            if self.abort:
                return
            self.freed = it + 1
            yield None

    def run(self):
        """True when every role came to its end."""
        roles = {r: None for r in [self.page(), self.consume(), *(self.unpack(w) for w in range(WARPS))]}
        while roles:
            able = [r for r, at in roles.items() if at is None or at()]
            if not able:
                return False
            r = self.rng.choice(able)
            try:
                roles[r] = next(r)
            except StopIteration:
                del roles[r]
        return True


@pytest.mark.parametrize("steps", [1, 2, 5, 9])
def test_roles_end_without_an_error(steps):
    for seed in range(50):
        k = Kernel(steps, random.Random(seed), 0.0, agree=True)
        assert k.run() and not k.abort and k.full == [steps] * WARPS


@pytest.mark.parametrize("steps", [1, 2, 5, 9])
def test_roles_end_after_any_wait_gave_up(steps):
    gave_up = 0
    for seed in range(400):
        k = Kernel(steps, random.Random(seed), 0.02, agree=True)
        assert k.run(), seed
        gave_up += k.abort
    assert gave_up > 40


def test_the_model_finds_warps_that_leave_by_themselves():
    """Without the word that all warps read after a barrier, some leave while others go on to it."""
    ends = [Kernel(5, random.Random(seed), 0.02, agree=False).run() for seed in range(400)]
    assert not all(ends)
