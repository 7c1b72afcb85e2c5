"""A model of how the roles of the wide 8-bit product (linear_kernel in
vidax_b200/csrc/fp8_linear.cuh) wait for one another, run under random
schedules in which waits may give up. Checked: every role ends, a named
barrier's generation is made of one arrival of each adding warp for one and the
same block, and a stage's barrier is armed for a load only when the load before
it has landed.

mbarrier waits go by parity. Any of them but the adding warps' for a product may
give up at any time (which raises the abort flag; with the flag up they give up
soon). Loads land and MMAs complete at any later time. The waits for scales and
row maxima hand nothing on that another role's progress needs and are left
out."""
import random

import pytest


class Cta:
    def __init__(self, rng, blocks, bufs, stages, warps, patient, give_up, silent=None):
        assert stages > bufs and bufs % 2 == 0
        self.rng, self.N, self.B, self.S, self.W = rng, blocks, bufs, stages, warps
        self.patient, self.p_give_up = patient, give_up
        self.abort = False
        self.full = [0] * stages          # completed phases
        self.armed = [False] * stages     # a load is on its way
        self.done = [0] * stages
        self.gen = [[] for _ in range(bufs)]  # arrivals of the open generation
        self.gens = [0] * bufs
        self.flight = []                  # loads and MMAs under way
        self.errors = []
        roles = {"load": self.load(), "mma0": self.mma(0), "mma1": self.mma(1)}
        roles.update({f"sum{w}": self.sums(w) for w in range(warps)})
        roles.pop(silent, None)
        self.roles = roles

    def wait(self, phases, i, parity, patient=False):
        """True, or False after it gave up."""
        while True:
            if phases[i] & 1 != parity:
                return True
            if not patient and self.rng.random() < (0.3 if self.abort else self.p_give_up):
                self.abort = True
                return False
            yield

    def arrive(self, b, who):
        self.gen[b].append(who)
        if len(self.gen[b]) == self.W + 1:
            if len({blk for _, blk in self.gen[b]}) != 1 or len({w for w, _ in self.gen[b]}) != self.W + 1:
                self.errors.append(("generation", b, self.gen[b]))
            self.gen[b] = []
            self.gens[b] += 1

    def load(self):
        for n in range(self.N):
            s = n % self.S
            if not (yield from self.wait(self.done, s, (n // self.S) & 1 ^ 1)):
                return
            if self.patient and not (yield from self.wait(self.full, s, (n // self.S) & 1 ^ 1)):
                return
            if self.armed[s]:
                self.errors.append(("armed twice", s, n))
            self.armed[s] = True
            self.flight.append(("load", s))
            yield

    def mma(self, first):
        for i in range(first, self.N + self.B, 2):
            b, s = i % self.B, i % self.S
            if i >= self.B and i - self.B < self.N:
                g = self.gens[b]
                self.arrive(b, ("mma", i - self.B))
                while self.gens[b] == g:
                    yield
            yield
            if i < self.N:
                yield from self.wait(self.full, s, (i // self.S) & 1)
                self.flight.append(("mma", s))
            yield

    def sums(self, w):
        for i in range(self.N):
            b, s = i % self.B, i % self.S
            yield from self.wait(self.done, s, (i // self.S) & 1, self.patient)
            yield
            self.arrive(b, (w, i))
            yield

    def run(self):
        """True if every role ends."""
        idle = 0
        while self.roles and idle < 20000:
            idle += 1
            if self.flight and self.rng.random() < 0.3:
                kind, s = self.flight.pop(self.rng.randrange(len(self.flight)))
                if kind == "load":
                    self.full[s] += 1
                    self.armed[s] = False
                else:
                    self.done[s] += 1
            name = self.rng.choice(list(self.roles))
            before = self.state()
            for _ in range(self.rng.choice((1, 1, 5, 40))):  # some run far ahead
                try:
                    next(self.roles[name])
                except StopIteration:
                    del self.roles[name]
                    idle = 0
                    break
            if self.state() != before:
                idle = 0
        return not self.roles

    def state(self):
        return (tuple(map(len, self.gen)), tuple(self.gens), len(self.flight),
                tuple(self.full), tuple(self.done))


SIZES = [(1, 2, 3), (2, 2, 4), (7, 2, 3), (24, 2, 4), (5, 4, 5), (25, 4, 6), (24, 4, 7)]


@pytest.mark.parametrize("blocks,bufs,stages", SIZES)
def test_no_give_up(blocks, bufs, stages):
    for seed in range(4):
        cta = Cta(random.Random(seed), blocks, bufs, stages, 4, True, 0.0)
        assert cta.run() and not cta.errors and not cta.abort


@pytest.mark.parametrize("blocks,bufs,stages", SIZES)
@pytest.mark.parametrize("give_up,silent", [(0.001, None), (0.02, None), (0.05, "load")])
def test_every_role_ends_after_any_give_up(blocks, bufs, stages, give_up, silent):
    for seed in range(12):
        cta = Cta(random.Random(seed), blocks, bufs, stages, 4, True, give_up, silent)
        assert cta.run(), (seed, cta.state())
        assert not cta.errors, (seed, cta.errors)


def test_the_model_sees_warps_that_run_ahead():
    """Where the adding warps' waits for a product give up too, warps lap one
    another, roles are left waiting and stages are armed twice."""
    stuck, kinds = 0, set()
    for seed in range(20):
        cta = Cta(random.Random(seed), 24, 2, 4, 4, False, 0.02)
        stuck += not cta.run()
        kinds |= {e[0] for e in cta.errors}
    assert stuck and kinds == {"generation", "armed twice"}
