"""The waits and arrivals of `tree_pair_kernel` (csrc/tree_pair.cuh), as a model of its roles that runs in any order: every role ends, no wait takes one
phase for another, and nothing is written over before its last reader is through.  No GPU.

A role is a generator that yields what it waits for.  Products are asynchronous: those of one shape are done in the order they were issued in, those of the
two shapes in any, and a commit comes when all before it are done.  A wait passes
where the barrier's parity says so, as on the device; that the phase is the one that was meant is checked beside it."""
import random

import pytest

RING, SCALES = 3, 8           # kPairRing, kPairScales
PER_ROLE = 2                  # warps of a role that arrive one by one (four on the device)


class Barrier:
    def __init__(self, name, count):
        self.name, self.count, self.pending, self.phase = name, count, count, 0

    def arrive(self):
        self.pending -= 1
        assert self.pending >= 0, f"{self.name}: one arrival too many"
        if self.pending == 0:
            self.pending, self.phase = self.count, self.phase + 1


class Pair:
    """One CTA with ``units``: (steps, whether there is a second tile).  ``mistake``: what is left out, to see that the model notices."""

    def __init__(self, units, rng, mistake=None):
        self.units, self.rng, self.mistake = units, rng, mistake
        many = lambda name, count, n=RING: [Barrier(f"{name}{i}", count) for i in range(n)]
        self.k, self.v = many("k", PER_ROLE), many("v", PER_ROLE)
        self.s, self.o, self.p = ([many(f"{name}{x}_", count) for x in range(2)] for name, count in (("s", 1), ("o", 1), ("p", PER_ROLE)))
        self.u, self.w, self.q = Barrier("u", 1), Barrier("w", 4 * PER_ROLE + 2), Barrier("q", PER_ROLE)
        self.scales = 2 if mistake == "two places for exponents" else SCALES
        self.t = many("t", 2 * PER_ROLE, self.scales)
        # what lies where: numbers of units and steps, by the warp that wrote them
        self.info = [None, None]
        self.queries = [[None] * PER_ROLE for _ in range(2)]
        self.stage = {x: [[None] * PER_ROLE for _ in range(RING)] for x in "kv"}
        self.meaning = [[None] * (2 * PER_ROLE) for _ in range(self.scales)]
        self.scores = [[("free",) for _ in range(2)] for _ in range(2)]        # of tile x, place g & 1
        self.weights = [[[None] * PER_ROLE for _ in range(2)] for _ in range(2)]
        self.output = [{"steps": None, "read": [True] * PER_ROLE} for _ in range(2)]
        self.issued = [[], []]                    # products of tile x that are not done or not committed: [shape, what it does, its commit, done]

    def by_step(self, bars, g):
        return bars[g % RING], g // RING

    def get(self, n):
        unit = self.info[n & 1]
        assert unit is not None and unit[0] == n, f"unit {n}: {unit} lies there"
        return unit[1]

    # ---- roles ----------------------------------------------------------------------------------------------------------
    def next_units(self):
        for n, unit in enumerate(self.units):
            if n:
                yield self.w, n - 1
            self.info[n & 1] = n, unit
            self.u.arrive()
            yield None
        n = len(self.units)
        if n:
            yield self.w, n - 1
        self.info[n & 1] = n, None
        self.u.arrive()

    def loader(self, of_k, me):
        step0 = 0
        for n in range(len(self.units) + 1):
            yield self.u, n
            unit = self.get(n)
            if unit is None:
                return
            steps, two = unit
            self.w.arrive()
            yield None
            if of_k:
                if step0 and self.mistake != "queries at once":
                    yield self.by_step(self.s[0], step0 - 1)
                    yield self.by_step(self.s[1], step0 - 1)
                for x in range(2 if two else 1):
                    self.queries[x][me] = n
                    yield None
                self.q.arrive()
                yield None
            left, stored, stages = (self.s, self.k, self.stage["k"]) if of_k else (self.o, self.v, self.stage["v"])
            for j in range(steps):
                g = step0 + j
                if g >= RING:
                    yield self.by_step(left[0], g - RING)
                    if not (of_k and self.mistake == "one tile's scores for both"):
                        yield self.by_step(left[1], g - RING)
                stages[g % RING][me] = g
                self.meaning[g % self.scales][me if of_k else PER_ROLE + me] = g
                self.t[g % self.scales].arrive()
                yield None
                stored[g % RING].arrive()
                yield None
                if j + 2 < steps:                 # (where the step after the next lies)
                    assert self.get(n) == unit
            step0 += steps

    def do_scores(self, x, n, g, on):
        if on:
            assert all(q == n for q in self.queries[x]) and all(i == g for i in self.stage["k"][g % RING]), f"scores of step {g}"
            assert self.scores[x][g & 1] == ("free",), f"scores of step {g}: {self.scores[x][g & 1]} lies there"
            self.scores[x][g & 1] = "scores", g

    def do_output(self, x, g, first, on):
        if on:
            assert self.scores[x][g & 1] == ("scores", g) and all(i == g for i in self.weights[x][g & 1]), f"weights of step {g}"
            assert all(i == g for i in self.stage["v"][g % RING]), f"values of step {g}"
            assert not first or all(self.output[x]["read"]), f"outputs before step {g} are still to be read"
            if first:
                self.output[x]["read"] = [False] * PER_ROLE
            self.output[x]["steps"] = g
            self.scores[x][g & 1] = ("free",)

    def issue(self, x, shape, does, barrier):
        self.issued[x].append([shape, does, barrier, False])

    def may_be_done(self, x):
        """Shapes of which a product is under way."""
        return sorted({shape for shape, _, _, done in self.issued[x] if not done})

    def finish(self, x, shape):
        product = next(p for p in self.issued[x] if p[0] == shape and not p[3])
        product[1]()
        product[3] = True
        while self.issued[x] and self.issued[x][0][3]:
            self.issued[x].pop(0)[2].arrive()

    def products(self, x):
        step0, behind, used, asked = 0, 0, 0, 0

        def scores(n, on):
            nonlocal behind, used, asked
            if behind == 2:
                if self.mistake != "scores over weights":
                    yield self.by_step(self.o[x], used)
                used += 1
            else:
                behind += 1
            g = asked
            asked += 1
            yield self.by_step(self.k, g)
            self.issue(x, "scores", lambda: self.do_scores(x, n, g, on), self.s[x][g % RING])
            yield None

        for n in range(len(self.units) + 1):
            yield self.u, n
            unit = self.get(n)
            if unit is None:
                return
            steps, two = unit
            on = x == 0 or two
            self.w.arrive()
            yield None
            yield self.q, n
            yield from scores(n, on)
            for j in range(steps):
                g = step0 + j
                if j + 1 < steps:
                    yield from scores(n, on)
                yield self.by_step(self.v, g)
                if on or self.mistake != "a tile alone does not wait":
                    yield self.by_step(self.p[x], g)
                self.issue(x, "outputs", lambda g=g, first=j == 0, on=on: self.do_output(x, g, first, on), self.o[x][g % RING])
                yield None
            step0 += steps

    def weighing(self, x, me):
        step0 = 0
        for n in range(len(self.units) + 1):
            yield self.u, n
            unit = self.get(n)
            if unit is None:
                return
            steps, two = unit
            self.w.arrive()
            yield None
            on = x == 0 or two
            for j in range(steps):
                g = step0 + j
                yield self.by_step(self.s[x], g)
                if on:
                    assert self.scores[x][g & 1] == ("scores", g) and self.get(n) == unit
                    yield self.t[g % self.scales], g // self.scales
                    assert all(i == g for i in self.meaning[g % self.scales]), f"exponents of step {g}"
                    yield None
                    if j and self.rng.random() < 0.3:                          # the reference moves
                        yield self.by_step(self.o[x], g - 1)
                        assert self.output[x]["steps"] == g - 1
                    assert all(i == g for i in self.meaning[g % self.scales]), f"exponents of step {g}"
                    self.weights[x][g & 1][me] = g
                self.p[x][g % RING].arrive()
                yield None
            yield self.by_step(self.o[x], step0 + steps - 1)
            if on and self.mistake != "outputs are not read":
                assert self.output[x]["steps"] == step0 + steps - 1
                self.output[x]["read"][me] = True
            step0 += steps

    def run(self):
        roles = {"units": self.next_units(), **{f"products {x}": self.products(x) for x in range(2)}}
        for me in range(PER_ROLE):
            roles.update({f"k {me}": self.loader(True, me), f"v {me}": self.loader(False, me), **{f"weights {x} {me}": self.weighing(x, me) for x in range(2)}})
        wants, rank = dict.fromkeys(roles), {}
        while roles or any(self.issued):
            if not rank or self.rng.random() < 0.05:                           # some are slow for a while
                rank = {name: self.rng.random() ** 3 for name in (*roles, *((x, shape) for x in range(2) for shape in ("scores", "outputs")))}
            ready = [name for name in roles if wants[name] is None or (wants[name][0].phase ^ wants[name][1]) & 1] + [(x, shape) for x in range(2) for shape in self.may_be_done(x)]
            assert ready, {name: (want[0].name, want[0].phase, want[1]) for name, want in wants.items() if name in roles}
            name = max(ready, key=lambda name: rank.get(name, 0) + 0.3 * self.rng.random())
            if isinstance(name, tuple):
                self.finish(*name)
                continue
            if wants[name] is not None:
                assert wants[name][0].phase == wants[name][1] + 1, f"{name} took phase {wants[name][0].phase - 1} of {wants[name][0].name} for {wants[name][1]}"
            try:
                wants[name] = next(roles[name])
            except StopIteration:
                del roles[name]


def _units(rng):
    return [(rng.choice([1, 1, 2, 3, 4, 5, 7, 9]), rng.random() < 0.6) for _ in range(rng.randint(1, 7))]


@pytest.mark.parametrize("seed", range(8))
def test_roles_in_any_order(seed):
    for i in range(60):
        rng = random.Random(1000 * seed + i)
        Pair(_units(rng), rng).run()


@pytest.mark.parametrize("steps", [1, 2, 3, 4, 8])
@pytest.mark.parametrize("two", ["all", "none", "in turn"])
def test_units_of_one_kind(steps, two):
    for i in range(30):
        rng = random.Random(i)
        Pair([(steps, two == "all" or (two == "in turn" and n % 2 == 0)) for n in range(6)], rng).run()


@pytest.mark.parametrize("mistake", ["two places for exponents", "queries at once", "one tile's scores for both", "scores over weights", "a tile alone does not wait", "outputs are not read"])
def test_the_model_notices(mistake):
    """Each of the waits that the kernel's comments explain, left out of the model, is missed in some order."""
    with pytest.raises(AssertionError):
        for i in range(400):
            rng = random.Random(i)
            Pair(_units(rng), rng, mistake).run()
