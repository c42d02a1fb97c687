"""The barriers of the tree attention's kernel, as a model on the CPU: its roles run in random orders, every barrier is
waited for by its parity as on the GPU, and every buffer remembers what was put into it.

What the model shows: with the numbers of the source (barriers per step, sets of row scales, places of the ring) no
role ever goes on too early, reads another tile's data or waits for good; with fewer barriers or sets some do.
"""
from __future__ import annotations

import pathlib
import random
import re

import pytest

SOURCE = (pathlib.Path(__file__).resolve().parents[1] / "in-c-test_b200" / "csrc" / "tree_attend.cu").read_text()


def constant(name):
    return int(re.search(rf"constexpr \w+ {name} = (\d+);", SOURCE).group(1))


STEPS, SCALES, UNITS = constant("kSteps"), constant("kScaleRing"), constant("kUnits")


class Stuck(Exception):
    pass


class Wrong(Exception):
    pass


def expect(ok, what):
    if not ok:
        raise Wrong(what)


class Bar:
    """An mbarrier: `count` arrivals complete a phase; a wait for a phase looks at its parity only."""

    arrivals = 0  # of all barriers

    def __init__(self, count):
        self.count = self.pending = count
        self.phases = 0

    def arrive(self, n=1):
        expect(n <= self.pending, "more arrivals than the phase has")
        self.pending -= n
        Bar.arrivals += 1
        if not self.pending:
            self.pending = self.count
            self.phases += 1

    def passed(self, phase):
        ok = (self.phases & 1) != (phase & 1)
        expect(not ok or self.phases > phase, "passed a phase that is not complete")
        return ok


class Kernel:
    """One CTA that walks items of the given numbers of tiles.  Roles are generators that yield between their steps
    and, "blocked", while they wait; `pipe` is the tensor core (in order), `loads` are copies in flight (any order)."""

    def __init__(self, items, q8, steps, scales, rng, early_rope=False):
        self.items, self.q8, self.steps, self.scales, self.rng = items, q8, steps, scales, rng
        self.early_rope = early_rope  # a mistake: the rope is loaded when the scores before are done
        self.rope_in = 0 if q8 else 1  # bf16: unit 1's barrier counts the rope too; Q8: that has its own
        self.full = [[Bar(1) for _ in range(steps)], [Bar(1 + self.rope_in) for _ in range(steps)]]
        self.r_full = [Bar(1), Bar(1)]
        self.done = [[Bar(1) for _ in range(steps)] for _ in range(2)]
        self.s_full, self.s_empty = [Bar(1), Bar(1)], [Bar(1), Bar(1)]
        self.q_done, self.qr_full, self.p_full, self.o_empty = Bar(1), Bar(1), Bar(1), Bar(1)
        self.ring, self.rope, self.scores, self.scale_set = {}, {}, {}, {}
        self.query = self.query_rope = self.p = self.o = self.stored = -1
        self.pipe, self.loads = [], []

    def wait(self, bar, phase):
        while not bar.passed(phase):
            yield "blocked"

    def wait_done(self, step, unit):
        yield from self.wait(self.done[unit][step % self.steps], step // self.steps)

    def wait_full(self, step, unit):
        yield from self.wait(self.full[unit][step % self.steps], step // self.steps)

    def fill(self, step, unit, arrivals):
        self.ring[(2 * step + unit) % UNITS] = step
        self.full[unit][step % self.steps].arrive(arrivals)

    def holds(self, step):
        return all(self.ring.get((2 * step + h) % UNITS) == step for h in range(2))

    def free(self, step, unit):
        if 2 * step + unit >= UNITS:
            yield from self.wait_done(step - UNITS // 2, unit)

    def producer(self):
        j = g = 0
        step = {}  # of each tile
        for tiles in self.items:
            for h in range(2):
                yield from self.free(j, h)
                self.loads.append(lambda j=j, h=h: self.fill(j, h, 1 + h * self.rope_in))
                yield
            j += 1
            for _ in range(tiles):
                for h in range(0 if self.q8 else 2):
                    yield from self.free(j, h)
                    self.loads.append(lambda j=j, h=h: self.fill(j, h, 1))
                    yield
                if g >= 2 and self.q8 and not self.early_rope:  # the place of the second weights of tile g - 2
                    yield from self.wait_done(step[g - 2], 1)
                elif g >= 2:
                    yield from self.wait(self.s_full[g & 1], (g >> 1) - 1)
                step[g] = j

                def rope(j=j, g=g):
                    self.rope[g & 1] = g
                    (self.r_full[g & 1] if self.q8 else self.full[1][j % self.steps]).arrive()

                self.loads.append(rope)
                j, g = j + 1, g + 1
                yield

    def converter(self, odd):
        j = g = 0
        for tiles in self.items:
            j += 1
            for _ in range(tiles):
                if (g & 1) == odd:
                    for h in range(2):
                        yield from self.free(j, h)
                        if h:
                            self.scale_set[g % self.scales] = g
                        self.fill(j, h, 1)
                        yield
                j, g = j + 1, g + 1

    def score_issuer(self):
        j = g = 0
        for n, tiles in enumerate(self.items):
            if n:
                yield from self.wait(self.q_done, n - 1)
            for h in range(2):
                yield from self.wait_full(j, h)

            def copy_query(j=j, n=n):
                expect(self.holds(j), "the query's place holds another step")
                self.query = n
                for h in range(2):
                    self.done[h][j % self.steps].arrive()

            self.pipe.append(copy_query)
            yield
            j += 1
            for t in range(tiles):
                yield from self.wait_full(j, 0)
                before = g - (1 if self.q8 else 2)
                if before >= 0:
                    yield from self.wait(self.s_empty[before & 1], before >> 1)
                if t == 0:
                    yield from self.wait(self.qr_full, n)
                yield from self.wait_full(j, 1)
                if self.q8:
                    yield from self.wait(self.r_full[g & 1], g >> 1)

                def score(j=j, g=g, n=n, last=t + 1 == tiles):
                    expect(self.holds(j), "scores of another step's keys")
                    expect(self.query == self.query_rope == n, "scores of another item's query")
                    expect(self.rope[g & 1] == g, "scores of another tile's rope")
                    self.scores[0 if self.q8 else g & 1] = g
                    self.s_full[g & 1].arrive()
                    if last:
                        self.q_done.arrive()

                self.pipe.append(score)
                j, g = j + 1, g + 1
                yield

    def pv_issuer(self):
        j = g = 0
        for n, tiles in enumerate(self.items):
            j += 1
            for t in range(tiles):
                if t == 0 and n:
                    yield from self.wait(self.o_empty, n - 1)
                for h in range(2):
                    yield from self.wait_full(j, h)
                yield from self.wait(self.p_full, g)

                def product(h, j=j, g=g, n=n):
                    expect(self.ring[(2 * j + h) % UNITS] == j, "P.V with another step's rows")
                    expect(self.p == g, "P.V with another tile's weights")
                    expect(not self.q8 or self.rope[g & 1] == ("second weights", g), "P.V with other second weights")
                    expect(self.stored >= n - 1, "P.V into an output that is not read yet")
                    self.o = g
                    self.done[h][j % self.steps].arrive()

                self.pipe += [lambda h=h, f=product: f(h) for h in range(2)]
                j, g = j + 1, g + 1
                yield

    def query_rope_loader(self):
        for n in range(len(self.items)):
            if n:
                yield from self.wait(self.q_done, n - 1)

            def load(n=n):
                self.query_rope = n
                self.qr_full.arrive()

            self.loads.append(load)
            yield

    def softmax(self):
        j = g = 0
        for n, tiles in enumerate(self.items):
            j += 1
            for t in range(tiles):
                yield from self.wait(self.s_full[g & 1], g >> 1)
                if self.q8:
                    yield from self.wait_full(j, 1)
                    yield
                    expect(self.scale_set[g % self.scales] == g, "row scales of another tile")
                expect(self.scores[0 if self.q8 else g & 1] == g, "scores of another tile")
                self.s_empty[g & 1].arrive()
                yield
                if t and self.rng.random() < 0.3:  # the accumulator is rescaled
                    yield from self.wait_done(j - 1, 1)
                    yield
                if g:
                    yield from self.wait_done(j - (1 if t else 2), 1)
                self.p = g
                if self.q8:
                    expect(self.rope[g & 1] == g, "the rope's place holds another tile's")
                    self.rope[g & 1] = ("second weights", g)
                self.p_full.arrive()
                j, g = j + 1, g + 1
                yield
            yield from self.wait_done(j - 1, 1)
            yield
            expect(self.o == g - 1, "an output without its last tile")
            self.stored = n
            self.o_empty.arrive()
            yield

    def run(self):
        rng = self.rng
        roles = [self.producer(), self.score_issuer(), self.pv_issuer(), self.query_rope_loader(), self.softmax()]
        roles += [self.converter(0), self.converter(1)] if self.q8 else []
        speed = {r: rng.choice([1, 1, 5, 20, 0.1]) for r in [*roles, "pipe"]}
        speed["load"] = rng.choice([1, 5, 0.2])
        blocked = set()
        while roles:
            picks = [r for r in roles if r not in blocked] + ["pipe"] * bool(self.pipe) + ["load"] * bool(self.loads)
            if not picks:
                raise Stuck
            pick = rng.choices(picks, [speed[p] for p in picks])[0]
            before = Bar.arrivals
            if pick == "pipe":
                self.pipe.pop(0)()
            elif pick == "load":
                self.loads.pop(0 if rng.random() < 0.8 else rng.randrange(len(self.loads)))()
            else:
                try:
                    if next(pick):
                        blocked.add(pick)
                except StopIteration:
                    roles.remove(pick)
            if Bar.arrivals != before:
                blocked = set()


def runs(q8, steps, scales, n, seed, **mistake):
    """How many of n random batches fail."""
    rng = random.Random(seed)
    bad = 0
    for _ in range(n):
        items = [rng.choice([1, 2, 2, 3, 4, 5]) if rng.random() < 0.8 else rng.randint(1, 9)
                 for _ in range(rng.randint(1, 10))]
        try:
            Kernel(items, q8, steps, scales, rng, **mistake).run()
        except (Stuck, Wrong):
            bad += 1
    return bad


@pytest.mark.parametrize("q8", [False, True], ids=["bf16", "q8"])
def test_no_order_of_the_roles_goes_wrong(q8):
    assert runs(q8, STEPS, SCALES, 150, 1) == 0


@pytest.mark.parametrize("q8", [False, True], ids=["bf16", "q8"])
def test_four_barriers_are_too_few(q8):
    """The softmax asks for a step that lies four behind the last one done."""
    assert runs(q8, 4, SCALES, 100, 2) > 0


def test_five_barriers_are_too_few_for_q8():
    """A converter group, which takes every second tile, asks for a step five ahead of one that is not done."""
    assert runs(True, 5, SCALES, 250, 3) > 0


def test_three_sets_of_row_scales_are_too_few():
    assert runs(True, STEPS, 3, 100, 4) > 0


def test_the_rope_has_to_wait_for_the_second_weights():
    assert runs(True, STEPS, SCALES, 50, 5, early_rope=True) > 0
