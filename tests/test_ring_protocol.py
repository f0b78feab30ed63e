"""CPU model of the barriers in the tensor-core projection
(csrc/k_project.cu, k_project_tc) under random schedules.

The TMA warp (shared slices) and the builders (low-rank slices, two units to
one) fill one ring of operand slices that the matrix instructions drain, tile
by tile.  A barrier's parity tells a phase from the one before only, so nobody
may wait for a slice more than one turn of the ring ahead: turn[0] and turn[1]
pass the ring to and fro.  The model's parts have the kernel's names; a slice
that is filled before it is drained, drained before it is filled, or a barrier
that gets an arrival too many fails an assertion, as does a schedule in which
nobody can go on."""
import random

import pytest

STAGES = 6


class Barrier:
    def __init__(self, count):
        self.count = self.pending = count
        self.phase = self.bytes = 0

    def _check(self):
        if self.pending == 0 and self.bytes == 0:
            self.phase += 1
            self.pending = self.count

    def arrive(self, expect=0):
        assert self.pending > 0, "an arrival too many"
        self.bytes += expect
        self.pending -= 1
        self._check()

    def complete(self, n):
        self.bytes -= n
        self._check()

    def wait(self, parity):
        while self.phase & 1 == parity:
            yield


class Ring:
    def __init__(self, n, phase):
        self.i, self.n, self.phase = 0, n, phase

    def skip(self, by):
        self.i += by
        self.phase ^= self.i // self.n & 1
        self.i %= self.n

    def next(self):
        self.skip(1)


def run(ctas, kblocks, tile_units, seed, turns=True):
    """The tiles' units: low-rank units of each tile of a CTA (or pair)."""
    rng, both = random.Random(seed), range(ctas)
    tile_units = [u if kblocks else max(1, u) for u in tile_units]  # something has to clear the accumulator
    tiles = len(tile_units)
    full = [Barrier(ctas) for _ in range(STAGES)]  # of the CTA that issues
    empty, counted = ([[Barrier(1) for _ in range(n)] for _ in both] for n in (STAGES, 8))
    turn, acc_full = ([[Barrier(1), Barrier(1)] for _ in both] for _ in range(2))
    acc_empty = [Barrier(ctas), Barrier(ctas)]
    units, bad = [[0] * 8 for _ in both], [[None] * 16 for _ in both]
    held = [[None] * STAGES for _ in both]
    flying, done = [], []

    def put(c, i, what):
        assert held[c][i] is None, f"{what} over {held[c][i]}"
        held[c][i] = "under way"
        flying.append((c, i, what))

    def tma(c):
        r = Ring(STAGES, 1)
        for t in range(tiles if kblocks else 0):
            for k in range(kblocks):
                yield from empty[c][r.i].wait(r.phase)
                full[r.i].arrive(ctas if c == 0 else 0)
                put(c, r.i, (t, "shared", k))
                yield
                r.next()
            if turns:
                turn[c][0].arrive()
                yield
                yield from turn[c][1].wait(t & 1)
            else:
                yield from counted[c][t & 7].wait(t >> 3 & 1)
            r.skip((units[c][t & 7] + 1) // 2)

    def builders(c):
        r = Ring(STAGES, 1)
        for t in range(tiles):
            bad[c][t & 15] = t
            units[c][t & 7] = tile_units[t]
            counted[c][t & 7].arrive()
            yield
            r.skip(kblocks)
            last = (tile_units[t] + 1) // 2
            if kblocks and turns:
                yield from turn[c][0].wait(t & 1)
                if last == 0:
                    turn[c][1].arrive()
                    yield
            for s in range(last):
                yield from empty[c][r.i].wait(r.phase)
                put(c, r.i, (t, "low", s))
                yield
                full[r.i].arrive(ctas if c == 0 else 0)
                if s + 1 == last and kblocks and turns:
                    turn[c][1].arrive()
                yield
                r.next()

    def drain(r, what):
        yield from full[r.i].wait(r.phase)
        for c in both:
            assert held[c][r.i] == what, f"{held[c][r.i]} taken for {what}"
            held[c][r.i] = None
        yield
        for c in both:
            empty[c][r.i].arrive()
        r.next()

    def instructions():
        r, acc = Ring(STAGES, 0), Ring(2, 1)
        for t in range(tiles):
            yield from acc_empty[acc.i].wait(acc.phase)
            for k in range(kblocks):
                yield from drain(r, (t, "shared", k))
            yield from counted[0][t & 7].wait(t >> 3 & 1)
            assert units[0][t & 7] == tile_units[t]
            for s in range((tile_units[t] + 1) // 2):
                yield from drain(r, (t, "low", s))
            for c in both:
                acc_full[c][acc.i].arrive()
            done.append(t)
            acc.next()

    def epilogue(c):
        acc = Ring(2, 0)
        for t in range(tiles):
            yield from acc_full[c][acc.i].wait(acc.phase)
            assert bad[c][t & 15] == t
            for _ in range(rng.randint(0, 20)):
                yield
            acc_empty[acc.i].arrive()
            acc.next()

    roles = [instructions()] + [part(c) for c in both for part in (tma, builders, epilogue)]
    speed = [rng.random() ** 2 + 0.01 for _ in roles]
    for _ in range(400000):
        if not roles:
            break
        if flying and rng.random() < 0.3:
            c, i, what = flying.pop(rng.randrange(len(flying)))
            held[c][i] = what
            full[i].complete(1)
        k = rng.choices(range(len(roles)), speed)[0]
        try:
            next(roles[k])
        except StopIteration:
            roles.pop(k), speed.pop(k)
    assert not roles and done == list(range(tiles)), "nobody can go on"


@pytest.mark.parametrize("ctas", [1, 2])
@pytest.mark.parametrize("kblocks", [0, 1, 2, 5, 6, 7, 24])
def test_ring_keeps_its_order(ctas, kblocks):
    rng = random.Random(100 * kblocks + ctas)
    for seed, units in enumerate(([0], [1], [2] * 3, [0] * 20, [3, 0, 4] * 6, [1, 0] * 9, [40, 13, 0, 2], [4] * 12,
                                  *([rng.choice([0, 0, 1, 2, 3, rng.randint(0, 30)]) for _ in range(rng.randint(9, 24))] for _ in range(4)))):
        run(ctas, kblocks, units, seed)


def test_ring_without_turns_fails():
    """The model finds the fault that the turns are there for."""
    failed = 0
    for seed in range(20):
        try:
            run(1, 24, [4] * 4, seed, turns=False)
        except AssertionError:
            failed += 1
    assert failed
