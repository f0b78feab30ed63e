"""CPU model of the ring of k_ring (csrc/k_loss.cu): one thread that starts
copies, a team that takes statistics, one that finishes rows, two teams that
write gradients, barriers that are waited for by parity, copies that land in
any order.  Random schedules must neither stop, nor let a team take a slot that
does not hold what it expects, nor let a wait take one phase for another."""
import random

import pytest


class Barrier:
    def __init__(self, count):
        self.count, self.left, self.phase = count, count, 0

    def arrive(self, phase):
        """An arrival that means the phase with this number."""
        assert self.phase == phase, "arrived in another phase"
        self.left -= 1
        if self.left == 0:
            self.phase, self.left = self.phase + 1, self.count

    def done(self, parity):
        return (self.phase & 1) != parity


class Ring:
    """Rows of `chunks[r]` slots; the first of them, beyond `keep`, are copied twice."""

    def __init__(self, chunks, slots, keep, s_teams, g_teams, seed, acknowledge=True):
        self.rng, self.slots, self.acknowledge = random.Random(seed), slots, acknowledge
        self.plan = []  # loads in their order: (row, chunk, taken by S, released by S)
        self.rows = []  # each row's (first load, its chunks, how many of them come twice)
        for r, n in enumerate(chunks):
            again = max(0, n - keep) if g_teams and s_teams else 0
            self.rows.append((len(self.plan), n, again))
            self.plan += [(r, c, bool(s_teams), bool(s_teams) and (not g_teams or c < again)) for c in range(n)]
            self.plan += [(r, c, False, False) for c in range(again)]
        self.both = bool(s_teams and g_teams)
        self.full, self.empty = [Barrier(1) for _ in range(slots)], [Barrier(2 if self.both and acknowledge else 1) for _ in range(slots)]
        self.stats_full, self.stats_free = [Barrier(s_teams or 1) for _ in range(2)], [Barrier(1) for _ in range(2)]
        self.coef_full, self.coef_free = [Barrier(1) for _ in range(4)], [Barrier(g_teams or 1) for _ in range(4)]
        self.held, self.flying = [None] * slots, []
        self.stats, self.coef = {}, {}
        self.taken, self.written = set(), set()
        self.tasks = [self.producer(), self.finisher(bool(s_teams), bool(g_teams))]
        self.tasks += [self.statistics(t, s_teams, bool(g_teams)) for t in range(s_teams)] + [self.gradient(t, g_teams) for t in range(g_teams)]

    def wait(self, barrier, phase):
        """Until the phase has ended; by its parity, as the hardware does."""
        while not barrier.done(phase & 1):
            yield
        assert barrier.phase > phase, "a wait took one phase for another"

    def producer(self):
        for x in range(len(self.plan)):
            slot, turn = x % self.slots, x // self.slots
            if turn:
                yield from self.wait(self.empty[slot], turn - 1)
            self.flying.append(x)
            yield

    def land(self):
        x = self.flying.pop(self.rng.randrange(len(self.flying)))
        self.held[x % self.slots] = x
        self.full[x % self.slots].arrive(x // self.slots)

    def statistics(self, team, teams, both):
        for r, (x0, n, again) in enumerate(self.rows):
            for x in range(x0, x0 + n):
                if x % self.slots % teams != team:
                    continue
                yield from self.wait(self.full[x % self.slots], x // self.slots)
                assert self.held[x % self.slots] == x, "statistics of another slot"
                self.taken.add(x)
                yield
                if self.both and self.acknowledge:
                    self.empty[x % self.slots].arrive(x // self.slots)
                if self.plan[x][3]:
                    self.empty[x % self.slots].arrive(x // self.slots)
            if r >= 2:
                yield from self.wait(self.stats_free[r % 2], r // 2 - 1)
            self.stats[r % 2] = r
            self.stats_full[r % 2].arrive(r // 2)
            for x in range(x0 + n, x0 + n + again):
                if x % self.slots % teams == team:
                    yield from self.wait(self.full[x % self.slots], x // self.slots)
                    if self.acknowledge:
                        self.empty[x % self.slots].arrive(x // self.slots)

    def finisher(self, s, g):
        for r in range(len(self.rows)):
            if s:
                yield from self.wait(self.stats_full[r % 2], r // 2)
                assert self.stats[r % 2] == r
                x0, n, _ = self.rows[r]
                assert all(x in self.taken for x in range(x0, x0 + n)), "a row was finished before all of it was seen"
                self.stats_free[r % 2].arrive(r // 2)
                yield
            if g:
                if r >= 4:
                    yield from self.wait(self.coef_free[r % 4], r // 4 - 1)
                self.coef[r % 4] = r
                self.coef_full[r % 4].arrive(r // 4)

    def gradient(self, team, teams):
        for r, (x0, n, again) in enumerate(self.rows):
            yield from self.wait(self.coef_full[r % 4], r // 4)
            assert self.coef[r % 4] == r
            for x in range(x0 + again, x0 + again + n):
                if x % self.slots % teams != team:
                    continue
                yield from self.wait(self.full[x % self.slots], x // self.slots)
                assert self.held[x % self.slots] == x, "gradient from another slot"
                self.written.add(self.plan[x][:2])
                yield
                self.empty[x % self.slots].arrive(x // self.slots)
            self.coef_free[r % 4].arrive(r // 4)

    def run(self, favour=None):
        """Steps of the tasks and landings at random; `favour` is a task that is seldom chosen."""
        live, idle = list(self.tasks), 0
        while live:
            if self.flying and self.rng.random() < 0.3:
                self.land()
                idle = 0
                continue
            task = self.rng.choice(live)
            if favour is not None and task is self.tasks[favour % len(self.tasks)] and self.rng.random() < 0.95:
                continue
            before = self.state()
            try:
                next(task)
            except StopIteration:
                live.remove(task)
                idle = 0
                continue
            idle = idle + 1 if self.state() == before and not self.flying else 0
            assert idle < 3000, "nothing goes on"

    def state(self):
        return (tuple(b.phase for b in self.full + self.empty + self.stats_full + self.stats_free + self.coef_full + self.coef_free),
                len(self.taken), len(self.written), len(self.flying))


SHAPES = [[1] * 30, [5] * 12, [10, 9, 10, 11, 10, 9], [19] * 5, [38, 38, 37], [1, 19, 2, 8, 9, 12, 13, 1, 1, 30]]


@pytest.mark.parametrize("chunks", SHAPES, ids=str)
def test_statistics_and_gradient(chunks):
    for seed in range(8):
        ring = Ring(chunks, 12, 8, 1, 2, seed)
        ring.run(favour=seed)
        assert ring.written == {(r, c) for r, n in enumerate(chunks) for c in range(n)}


@pytest.mark.parametrize("chunks", SHAPES, ids=str)
def test_one_role_alone(chunks):
    for seed in range(6):
        ring = Ring(chunks, 6, 8, 2, 0, seed)
        ring.run(favour=seed)
        assert len(ring.taken) == sum(chunks)
        ring = Ring(chunks, 12, 8, 0, 2, seed)
        ring.run(favour=seed)
        assert ring.written == {(r, c) for r, n in enumerate(chunks) for c in range(n)}


def test_slots_that_go_on_without_the_statistics():
    """Were a slot that is copied again free without the statistics' team, that team, when it
    is slow, would wait for a phase that lies two back."""
    with pytest.raises(AssertionError, match="phase|slot|goes on"):
        for seed in range(40):
            Ring([19] * 5, 12, 8, 1, 2, seed, acknowledge=False).run(favour=2)
