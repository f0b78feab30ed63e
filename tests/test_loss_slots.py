"""CPU model of the slots of k_ring (csrc/k_loss.cu) whose loads come back late:
a warp that gives a slot back while they are under way meets the next copy's
elements.  The ring and its random schedules are test_loss_ring.py's."""
import pytest

from tests.test_loss_ring import SHAPES, Ring


class Loads(set):
    """What has been taken from slots: each entry starts a load that comes back later."""

    def __init__(self, ring):
        super().__init__()
        self.ring = ring

    def add(self, what):
        x = what if isinstance(what, int) else next(x for x in self.ring.held if x is not None and self.ring.plan[x][:2] == what)
        self.ring.under_way.append((self.ring.current, x))
        super().add(what)


class LateRing(Ring):
    """`fence`: a team goes on, to where it gives the slot back, when its loads are back."""

    def __init__(self, *args, fence, **kw):
        super().__init__(*args, **kw)
        self.fence, self.under_way, self.current = fence, [], None
        self.taken, self.written = Loads(self), Loads(self)

    def come_back(self):
        _, x = self.under_way.pop(self.rng.randrange(len(self.under_way)))
        assert self.held[x % self.slots] == x, "a load met another copy's elements"

    def run(self):
        live, idle = list(self.tasks), 0
        while live or self.under_way:
            if self.under_way and (not live or self.rng.random() < 0.1):
                self.come_back()
                continue
            if self.flying and self.rng.random() < 0.3:
                self.land()
                continue
            task = self.rng.choice(live)
            if self.fence and any(t is task for t, _ in self.under_way):
                continue
            self.current, before = task, self.state()
            if next(task, "end") == "end":
                live.remove(task)
            idle = idle + 1 if self.state() == before and not self.flying and not self.under_way else 0
            assert idle < 3000, "nothing goes on"


@pytest.mark.parametrize("chunks", SHAPES, ids=str)
@pytest.mark.parametrize("slots,s_teams,g_teams", [(12, 1, 2), (6, 2, 0), (12, 0, 2)])
def test_loads_are_back_before_the_slot_goes_on(chunks, slots, s_teams, g_teams):
    for seed in range(4):
        ring = LateRing(chunks, slots, 8, s_teams, g_teams, seed, fence=True)
        ring.run()
        if g_teams:
            assert ring.written == {(r, c) for r, n in enumerate(chunks) for c in range(n)}
        if s_teams:
            assert len(ring.taken) == sum(chunks)


def test_slots_given_back_with_loads_under_way():
    """Without the fence, some load meets the next copy."""
    with pytest.raises(AssertionError, match="another copy"):
        for seed in range(20):
            LateRing([19] * 5, 12, 8, 1, 2, seed, fence=False).run()
