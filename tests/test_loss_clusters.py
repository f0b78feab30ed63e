"""CPU model of the clusters of k_ring (csrc/k_loss.cu) that write gradients in
place of the logits, from known statistics: nothing orders a cluster's CTAs then.
Random schedules must give every target the gradient from its own logit."""
import random

import pytest

SLOT = 16384  # bytes
TEAM = 8      # warps to a slot


class Parts:
    """A row's parts as struct Span has them, and the warps' pieces of their slots."""

    def __init__(self, vocab, size, head, log):
        self.head, self.vocab, self.slot = head, vocab, SLOT // size
        end = head + vocab
        span = ((end + (1 << log) - 1 >> log) + 127) // 128 * 128
        self.parts = [(min(end, r * span), min(end, r * span + span)) for r in range(1 << log)]

    def pieces(self, rank):
        first, last = self.parts[rank]
        piece = self.slot // TEAM
        for p0 in range(first, last, self.slot):
            for w in range(TEAM):
                yield p0 + w * piece, piece

    def fixes(self, rank, y, own):
        """Whether the CTA adds the target's g to its place; `own`: only in its part of the row."""
        last = self.parts[rank][1]
        return any(0 <= y + self.head - p < n and (not own or y + self.head < last) for p, n in self.pieces(rank))

    def owner(self, y):
        return next(r for r, (a, b) in enumerate(self.parts) if a <= y + self.head < b)


SHAPES = [(151936, 2, 0, 1), (151936, 2, 3, 1), (151936, 4, 0, 2), (151936, 4, 1, 3), (50257, 2, 5, 1), (20000, 4, 0, 2), (400003, 4, 0, 1)]


def _targets(parts):
    """The row's ends, and the places around each part's end and its last slot's."""
    at = {0, parts.vocab - 1}
    for r, (first, last) in enumerate(parts.parts):
        slots = -(-(last - first) // parts.slot)
        for p in (last, first + slots * parts.slot):
            at |= {p - parts.head + d for d in (-129, -128, -1, 0, 1, 127, 128)}
    return sorted(y for y in at if 0 <= y < parts.vocab)


@pytest.mark.parametrize("vocab,size,head,log", SHAPES)
def test_a_target_is_fixed_by_the_cta_that_has_it(vocab, size, head, log):
    parts = Parts(vocab, size, head, log)
    for y in _targets(parts):
        assert [r for r in range(1 << log) if parts.fixes(r, y, True)] == [parts.owner(y)]


def _in_place(parts, targets, own, rng):
    """Rows of a gradient from known statistics, in place, by CTAs that nothing orders: each
    reads the targets' logits of up to 32 rows ahead, then writes row after
    row.  Returns the rows whose target did not get the gradient from its logit."""
    logit = {r: ("logit", r) for r in range(len(targets))}  # what lies in the target's place of a row

    def cta(rank):
        for b in range(0, len(targets), 32):
            seen = {r: logit[r] for r in range(b, min(b + 32, len(targets)))}
            yield
            for r, zy in seen.items():
                if rank == parts.owner(targets[r]):
                    logit[r] = ("-g p", r)
                if parts.fixes(rank, targets[r], own):
                    logit[r] = ("g - g p", zy)
                yield

    live = [cta(rank) for rank in range(len(parts.parts))]
    slow = rng.choice(live)
    while live:
        task = rng.choice(live)
        if task is slow and len(live) > 1 and rng.random() < 0.9:
            continue
        if next(task, "end") == "end":
            live.remove(task)
    return [r for r in range(len(targets)) if logit[r] != ("g - g p", ("logit", r))]


@pytest.mark.parametrize("vocab,size,head,log", SHAPES)
def test_gradient_in_place_by_ctas_that_nothing_orders(vocab, size, head, log):
    parts, rng = Parts(vocab, size, head, log), random.Random(vocab + head)
    targets = _targets(parts)
    for _ in range(6):
        assert _in_place(parts, rng.choices(targets, k=70), True, rng) == []


def test_a_target_behind_a_part_must_not_be_fixed():
    """Were it fixed wherever a warp's piece reaches, beyond the part's end too, a CTA
    could read what its neighbour has put in the target's place."""
    parts, rng = Parts(151936, 2, 0, 1), random.Random(1)
    y = parts.parts[0][1]
    assert parts.fixes(0, y, False) and parts.owner(y) == 1
    assert any(_in_place(parts, [y] * 70, False, rng) for _ in range(6))
