"""The stage ring of the 8-bit integer tensor-core kernel as a model with random interleavings: weights, row copies by a team of warps, products, barriers whose turns are told
apart by parity alone. Every arrival has to fall into the turn it is meant for, and every run has to end; a team larger than the ring does neither, and the kernel's ring has
as many stages as copying warps at least."""
import random

import pytest


class Barrier:
    """an mbarrier: `count` arrivals complete a phase; a wait on a parity passes when the phase of that parity is the one completed last"""

    def __init__(self, count):
        self.count, self.left, self.phase = count, count, 0

    def arrive(self, turn):
        assert self.phase == turn, "an arrival meant for turn %d falls into turn %d" % (turn, self.phase)
        self.left -= 1
        assert self.left >= 0
        if self.left == 0:
            self.left, self.phase = self.count, self.phase + 1

    def passed(self, parity):
        return (self.phase & 1) != parity


def run(seed, stages, team, lag, kb, units, gather):
    rng = random.Random(seed)
    full, empty = [Barrier(2) for _ in range(stages)], [Barrier(1) for _ in range(stages)]
    total, landed, freed = kb * units, [0] * (kb * units), [0] * (kb * units)

    def wait(bar, parity):
        while not bar.passed(parity):
            yield

    def weights():
        for g in range(total):
            s, turn = g % stages, g // stages
            yield from wait(empty[s], (turn & 1) ^ 1)
            assert turn == 0 or freed[g - stages], "stage %d is overwritten before its products" % s
            full[s].arrive(turn)
            landed[g] += 1
            yield

    def rows(me, step):
        pending = []
        for g in range(me, total, step):
            s, turn = g % stages, g // stages
            yield from wait(empty[s], (turn & 1) ^ 1)
            assert turn == 0 or freed[g - stages], "stage %d is overwritten before its products" % s
            yield
            pending.append(g)
            while len(pending) > lag:
                p = pending.pop(0)
                full[p % stages].arrive(p // stages)
                landed[p] += 1
                yield
        for p in pending:
            full[p % stages].arrive(p // stages)
            landed[p] += 1
            yield

    def products():
        for u in range(units):
            for i in range(kb):
                g = u * kb + i
                yield from wait(full[g % stages], (g // stages) & 1)
                assert landed[g] == 2
                freed[g] = 1
                empty[g % stages].arrive(g // stages)
                yield

    actors = [weights(), products()] + ([rows(i, team) for i in range(team)] if gather else [rows(0, 1)])
    idle = 0
    while actors:
        a = rng.choice(actors)
        before = (tuple(b.phase * 9 + b.left for b in full + empty), sum(landed))
        try:
            for _ in range(rng.choice((1, 1, 2, 9))):
                next(a)
        except StopIteration:
            actors.remove(a)
            idle = 0
            continue
        idle = idle + 1 if before == (tuple(b.phase * 9 + b.left for b in full + empty), sum(landed)) else 0
        assert idle < 4000, "nothing moves any more"
    assert all(v == 2 for v in landed) and all(freed)


@pytest.mark.parametrize("stages", [4, 5, 6, 7, 8, 11, 12])
@pytest.mark.parametrize("kb,units", [(1, 9), (2, 7), (3, 6), (4, 5), (6, 5), (16, 3)])
def test_every_arrival_falls_into_its_turn(stages, kb, units):
    for seed in range(20):
        run(seed, stages, 4, int(stages > 7), kb, units, True)
    run(99, stages, 1, 0, kb, units, False)


def test_a_team_larger_than_the_ring_is_caught():
    with pytest.raises(AssertionError):
        for seed in range(200):
            run(seed, 3, 4, 0, 16, 3, True)


def test_stages_held_back_by_more_than_the_ring_are_caught():
    with pytest.raises(AssertionError):
        for seed in range(200):
            run(seed, 4, 4, 1, 16, 3, True)
