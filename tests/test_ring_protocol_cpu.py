"""The draft-tree decode's ring of loads between one producer and two issuers that take
alternate tiles, as a model of its barriers.

A wait by parity returns when the phase before the current one has the awaited parity.
An issuer never waits for the other's slots, so on ONE set of barriers a late load lets
it take an older phase for the awaited one: it reads a slot that has not landed and frees
it, and the producer arms a barrier whose load is still on its way, which is an error of
the hardware's counters.  With a set of barriers for each issuer every wait is exact."""
import random

import pytest

SLOTS, PER_TILE = 5, 3


class Barrier:
    """One arrival and its bytes a phase."""

    def __init__(self):
        self.phase, self.armed = 0, False

    def arm(self):
        assert not self.armed, "armed with a load on its way"
        self.armed = True

    def complete(self):
        self.phase, self.armed = self.phase + 1, False

    def passed(self, parity):
        return (self.phase - 1) % 2 == parity


def run(own_sets, tiles, seed):
    rng = random.Random(seed)
    full = [[Barrier() for _ in range(SLOTS)] for _ in range(2 if own_sets else 1)]
    freed = [0] * SLOTS     # uses of a slot that were given back
    content = [-1] * SLOTS  # index whose load landed in it last
    loads = []              # (time, index, barrier)
    now, filled = 0.0, 0
    at = [0, PER_TILE]      # issuer i's next slot index
    mine = [[0] * SLOTS, [0] * SLOTS]
    done = 0
    while done < tiles * PER_TILE:
        now += 1
        for load in [x for x in loads if x[0] <= now]:
            loads.remove(load)
            content[load[1] % SLOTS] = load[1]
            load[2].complete()
        if filled < tiles * PER_TILE and freed[filled % SLOTS] >= filled // SLOTS:
            bar = full[(filled // PER_TILE) % 2 if own_sets else 0][filled % SLOTS]
            bar.arm()
            loads.append((now + (400 if rng.random() < 0.02 else 20 + 10 * rng.random()), filled, bar))
            filled += 1
        for i in rng.sample((0, 1), 2):
            n = at[i]
            if n >= tiles * PER_TILE:
                continue
            s = n % SLOTS
            use = mine[i][s] if own_sets else n // SLOTS
            if not full[i if own_sets else 0][s].passed(use % 2):
                continue
            assert content[s] == n, "read before it landed"
            mine[i][s] += 1
            freed[s] += 1
            done += 1
            at[i] = n + 1 if (n + 1) % PER_TILE else n + 1 + PER_TILE
        assert now < 1e6
    return now


@pytest.mark.parametrize("seed", range(20))
def test_every_load_is_read_once_it_landed(seed):
    run(True, 200, seed)


def test_one_set_of_barriers_is_not_enough():
    bad = 0
    for seed in range(20):
        try:
            run(False, 200, seed)
        except AssertionError:
            bad += 1
    assert bad > 0
