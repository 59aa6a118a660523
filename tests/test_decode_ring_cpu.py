"""The barriers between the S-CTA's producer, its two GEMM1 issuers and the softmax of the
decode kernels, as a model that takes ring sizes, barrier sets and the order of waits from
the kernels' sources.

A wait by parity returns when the phase before the barrier's current one has the awaited
parity, so it is exact only while the phase before the awaited one is known to be
complete.  The model's loads and tensor operations take random times; it fails where an
issuer reads a slot that has not landed or a Q that is not copied, overwrites an S tile
that is not read, or where a barrier is armed with a load on its way."""
import os
import random
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ada-mla_b200", "csrc")


def source(name):
    with open(os.path.join(CSRC, name)) as f:
        return f.read()


def number(text, name, default=None):
    m = re.search(r"\b%s = (\d+)[;,]" % name, text)
    return int(m.group(1)) if m else default


def order_of_waits(text):
    """Whether an issuer waits for its S buffer before the barriers that both issuers use."""
    s_empty = text.index("mbar_spin(bar(kBarSEmpty + sb)")
    return s_empty < text.index("mbar_spin(bar(kBarSFull + (pj & 1))") and s_empty < text.index("mbar_spin(bar(kBarQReady)")


class Barrier:
    def __init__(self, count=1):
        self.phase, self.count, self.arrived, self.armed = 0, count, 0, False

    def arm(self):
        assert not self.armed, "armed with a load on its way"
        self.armed = True

    def arrive(self):
        self.arrived += 1
        if self.arrived == self.count:
            self.phase, self.arrived, self.armed = self.phase + 1, 0, False

    def passed(self, parity):
        return (self.phase - 1) % 2 == parity


def run(slots, per_tile, q_slots, sets, s_empty_first, seed, tiles=120):
    rng = random.Random(seed)
    # (sequence, first tile of it) of every S tile; sequences of one tile are common
    plan, seq = [], 0
    while len(plan) < tiles:
        n = rng.choice((1, 1, 2, 3, 8))
        plan += [(seq, i == 0) for i in range(n)]
        seq += 1
    full = [[Barrier() for _ in range(slots)] for _ in range(sets)]
    empty = [Barrier() for _ in range(slots)]
    s_full, s_empty = [Barrier(), Barrier()], [Barrier(), Barrier()]
    q_free, q_ready = [Barrier(), Barrier()], Barrier()
    content = [None] * slots     # what landed in a slot last
    copied = {"q": {}, "s": [None, None], "read": -1}
    loads, pipe = [], ([], [])   # in flight; each issuer's tensor operations, in order
    now = [0]

    def producer():
        use, at = [0] * slots, 0
        for jt, (sq, first) in enumerate(plan):
            own = full[jt % 2 if sets == 2 else 0]
            todo = [("q", sq, i) for i in range(q_slots)] if first else []
            for what in todo + [("c", jt, i) for i in range(per_tile)]:
                s = at % slots
                yield lambda: empty[s].passed((use[s] % 2) ^ 1)
                own[s].arm()
                late = rng.random() < 0.02
                loads.append((now[0] + (400 if late else 10 + rng.randrange(20)), s, what, own[s]))
                use[s] += 1
                at += 1

    def issuer(me):
        at, nseq, ready, q_phase, use = 0, 0, 0, 0, [0] * slots
        ops = pipe[me]

        def slot_full(s):
            phase = use[s] if sets == 2 else at // slots
            return lambda: full[me if sets == 2 else 0][s].passed(phase % 2)

        for jt, (sq, first) in enumerate(plan):
            mine, sb = jt % 2 == me, jt % 2

            def s_free():
                return s_empty[sb].passed(((jt >> 1) % 2) ^ 1)

            if mine and s_empty_first:
                yield s_free
            if first:
                nseq += 1
                if mine:
                    if jt > 0:
                        ops.append((2, q_free[me].arrive))
                        yield lambda: q_free[me].passed(q_phase)
                        q_phase ^= 1
                        yield lambda: s_full[(jt - 1) % 2].passed(((jt - 1) >> 1) % 2)
                        assert copied["s"][(jt - 1) % 2] is not None and copied["s"][(jt - 1) % 2] >= jt - 1, "Q copied over before the last GEMM1 was done"
                    for i in range(q_slots):
                        s = at % slots
                        yield slot_full(s)
                        assert content[s] == ("q", sq, i), "Q read before it landed"
                        use[s] += 1
                        ops.append((3, lambda s=s, i=i, sq=sq: (empty[s].arrive(), copied["q"].update({sq: i}))))
                        at += 1
                    ops.append((1, q_ready.arrive))
                    ready = nseq
                else:
                    at += q_slots
            if not mine:
                at += per_tile
                continue
            if ready != nseq:
                yield lambda: q_ready.passed((nseq - 1) % 2)
                assert copied["q"].get(sq) == q_slots - 1, "GEMM1 with a Q that is not copied"
                ready = nseq
            if not s_empty_first:
                yield s_free
            assert copied["read"] >= jt - 2, "S tile overwritten before it was read"
            for i in range(per_tile):
                s = at % slots
                yield slot_full(s)
                assert content[s] == ("c", jt, i), "rows read before they landed"
                use[s] += 1
                ops.append((4, empty[s].arrive))
                at += 1
            ops.append((1, lambda jt=jt: (copied["s"].__setitem__(jt % 2, jt), s_full[jt % 2].arrive())))

    def softmax():
        for jt in range(len(plan)):
            yield lambda: s_full[jt % 2].passed((jt >> 1) % 2)
            assert copied["s"][jt % 2] == jt, "softmax of another S tile"
            due = now[0] + rng.choice((2, 6, 40))
            yield lambda: now[0] >= due
            copied["read"] = jt
            s_empty[jt % 2].arrive()

    roles = [producer(), issuer(0), issuer(1), softmax()]
    waits = [next(r) for r in roles]
    busy = [0, 0]
    while any(w is not None for w in waits):
        now[0] += 1
        assert now[0] < 200000, "no role gets on"
        for load in [x for x in loads if x[0] <= now[0]]:
            loads.remove(load)
            content[load[1]] = load[2]
            load[3].arrive()
        for i in (0, 1):
            if pipe[i] and now[0] >= busy[i]:
                took, done = pipe[i].pop(0)
                done()
                busy[i] = now[0] + rng.randrange(1, took + 1)
        for i in rng.sample(range(4), 4):
            if waits[i] is not None and waits[i]():
                waits[i] = next(roles[i], None)


def decode_ring(fp8):
    tc = source("mla_tc.cuh")
    return (number(tc, "kSlotsS8" if fp8 else "kSlotsS"), 3, 9 if fp8 else 5, number(tc, "kFullSets", 1), order_of_waits(tc))


@pytest.mark.parametrize("seed", range(10))
@pytest.mark.parametrize("fp8", [False, True])
def test_decode_ring(fp8, seed):
    run(*decode_ring(fp8), seed)


@pytest.mark.parametrize("seed", range(10))
def test_tree_ring(seed):
    tree = source("mla_tree.cuh")
    assert "kBarFull1" in tree
    run(5, 3, 5, 2, order_of_waits(tree), seed)


@pytest.mark.parametrize("slots, q_slots, sets, s_empty_first", [(5, 5, 1, True), (5, 5, 2, False), (10, 9, 1, False), (10, 9, 2, False)])
def test_the_model_tells(slots, q_slots, sets, s_empty_first):
    """One set of slot barriers, or the shared barriers first, is not enough.  (Ten slots
    hold three tiles: with the S buffer's barrier first, one set would do there.)"""
    bad = 0
    for seed in range(20):
        try:
            run(slots, 3, q_slots, sets, s_empty_first, seed)
        except AssertionError:
            bad += 1
    assert bad > 0


def test_gemm2_done_before_its_slot_is_free():
    """Once a message has come through a freed slot, the slot's last kBarMmaDone phase is
    known to be complete only if its commit came before the one that freed the slot."""
    for name in ("mla_tc.cuh", "mla_tree.cuh"):
        text = source(name)
        assert text.index("bar(kBarMmaDone + ms)") < text.index("bar(kBarPFree + ms), 0x3")
