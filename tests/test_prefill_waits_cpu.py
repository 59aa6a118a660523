"""What the prompt kernel's roles do when a bounded wait runs out, as models that take the
places of votes and counts from the kernel's source."""
import os
import random
import re

import pytest

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ada-mla_b200", "csrc", "mla_prefill.cuh")


def role(first, last):
    """The source between two comments, without comments and white space."""
    with open(SOURCE) as f:
        text = f.read()
    text = text[text.index(first):text.index(last)]
    return re.sub(r"\s+", "", re.sub(r"//[^\n]*", "", text))


def issuer_votes_after_item():
    """Whether the issuing warp agrees on `ok` between an item's last wait and the next item."""
    text = role("-- MMA issuers", "-- V tail")
    return "ok=__all_sync(0xffffffffu,ok);}if(!" in text


def vote(lanes, site_of):
    """All lanes that still run meet at one vote: the sites they come to must be the same."""
    assert len({site_of(i) for i in lanes}) == 1, "lanes of a warp vote in different places"


@pytest.mark.parametrize("seed", range(50))
def test_issuer_lanes_stay_together(seed):
    """Each lane reads the clock itself, so one lane's wait may run out and another's not."""
    rng = random.Random(seed)
    lanes, after = range(32), issuer_votes_after_item()
    items = [(n, n + rng.choice((0, 0, 1, 2))) for n in (rng.randrange(0, 4) for _ in range(6))]
    runs_out = rng.randrange(1, 12)  # the wait at which some lanes give up
    ok = [True] * 32
    waits = [0]

    def wait():
        waits[0] += 1
        if waits[0] == runs_out:
            some = rng.randrange(1, 32)
            for i in rng.sample(lanes, some):
                ok[i] = False

    for n, nmax in items:
        # the vote inside next_item(), or the exit's, by each lane's own flag
        vote(lanes, lambda i: "next" if ok[i] else "exit")
        if not ok[0]:
            return
        if n > 0:
            wait()
        for j in range(n):
            ok = [all(ok)] * 32  # the vote at the head of a tile
            if not ok[0]:
                break
            wait()
        if n < nmax:
            wait()
        if after:
            ok = [all(ok)] * 32


def counts_on_success():
    """Whether the producer counts a slot only once it has it, and takes none back."""
    text = role("-- TMA producer", "-- MMA issuers")
    return "if(ok)++at;" in text and "--at" not in text


@pytest.mark.parametrize("fails", ["slot", "q"])
@pytest.mark.parametrize("before", [0, 1, 7, 8, 9, 20])
def test_producer_drains_every_load(fails, before):
    """After a wait that ran out, for a slot or for Q's buffer, the producer waits for the
    loads it has issued: the last eight slots' may be on their way."""
    slots, success = 8, counts_on_success()
    at = before
    if not success:
        at += 1 if fails == "slot" else 0  # counted before the wait ran out
        at -= 1
    drained = set(range(max(at - slots, 0), at))
    assert set(range(max(before - slots, 0), before)) <= drained
