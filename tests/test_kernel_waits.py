"""Bounded waits of the cross-attention kernels, read in their source: a wait that runs out ends for a whole warp at once.

A lane that gave up alone would be missing from the warp's next vote, shuffle or tensor-memory access, and the rest would
wait for it without end, so nothing of this may run on a GPU."""

import heapq
import os
import random
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "csrc")


@pytest.mark.parametrize("name,start,end", [
    ("cross_attn.cuh", "} else if (warp == C::kCleanWarp) {", "tmem_dealloc(tmem, C::kTmemCols)"),  # the cleaning and softmax warps
    ("cross_decode.cu", "uint4 qf[KC][NB];", "decode_join<DH, F16>(a, hk"),  # the warps that walk the keys
])
def test_waits_of_whole_warps_have_one_outcome(name, start, end):
    with open(os.path.join(CSRC, name)) as f:
        source = f.read()
    part = source[source.index(start):]
    part = part[:part.index(end)]
    assert re.findall(r"mbar_wait_warp\(", part) and not re.findall(r"mbar_wait\(", part)


class _Barrier:
    """Phases as an mbarrier shows them: a wait names a parity, and passes when the last completed phase has it."""

    def __init__(self):
        self.phase = 0

    def passed(self, parity):
        return (self.phase & 1) != parity

    def complete(self):
        self.phase += 1


def _ring(slots, tiles, latency, rng):
    """The K / V ring of the cross-attention kernel with cleaning: load L = 2 s (K of step s) or 2 s + 1 (V) goes to slot
    L % slots; copies land after 1 .. latency steps' shares, in any order.  Returns (finished, loads cleaned before they landed)."""
    full, empty, clean = ([_Barrier() for _ in range(slots)] for _ in range(3))
    scores, weights = _Barrier(), _Barrier()
    holds, early, events = [None] * slots, [], []

    def later(delay, what):
        heapq.heappush(events, (now[0] + delay, len(order), what))
        order.append(what)

    now, order = [0.0], []

    def producer():
        for load in range(2 * tiles):
            s = load % slots
            while not empty[s].passed(((load // slots) & 1) ^ 1):
                yield

            def land(s=s, load=load):
                holds[s] = load
                full[s].complete()

            later(rng.uniform(1, latency), land)
            yield

    def cleaner():
        for step in range(tiles):
            load = 2 * step + 1
            while not full[load % slots].passed((load // slots) & 1):
                yield
            if holds[load % slots] != load:
                early.append(load)
            clean[load % slots].complete()
            yield

    def multiplier():
        parity = [0] * slots
        for step in range(tiles + 1):
            if step < tiles:
                while not full[2 * step % slots].passed((2 * step // slots) & 1):
                    yield
            if step:
                load = 2 * step - 1
                while not full[load % slots].passed((load // slots) & 1):
                    yield
                while not clean[load % slots].passed(parity[load % slots]):
                    yield
                parity[load % slots] ^= 1
                while not weights.passed((step - 1) & 1):
                    yield
                later(0.2, empty[load % slots].complete)
            if step < tiles:
                later(0.2, scores.complete)
                later(0.2, empty[2 * step % slots].complete)
            yield

    def softmax():
        for step in range(tiles):
            while not scores.passed(step & 1):
                yield
            later(rng.uniform(0.2, 1), weights.complete)
            while not weights.passed(step & 1):
                yield

    roles = [producer(), cleaner(), multiplier(), softmax()]
    while True:
        for _ in range(3):
            for role in list(roles):
                try:
                    next(role)
                except StopIteration:
                    roles.remove(role)
        if not roles or not events:
            return not roles, early
        now[0], _, what = heapq.heappop(events)
        what()


def _ring_slots():
    """Slots per (head dim, Q tiles) as the kernel's source states them."""
    with open(os.path.join(CSRC, "cross_attn.cuh")) as f:
        line = next(li for li in f if "static constexpr int kRing" in li)
    expr = line.split("=", 1)[1].split(";")[0]
    expr = re.sub(r"(.+?)\?(.+?):(.+)", r"(\2 if \1 else (\3))", expr)
    expr = re.sub(r"\((\w+ == \d+) \?(.+?):(.+?)\)", r"(\2 if \1 else (\3))", expr)
    return {(dh, qt): eval(expr, {"DH": dh, "QT": qt}) for dh in (64, 128) for qt in (1, 2)}


@pytest.mark.parametrize("latency", [1.5, 6, 40])
def test_the_ring_survives_copies_that_land_out_of_order(latency):
    """The cleaning warp waits for the V loads alone, by parity: in a ring of an odd number of slots K and V alternate in a slot, and
    its wait passes on the phase before (or misses its own) when copies land out of order; the kernel then stands still."""
    for slots in set(_ring_slots().values()):
        for seed in range(150):
            assert _ring(slots, 12, latency, random.Random(seed)) == (True, [])
    if latency > 2:
        assert any(_ring(5, 12, latency, random.Random(seed)) != (True, []) for seed in range(150))
