"""The rings of the packed-word tiles (scaled_config.h) under every order in which copies can land: a model of the barriers, their
parity waits and the agents that share them, with the counts of the compiled configuration.  Nobody may read words that have
not landed, write over decoded weights that are still to be multiplied, or multiply what is not there."""
import os
import random
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
#include <cstdio>
#include "scaled_config.h"
template <int WK, int BN> void show() {
    using C = tmq::ScaledCfg<WK, BN>;
    std::printf("%d %d %d %d %d %d\n", WK, BN, C::RAW_STAGES, C::SETS / 2, C::NA, C::RAWK / C::KB);
}
template <int WK> void all() { show<WK, 32>(); show<WK, 64>(); show<WK, 128>(); show<WK, 256>(); }
int main() { all<tmq::W_TERNARY_BF16>(); all<tmq::W_TERNARY_I8>(); }
"""


@pytest.fixture(scope="module")
def configurations(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("needs a host compiler")
    d = tmp_path_factory.mktemp("rings")
    (d / "show.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-I", os.path.join(ROOT, "include"), "-I", os.path.join(ROOT, "tmq_b200", "csrc"),
                    str(d / "show.cpp"), "-o", str(d / "show")], check=True)
    out = subprocess.run([str(d / "show")], check=True, capture_output=True, text=True).stdout
    return [tuple(int(v) for v in line.split()) for line in out.splitlines()]


class Barrier:
    """One arrival per phase; a parity wait passes when the phase of that parity is the last that ended."""

    def __init__(self):
        self.ended = 0

    def arrive(self):
        self.ended += 1

    def passed(self, parity):
        return (self.ended & 1) != (parity & 1)


def fault(raw_slots, pairs, slots, stages_per_box, units, stages, rng):
    """A fault that one schedule shows, or None.  A unit has `stages` stages, whose packed words come in boxes."""
    boxes = []
    for _ in range(units):
        left = stages
        while left > 0:
            boxes.append(min(stages_per_box, left))
            left -= stages_per_box
    first = [0]
    for n in boxes:
        first.append(first[-1] + n)
    raw_full, raw_empty = [Barrier() for _ in range(raw_slots)], [Barrier() for _ in range(raw_slots)]
    ready, taken = [Barrier() for _ in range(slots)], [Barrier() for _ in range(slots)]
    words, weights, flying, done, seen = [None] * raw_slots, [None] * slots, [], [0], []

    def producer():
        for b in range(len(boxes)):
            s, use = b % raw_slots, b // raw_slots
            while not raw_empty[s].passed((use & 1) ^ 1):
                yield False
            flying.append(b)
            words[s] = None
            yield True

    def copies():
        while True:
            if flying:
                b = flying.pop(rng.randrange(len(flying)))
                words[b % raw_slots] = b
                raw_full[b % raw_slots].arrive()
            yield bool(flying)

    def decoders(p):
        for b in range(p, len(boxes), pairs):
            s, use = b % raw_slots, b // raw_slots
            for t in range(first[b], first[b + 1]):
                landed = free = False                          # half of the lanes watch each of the two
                while not (landed and free):
                    landed = landed or raw_full[s].passed(use & 1)
                    free = free or taken[t % slots].passed(((t // slots) & 1) ^ 1)
                    if not (landed and free):
                        yield False
                if words[s] != b:
                    seen.append(("words that have not landed", b))
                if weights[t % slots] is not None:
                    seen.append(("weights still to be multiplied", t))
                weights[t % slots] = t
                yield True
                ready[t % slots].arrive()
            raw_empty[s].arrive()
            yield True

    def products():
        for t in range(first[-1]):
            while not ready[t % slots].passed((t // slots) & 1):
                yield False
            if weights[t % slots] != t:
                seen.append(("weights that are not there", t))
            weights[t % slots] = None
            yield True
            taken[t % slots].arrive()
            done[0] = t + 1

    agents = [producer(), copies(), products()] + [decoders(p) for p in range(pairs)]
    pace = [0.02 + rng.random() for _ in agents]
    idle = 0
    while done[0] < first[-1]:
        i = rng.choices(range(len(agents)), pace)[0]
        try:
            idle = 0 if next(agents[i]) else idle + 1
        except StopIteration:
            agents.pop(i)
            pace.pop(i)
        if seen:
            return seen[0]
        if idle > 3000:
            return ("nobody moves", done[0])
    return None


def schedules(raw_slots, pairs, slots, per_box, count, seed):
    rng = random.Random(seed)
    for _ in range(count):
        found = fault(raw_slots, pairs, slots, per_box, rng.choice([3, 7, 11]), rng.choice([1, 1, 2, 3, 4, 8]), rng)
        if found:
            return found
    return None


def test_every_configuration_is_free_of_faults(configurations):
    assert len(configurations) == 8
    for wk, bn, raw_slots, pairs, slots, per_box in configurations:
        assert schedules(raw_slots, pairs, slots, per_box, 500, bn + wk) is None, (wk, bn)


def test_the_model_finds_an_odd_ring_shared_by_two_pairs():
    assert schedules(3, 2, 4, 2, 500, 1) is not None
