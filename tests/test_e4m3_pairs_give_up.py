"""A pair of blocks that gives up leaves when, and not before, every copy that either asked for has landed: what the first block does
with the stages' barriers, followed on the host through every state that the two producers can stop in."""
import ctypes
import os
import random
import subprocess

import pytest

import harness as H  # noqa: F401  (path setup)

STAGES, HALF = 6, 1 << 15       # (a block's bytes of a stage)
SOURCE = """
#include "e4m3_tc.cuh"
int leb_fail(const char*, ...) { return 1; }
LEB_API int first_out(int own, int theirs, int stages) { return e8_first_out(own, theirs, stages); }
LEB_API int owed(int i, int own, int theirs, int half) { return e8_owed(i, own, theirs, half); }
"""


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    """The functions that the kernel calls, compiled for the host."""
    from lastengine_b200.ops import build
    d = tmp_path_factory.mktemp("pairs")
    (d / "plan.cu").write_text(SOURCE)
    so = str(d / "plan.so")
    subprocess.run([build._find_nvcc(), *build.NVCC_FLAGS, "-I", build.CSRC, "-shared", "-o", so, str(d / "plan.cu")], check=True, timeout=300)
    return ctypes.CDLL(so)


class Barrier:
    """One arrival and any number of bytes a phase, as the stages' barriers are; bytes may land before they are announced."""

    def __init__(self):
        self.phase, self.pending, self.bytes = 0, 1, 0

    def _ends(self):
        if self.pending == 0 and self.bytes == 0:
            self.phase, self.pending = self.phase + 1, 1

    def announce(self, n):
        self.bytes += n
        self.pending -= 1
        assert self.pending == 0
        self._ends()

    def land(self, n):
        self.bytes -= n
        self._ends()

    def passed(self, phase):          # a test of the phase's parity
        return (self.phase - 1) & 1 == phase & 1


def states():
    """(stages whose products are done, stages the first block asked for, stages the other did): a stage is asked for again once its products are
    done, and products need both halves."""
    for done in range(0, 2 * STAGES + 2):
        for own in range(done, done + STAGES + 1):
            for theirs in range(done, done + STAGES + 1):
                yield done, own, theirs


def test_a_pair_leaves_when_all_copies_have_landed(plan):
    rng = random.Random(5)
    ahead = 0
    for done, own, theirs in states():
        for _ in range(6):
            bars = [Barrier() for _ in range(STAGES)]
            flying = []
            for i in range(max(own, theirs)):
                b = bars[i % STAGES]
                asked = [i < own, i < theirs]
                copies = [b] * sum(asked)
                steps = [lambda b=b: b.announce(2 * HALF)] if asked[0] else []
                early = len(copies) if i < done else rng.randint(0, len(copies))
                steps += [lambda b=b: b.land(HALF)] * early
                rng.shuffle(steps)
                for s in steps:
                    s()
                flying += copies[early:]
            most = max(own, theirs)
            begin = plan.first_out(own, theirs, STAGES)
            assert 0 <= begin <= most and most - begin <= STAGES and begin <= done
            for i in range(begin, most):
                n = plan.owed(i, own, theirs, HALF)
                if n > 0:
                    bars[i % STAGES].announce(n)
                if n < 0:
                    bars[i % STAGES].land(-n)
            may_leave = lambda: all(bars[i % STAGES].passed(i // STAGES) for i in range(begin, most))  # noqa: E731
            rng.shuffle(flying)
            while flying:
                assert not may_leave(), (done, own, theirs, len(flying))
                flying.pop().land(HALF)
            assert may_leave(), (done, own, theirs)
            ahead += theirs > own
    assert ahead > 500
