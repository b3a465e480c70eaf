"""Barrier protocol of the dense GEMM kernels (csrc/dense_gemm.cu and
csrc/dense_skinny.cu: a ring of stages, two accumulators), restated on the CPU.

An arrival that nobody waits for may reach a CTA's shared memory after the CTA
has left. The barriers here are as slow as they may be: an arrival lands only
when a wait cannot pass without it. What is still on its way when a CTA's roles
have ended is then exactly what nobody waited for, and must be nothing.
"""
from __future__ import annotations

import os
import re

import pytest


class Barrier:
    """A barrier of one arrival per phase; `posted` arrivals are on their way."""

    def __init__(self):
        self.phases = 0
        self.posted = 0

    def post(self):
        self.posted += 1

    def wait(self, parity):
        """Passes once the phase of that parity is complete."""
        while self.phases & 1 == parity:
            assert self.posted > 0, "waits for an arrival that never comes"
            self.posted -= 1
            self.phases += 1


def pair_producer(steps, stages, early, tail=True):
    """Empty-stage barriers of either CTA of a pair after its producer and the
    MMAs of `steps` K steps in all; B of the first `early` steps is requested
    ahead without a wait."""
    empty = [Barrier() for _ in range(stages)]
    stage, ph = 0, 0
    for i in range(steps):
        if i >= early:
            empty[stage].wait(ph ^ 1)
        empty[stage].post()          # the MMAs of this step hand the stage back
        stage += 1
        if stage == stages:
            stage, ph = 0, ph ^ 1
    for _ in range(stages if tail else 0):
        empty[stage].wait(ph ^ 1)
        stage += 1
        if stage == stages:
            stage, ph = 0, ph ^ 1
    return empty


def streaming_producer(steps, stages, tail=True):
    """The same for the streaming form: the first ring is requested at once."""
    empty = [Barrier() for _ in range(stages)]
    first = min(stages, steps)
    for i in range(first):
        empty[i].post()
    stage, ph = (0 if first == stages else first), 0
    for _ in range(first, steps):
        empty[stage].wait(ph)
        empty[stage].post()
        stage += 1
        if stage == stages:
            stage, ph = 0, ph ^ 1
    for i in range(steps - first, steps if tail else 0):
        empty[i % stages].wait((i // stages) & 1)
    return empty


def on_the_way(barriers):
    return sum(b.posted for b in barriers)


@pytest.mark.parametrize("stages", [1, 2, 5, 7, 12])
def test_every_stage_is_awaited(stages):
    for steps in range(1, 4 * stages + 3):
        for early in {0, min(1, steps), min(stages, steps)}:
            assert on_the_way(pair_producer(steps, stages, early)) == 0
        assert on_the_way(streaming_producer(steps, stages)) == 0
        # without the closing waits a ring, or what there was of it, is left
        assert on_the_way(pair_producer(steps, stages, 0, tail=False)) == min(steps, stages)
        assert on_the_way(streaming_producer(steps, stages, tail=False)) == min(steps, stages)


@pytest.mark.parametrize("shared_columns", [False, True])
def test_every_accumulator_is_awaited(shared_columns):
    """Arrivals between MMAs and epilogue: `shared_columns` (4-bit) hands every
    accumulator to the next tile through one barrier, otherwise each
    accumulator has its own and serves every other tile."""
    for tiles in range(1, 12):
        complete = [Barrier(), Barrier()]
        handed = [Barrier(), Barrier()]
        for it in range(tiles):
            buf = it & 1
            if shared_columns:
                if it >= 1:
                    handed[0].wait((it - 1) & 1)
            elif it >= 2:
                handed[buf].wait(((it >> 1) - 1) & 1)
            complete[buf].post()
            complete[buf].wait((it >> 1) & 1)                    # epilogue
            if it + (1 if shared_columns else 2) < tiles:        # a tile to come needs the columns
                handed[0 if shared_columns else buf].post()
        assert on_the_way(complete + handed) == 0


def _kernels():
    """(name, text) of every kernel of the dense operators."""
    here = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    for name in ("dense_gemm.cu", "dense_skinny.cu", "mxfp4.cu"):
        with open(os.path.join(here, "flashinfer-bench-avengers_b200", "csrc", name)) as f:
            text = f.read()
        for m in re.finditer(r"^(__global__[^;{]*?(\w+_kernel)\([^;{]*\) \{\n)(.*?)^\}", text, re.M | re.S):
            yield m.group(2), m.group(3)


def test_kernels_wait_before_they_let_the_next_one_start():
    """Weights are read ahead of a kernel's wait, behind another kernel of the
    same call: whatever wrote them is complete because that one has waited
    before it let this one start."""
    seen = dict(_kernels())
    assert set(seen) == {"dense_pair_kernel", "dense_skinny_kernel", "mxfp4_quantize_kernel", "mxfp4_gate_kernel",
                         "mxfp4_dequantize_kernel"}
    for name, body in seen.items():
        assert 0 <= body.find("pdl_wait();") < body.find("pdl_launch_next();"), name
