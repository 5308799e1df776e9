"""Waits and shared memory of the attention kernels, as their sources have them: what happens once a bounded wait has run out cannot be tried on a GPU that others share."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(__file__), "..", "linear_moe_b200", "csrc")


def kernel(file, name):
    """The text of a kernel, from its parameters to the next function of the file."""
    text = open(os.path.join(CSRC, file)).read()
    text = text[re.search(r"\b%s\(" % name, text).end():]
    return text[:re.search(r"^}", text, re.M).start()]


@pytest.mark.parametrize("name", ["scored_fwd_kernel", "scored_dq_kernel", "scored_dkv_kernel"])
def test_a_warp_leaves_a_wait_as_a_whole(name):
    """Behind a wait come instructions of the whole warp (tcgen05.ld, reductions): only warp 0, one lane of which issues the loads, decides lane by lane."""
    text = kernel("flash_attn_scored.cuh", name)
    loads = re.search(r"if \(warp == 0\) \{\n\s+if \(lane == 0\) \{.*?\} else if \(warp == 1", text, re.S)
    assert loads and "wait_for(" in loads.group()
    assert not re.search(r"\bwait_for\(", text[:loads.start()] + text[loads.end():])
    assert re.search(r"\bwait_warp\(", text[loads.end():])


def test_gradients_behind_a_wait_that_ran_out_are_nan():
    """Zeros are what keys get that nobody sees; where a CTA or its partner gave up, dk and dv must not look like that."""
    text = kernel("flash_attn_scored.cuh", "scored_dkv_kernel")
    out = text[text.index("given = reinterpret_cast"):]
    assert not re.search(r"alive \? pack16<F>\([^?]*\) : 0u", out)
    assert re.search(r"n_it == 0 \? 0u", out) and re.search(r"alive \? pack16<F>.* : NAN16", out)
    sent = out[:out.index("rows_out")]
    assert re.search(r"theirs\[c / 4 \* 512\] = alive \?", sent)          # the partner's half of a sum


def test_lengths_lie_beside_the_rings():
    """The one-token kernel's list of lengths is written and read by ordinary accesses: not where bulk copies go next without a fence between the two."""
    text = kernel("paged_step.cu", "paged_step_kernel")
    assert re.search(r"__shared__ int [^;]*\blens\[WARPS \* 32\]", text)
    assert not re.search(r"int\* lens", text)
