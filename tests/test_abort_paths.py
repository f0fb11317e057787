"""Source-level check of what the block-scaled product does after a wait that ran out (no GPU needed, and none could be made
to fail there: nothing in these kernels' protocol can be left unset from outside).

A role that gives up must do so as a whole warp: the instructions that follow a wait (elect.sync, tcgen05.ld) need every lane,
and lanes that left the loop alone would leave the others waiting.  And what is under way has to end before the CTA frees its
tensor memory and leaves: loads write into its shared memory, MMAs read it and write tensor memory.
"""

from __future__ import annotations

import pathlib
import re

import pytest

from test_launch_rule import CSRC, _kernel_bodies

SOURCE = pathlib.Path(CSRC) / "gemm_fp8.cu"


@pytest.mark.parametrize("kernel", ["gemm_fp8_kernel", "gemm_fp8_few_kernel"])
def test_a_warp_gives_up_as_a_whole(kernel) -> None:
    body = _kernel_bodies(SOURCE.read_text())[kernel]
    alone = re.search(r"if \(rank == 0 && ptx::elect_one\(\)\) \{.*?\n      \}\n", body, re.S)
    if alone:  # a role that one lane runs needs no agreement, and must ask for none
        assert "_sync(0x" not in alone.group(0) and "elect_one" not in alone.group(0)[40:]
        body = body.replace(alone.group(0), "")
    waits = [m.end() for m in re.finditer(r"mbar_wait\(", body)]
    assert len(waits) >= 3
    for at in waits:
        # From the wait on: a vote comes before the first branch that leaves on the result.
        leaves = re.search(r"if \([^)\n]*!ok\) (break|return)|if \(!ok\) \{|&& ok; [^)]*\) \{", body[at:])
        assert leaves, body[at:at + 200]
        between = body[at:at + leaves.start()]
        assert "__all_sync(0xFFFFFFFFu, ok)" in between, f"{kernel}: lanes may leave alone after {body[at - 40:at + 120]}"


@pytest.mark.parametrize("kernel", ["gemm_fp8_kernel", "gemm_fp8_few_kernel"])
def test_what_is_under_way_is_waited_for(kernel) -> None:
    body = _kernel_bodies(SOURCE.read_text())[kernel]
    assert re.search(r"if \(!ok[^)]*\) drain_loads", body)
    assert re.search(r"if \(!ok( && ptx::elect_one\(\))?\) drain_mmas", body), f"{kernel}: tensor memory is freed while MMAs may write it"
    # ... before the tensor memory is freed.
    assert body.index("drain_mmas") < body.index("tmem_dealloc")
    assert "mbar_init(bar_done, 1)" in body


def test_drains_are_bounded() -> None:
    text = SOURCE.read_text()
    for name in ("drain_loads", "drain_mmas"):
        start = text.index(f"void {name}(")
        body = text[start:text.index("\n}\n", start)]
        assert re.search(r"globaltimer_ns\(\) - start < \w+", body), name
