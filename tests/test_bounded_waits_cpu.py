"""Waits whose verdict several warps or lanes act on, read from the kernels' sources.

A wait that runs out must end the kernel, not hang it: a warp that left its loop
early would leave the others at a named barrier for good, and lanes that disagree
would leave a warp-wide instruction without some of them.
"""

from __future__ import annotations

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "myelin_b200" / "csrc"


def _code(name: str) -> str:
    return re.sub(r"//[^\n]*", "", (CSRC / name).read_text())


def _workers(code: str, kernel: str) -> str:
    """The branches of a kernel whose warps work with all their lanes."""

    body = code[code.index(f"{kernel}(const"):]
    return body[body.index("} else if (warp < 12) {"):body.index("tmem_free(tmem, warp);")]


def test_warps_that_share_named_barriers_run_their_loops_to_the_end():
    workers = _workers(_code("decay_attention_tc.cu"), "attn_out_kernel")
    assert workers.count("bar_sync(") >= 4
    assert "break;" not in workers and "&& ok; unit" not in workers


@pytest.mark.parametrize("kernel", ["attn_out_kernel", "attn_states_kernel"])
def test_worker_warps_go_on_after_a_wait_that_ran_out(kernel):
    workers = _workers(_code("decay_attention_tc.cu"), kernel)
    assert workers.count("Waits wait;") == 2 and "mbar_wait_bounded(" not in workers


@pytest.mark.parametrize("name", ["gemm_i8.cu", "gemm_tcgen05.cu"])
def test_drain_warps_go_on_after_a_wait_that_ran_out(name):
    code = _code(name)
    assert code.count("    wait(&acc_full[b]") == code.count("Waits wait;") == 2
    assert "mbar_wait_bounded(&acc_full[b]" not in code
