"""Waits in the packed operators' kernels, by reading their sources: a warp that
gives up after a timeout leaves its loop, so nothing may wait for it without a
limit."""

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "dit_sparse_atten_b200" / "csrc"
PACKED = ["lora.cu", "residual_norm.cu", "packed_attention.cu", "packed_attention.cuh", "packed_common.cuh"]


def code(name):
    """The source without its comments."""
    return re.sub(r"//[^\n]*", "", (CSRC / name).read_text())


@pytest.mark.parametrize("name", PACKED)
def test_no_wait_without_a_limit(name):
    """Whole-block and whole-cluster barriers, which every thread reaches, and
    mbar_wait; no wait of its own, and some of the warps meet only to agree
    whether to go on (bar.red), in one place a file."""
    text = code(name)
    assert not re.search(r"\bbar\.sync|\bbarrier\.sync|named_bar_sync|\btry_wait|\btest_wait", text)
    assert text.count("bar.red") == (name == "lora.cu")
