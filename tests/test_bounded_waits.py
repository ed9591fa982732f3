"""Waits in the kernels, by reading their sources: a warp that gives up after a
timeout leaves its loop, so nothing may wait for it without a limit, and what
is in flight is waited for all the same."""

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
    whether to go on (named_bar_and)."""
    text = code(name)
    assert not re.search(r"\bbar\.sync|\bbarrier\.sync|named_bar_sync|\btry_wait|\btest_wait", text)
    assert "bar.red" not in text


def test_producers_count_their_loads_in_one_place():
    """lora.cu's producers wait, when they give up, for the loads that their ring
    has counted, and a ring counts behind an issued load only."""
    text = code("lora.cu")
    assert len(re.findall(r"LoadRing<", text)) == 3 == len(re.findall(r"\.arm\(\)", text))
    assert len(re.findall(r"for_each_open\(", text)) == 3
    assert not re.search(r"for \(int j = [^;]*>", text)      # no window of its own
    assert not re.search(r"\*abort_flag\) *{", text)         # whoever gives up, and whenever


@pytest.mark.parametrize("slots", [1, 2, 3, 4, 8])
@pytest.mark.parametrize("loads", range(0, 27))
def test_ring_of_loads(slots, loads):
    """Against barriers that complete phase after phase: a load waits for the
    phase that its slot's last reader completes, and after the last load exactly
    the last one of each slot is waited for, at its own phase."""
    import diag
    taken, open_ = diag.load_ring(slots, loads)
    phases = [0] * slots                    # loads of each slot so far
    for j, (slot, parity) in enumerate(taken):
        assert slot == j % slots
        # phase k of "empty" completes when load k of the slot has been read; the
        # wait before load k is for phase k - 1, and passes at once for k = 0
        assert parity == (phases[slot] - 1) % 2
        phases[slot] += 1
    assert sorted(s for s, _ in open_) == [s for s in range(slots) if phases[s]]
    for slot, parity in open_:
        assert parity == (phases[slot] - 1) % 2


@pytest.mark.parametrize("name", sorted(p.name for p in CSRC.glob("*.cu")))
def test_last_waits_have_their_own_limit(name):
    """A wait that must outlast an abort does not go by the abort flag's rules."""
    text = code(name)
    for call in re.findall(r"mbar_wait\([^;]*;", text):
        assert re.search(r",\s*(abort_flag|&abort_flag)\s*,", call), call
    assert len(re.findall(r"int late = 0;", text)) <= len(re.findall(r"mbar_drain\(", text))


def test_pair_kernel_leaves_its_loop_together():
    """The halves of a row meet once a block inside the loop; no way out of the
    loop lies before that meeting."""
    text = code("attention_pair.cu")
    loop = text[text.index("for (int j = 0; ok && j < n; ++j) {"):]
    loop = loop[:loop.index("named_bar_and(pair_bar, 64, ok)")]
    assert re.findall(r"[^\n]*break;", loop) == ["      if (kHalves == 1 && !ok) break;"]


@pytest.mark.parametrize("kernel", ["lora_expand_few_kernel", "lora_expand_tiles_kernel"])
def test_dependent_kernels_outlast_the_one_before(kernel):
    """A kernel that may start while the one before it runs waits for that one on
    every way out: the caller frees the workspace, and the next kernel of the
    stream starts, when this one ends."""
    text = code("lora.cu")
    body = re.search(kernel + r"\([^{]*\{\n(.*?)\n\}\n", text, re.S).group(1)
    before = [body[:m.start()].rstrip() for m in re.finditer(r"\breturn;", body)]
    assert before and all(b.endswith("pdl_wait();") for b in before)
    assert len(re.findall(r"pdl_wait\(\);", body)) >= len(before) + 1      # and the ordinary way
