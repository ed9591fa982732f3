"""Values that are not finite at keys which some of a request's queries see and
some do not (``kernels.packed_attention``, causal): they reach exactly the
features of the queries that see them, every other result keeps its bits, and
the call costs no key-by-key way out."""

import pytest
import torch

from test_gpu_packed_attention import DEV, call, make

pytestmark = pytest.mark.gpu
NAN, INF = float("nan"), float("inf")


def not_finite(t):
    """Which results are NaN, +inf and -inf: a weight is positive, so a feature
    is what the values that its query sees add up to."""
    v, heads = t["v"], t["q"].shape[1]
    qs, ks = t["qs"].tolist(), t["ks"].tolist()
    out = torch.zeros(t["q"].shape, device=DEV)
    for s in range(len(qs) - 1):
        n, m = qs[s + 1] - qs[s], ks[s + 1] - ks[s]
        one = v[ks[s]:ks[s + 1]].float()
        one = torch.where(one.isfinite(), 0.0, one)
        seen = torch.cat([torch.zeros_like(one[:1]), one.cumsum(0)])      # inf - inf and NaN stay NaN
        limit = (torch.arange(n, device=DEV) + 1 + m - n).clamp(0, m)
        out[qs[s]:qs[s + 1]] = seen[limit].repeat_interleave(heads // v.shape[1], 1)
    return out


def check(t, clean):
    out, want = call(t, causal=True), not_finite(t)
    finite = want == 0
    assert (~finite).any() and torch.equal(out[finite], clean[finite])
    assert torch.equal(out[~finite].float().nan_to_num(1.0, 2.0, 3.0), want[~finite].nan_to_num(1.0, 2.0, 3.0))


CASES = [
    ([400], [400], 1, 1), ([256], [256], 2, 1), ([300, 40], [300, 40], 8, 1), ([200, 77], [150, 77], 6, 2),
    ([9, 5], [9, 130], 128, 1),                       # items of both tiles
    ([4], [3000], 4, 1), ([7, 1, 2], [2500, 4000, 1300], 5, 1),      # parts of keys, paired tiles
    ([70, 17], [4000, 2051], 16, 2), ([300], [5000], 2, 2),          # parts of keys, both tiles
]


@pytest.mark.parametrize("q_lengths,k_lengths,heads,kv_heads", CASES)
@pytest.mark.parametrize("seed", range(4))
def test_reach_only_what_sees_them(q_lengths, k_lengths, heads, kv_heads, seed):
    """Single elements among the last keys, and a few that every query sees."""
    t = make(q_lengths, k_lengths, heads, kv_heads, seed=seed)
    clean = call(t, causal=True)
    g = torch.Generator().manual_seed(100 + seed)
    begin = 0
    for n, m in zip(q_lengths, k_lengths):
        for i in range(2 + 4 * seed):
            back = int(torch.randint(1, min(n, m) + (2 if i == 0 else 0) + 1, (1,), generator=g))
            key, head = begin + m - min(back, m), int(torch.randint(0, kv_heads, (1,), generator=g))
            feature = int(torch.randint(0, 128 if seed < 3 else 4, (1,), generator=g))
            t["v"][key, head, feature] = (NAN, INF, -INF)[int(torch.randint(0, 3, (1,), generator=g))]
        begin += m
    check(t, clean)


@pytest.mark.parametrize("q_lengths,k_lengths,heads,kv_heads", CASES)
@pytest.mark.parametrize("value", [NAN, INF, -INF])
def test_whole_rows(q_lengths, k_lengths, heads, kv_heads, value):
    """Every value of the first request's last keys, as many as it has queries."""
    t = make(q_lengths, k_lengths, heads, kv_heads, seed=9)
    clean = call(t, causal=True)
    m = k_lengths[0]
    t["v"][m - min(q_lengths[0], m):m] = value
    check(t, clean)


def test_infinities_of_both_signs_meet():
    t = make([130], [130], 3, 3, seed=2)
    clean = call(t, causal=True)
    t["v"][3, 1, 7] = INF
    t["v"][100, 1, 7] = -INF
    t["v"][129, 2] = -INF
    check(t, clean)


def test_long_past():
    """300 new tokens over 262,144 keys, an infinity in the last one."""
    t = make([300], [262144], 1, 1, seed=3)
    clean = call(t, causal=True)
    t["v"][-1, 0, 5] = INF
    t["v"][-100, 0, 70] = NAN
    check(t, clean)


def test_a_broken_request_takes_no_longer():
    """8,192 causal tokens, half of the values NaN: the time of finite ones, but
    for the look at the keys on the diagonal (recomputing the rows that have one
    key by key would take hundreds of times as long)."""
    t = make([8192], [8192], 8, 1, seed=4)
    clean = call(t, causal=True)

    def microseconds():
        times = []
        for _ in range(5):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            call(t, causal=True)
            b.record()
            b.synchronize()
            times.append(a.elapsed_time(b) * 1e3)
        return min(times)
    before = microseconds()
    t["v"][4096:] = NAN
    check(t, clean)
    assert microseconds() <= 8 * before
