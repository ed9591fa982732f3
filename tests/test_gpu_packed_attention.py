"""``kernels.packed_attention`` on a B200 against the float64 definition
(``oracle/packed.py``)."""

import numpy as np
import pytest
import torch

from dit_sparse_atten_b200 import _native, kernels
from oracle import packed as opacked

pytestmark = pytest.mark.gpu
DEV = "cuda"
U16 = 2.0 ** -8     # rounding to bf16, relative
U32 = 2.0 ** -24


def starts_of(lengths):
    return torch.tensor(np.cumsum([0] + list(lengths)), dtype=torch.int32, device=DEV)


def make(q_lengths, k_lengths, heads, kv_heads, seed=0, std=1.5):
    g = torch.Generator().manual_seed(seed)

    def rnd(rows, h, s=1.0):
        return (torch.randn((rows, h, 128), generator=g) * s).to(torch.bfloat16).to(DEV)
    return dict(q=rnd(sum(q_lengths), heads, std), k=rnd(sum(k_lengths), kv_heads),
                v=rnd(sum(k_lengths), kv_heads), qs=starts_of(q_lengths), ks=starts_of(k_lengths))


def call(t, **kw):
    out = kernels.packed_attention(t["q"], t["k"], t["v"], t["qs"], t["ks"], **kw)
    torch.cuda.synchronize()
    _native.check_device_errors()
    return out


def check(out, t, causal, scale=None):
    """Of every value v the result takes the share p: p is rounded to bf16
    once (U16) and carries the score's float32 error in its exponent (128
    products and additions of magnitude |q||k|, then 2^-22 of the exponent's
    size for the multiplication by scale * log2 e and the exponential); the
    sums over n keys and the final division add a unit a term; the result is
    rounded once."""
    q, k, v = (t[x].double().cpu().numpy() for x in "qkv")
    qs, ks = t["qs"].cpu().numpy(), t["ks"].cpu().numpy()
    sc = 128 ** -0.5 if scale is None else scale
    ref = opacked.packed_attention(q, k, v, qs, ks, causal, scale)
    mag = opacked.packed_attention(q, k, np.abs(v), qs, ks, causal, scale)
    got = out.double().cpu().numpy()
    assert got.shape == q.shape
    for s in range(len(qs) - 1):
        qr, kr = slice(qs[s], qs[s + 1]), slice(ks[s], ks[s + 1])
        n = ks[s + 1] - ks[s]
        if not n or qs[s + 1] == qs[s]:
            assert not got[qr].any()
            continue
        big = sc * np.abs(q[qr]).sum(-1).max() * np.abs(k[kr]).max()
        top = sc * np.sqrt((q[qr] ** 2).sum(-1).max() * (k[kr] ** 2).sum(-1).max())
        share = 1.01 * U16 + 2 * (136 * U32 * big + 4 * 2.0 ** -22 * (1 + top)) + (n + 4) * U32
        tol = 1.01 * U16 * np.abs(ref[qr]) + share * mag[qr] + 1e-30
        assert (np.abs(got[qr] - ref[qr]) <= tol).all()


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 3), (2, 1), (6, 2), (10, 2), (8, 1), (7, 1),
                                            (40, 1), (64, 1), (65, 1), (128, 1)])
def test_groups(heads, kv_heads, causal):
    lengths = [1, 30, 0, 19] if heads > 16 else [1, 130, 0, 65, 128, 33]
    t = make(lengths, lengths, heads, kv_heads, seed=heads)
    check(call(t, causal=causal), t, causal)


@pytest.mark.parametrize("n", [1, 2, 16, 31, 32, 33, 127, 128, 129, 255, 256, 257, 383, 385])
@pytest.mark.parametrize("causal", [False, True])
def test_lengths(n, causal):
    t = make([n], [n], 2, 1, seed=n)
    check(call(t, causal=causal), t, causal)


@pytest.mark.parametrize("q_lengths,k_lengths", [
    ([1, 1, 1], [1, 129, 1000]),            # single new tokens over their past
    ([5, 17, 2], [5, 400, 258]),            # chunks of new tokens
    ([40, 3, 9], [10, 0, 9]),               # more queries than keys: rows that see nothing
    ([200, 64, 0, 7], [77, 512, 30, 0]),    # text lengths unrelated to the clips'
    ([300, 1], [129, 128]),
])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("heads,kv_heads", [(2, 2), (5, 1)])
def test_different_lengths(q_lengths, k_lengths, causal, heads, kv_heads):
    t = make(q_lengths, k_lengths, heads, kv_heads, seed=len(q_lengths))
    check(call(t, causal=causal), t, causal)


def reference64(t, causal):
    """The definition in float64 torch on the GPU (larger cases), and with |v|."""
    q, k, v = (t[x].double() for x in "qkv")
    group = q.shape[1] // k.shape[1]
    k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    qs, ks = t["qs"].tolist(), t["ks"].tolist()
    ref, mag = torch.zeros_like(q), torch.zeros_like(q)
    for s in range(len(qs) - 1):
        a, b = slice(qs[s], qs[s + 1]), slice(ks[s], ks[s + 1])
        n, m = a.stop - a.start, b.stop - b.start
        if not n or not m:
            continue
        w = torch.einsum("ihd,jhd->hij", q[a], k[b]) * 128 ** -0.5
        if causal:
            hidden = (torch.arange(m, device=DEV)[None]
                      > torch.arange(n, device=DEV)[:, None] + (m - n))
            w = w.masked_fill(hidden, float("-inf"))
        w = torch.softmax(w, -1).nan_to_num(0.0)
        ref[a] = torch.einsum("hij,jhd->ihd", w, v[b])
        mag[a] = torch.einsum("hij,jhd->ihd", w, v[b].abs())
    return ref, mag


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("heads,kv_heads", [(16, 16), (16, 4), (40, 8), (12, 4), (24, 3)])
def test_many_items(heads, kv_heads, causal):
    """Several items a CTA: requests of very different lengths, among them
    empty ones and ones without keys, blocks of every kind next to each other."""
    q_lengths = [700, 1, 0, 333, 1500, 64, 129, 9, 256, 40, 2, 511]
    k_lengths = [700, 1, 5, 333, 900, 2000, 129, 0, 512, 39, 300, 511]
    t = make(q_lengths, k_lengths, heads, kv_heads, seed=heads + causal)
    out = call(t, causal=causal)
    ref, mag = reference64(t, causal)
    big = 128 ** -0.5 * t["q"].double().abs().sum(-1).max() * t["k"].double().abs().max()
    top = 128 ** -0.5 * (t["q"].double().pow(2).sum(-1).max() * t["k"].double().pow(2).sum(-1).max()).sqrt()
    share = 1.01 * U16 + 2 * (136 * U32 * big + 4 * 2.0 ** -22 * (1 + top)) + 2004 * U32
    tol = 1.01 * U16 * ref.abs() + share * mag + 1e-30
    assert ((out.double() - ref).abs() <= tol).all()
    assert all(torch.equal(call(t, causal=causal), out) for _ in range(5))


def test_long_single_tokens_split():
    """Few rows over long keys: the keys are split over CTAs and joined."""
    k_lengths = [5000, 1, 2048, 0, 777]
    assert _native.load_library().bsa_packed_attention_workspace_bytes(5, sum(k_lengths), 5, 4, 1) > 0
    t = make([1] * 5, k_lengths, 4, 1, seed=3)
    want = call(t, causal=True)
    check(want, t, True)
    check(call(t), t, False)
    assert all(torch.equal(call(t, causal=True), want) for _ in range(3))
    t = make([3, 0, 9], [4100, 9, 2050], 2, 2, seed=5)
    check(call(t, causal=True), t, True)


def test_many_requests():
    for s in (31, 33, 200, 1030):
        lengths = [(5 * i) % 4 for i in range(s)]
        t = make(lengths, lengths, 2, 1, seed=s)
        check(call(t, causal=True), t, True)


@pytest.mark.parametrize("scale", [0.01, 1.0, 6.0])
def test_scales_and_extreme_scores(scale):
    """Peaked rows (scores far apart move the stabiliser) and flat ones."""
    t = make([150], [300], 2, 1, seed=7, std=3.0)
    check(call(t, scale=scale), t, False, scale)


@pytest.mark.parametrize("causal", [False, True])
def test_other_requests_values_never_leak(causal):
    lengths = [70, 130, 45]
    t = make(lengths, lengths, 4, 2, seed=9)
    clean = call(t, causal=causal)
    for name in ("q", "k", "v"):
        t[name] = t[name].clone()
        t[name][70:200] = float("nan")
        t[name][71] = float("inf")
    out = call(t, causal=causal)
    assert torch.equal(out[:70], clean[:70]) and torch.equal(out[200:], clean[200:])
    assert out[70:200].isnan().any()


@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("at", [1, 100, 127, 128, 200, 255])
def test_causal_future_never_leaks(value, at):
    """Non-finite keys and values at position ``at`` reach no earlier query,
    those in the same tile included."""
    t = make([256], [256], 2, 1, seed=11)
    clean = call(t, causal=True)
    bad = dict(t, k=t["k"].clone(), v=t["v"].clone())
    bad["v"][at] = value
    out = call(bad, causal=True)
    ref = opacked.packed_attention(*(t[x].double().cpu().numpy()[:at] for x in "qkv"),
                                   [0, at], [0, at], True)
    assert out[:at].isfinite().all()
    assert np.abs(out[:at].double().cpu().numpy() - ref).max() <= 2 * U16 * np.abs(
        clean[:at].double().cpu().numpy()).max() + 2 * U16
    assert not out[at].isfinite().all()
    bad = dict(t, k=t["k"].clone())
    bad["k"][at] = value
    out = call(bad, causal=True)
    assert torch.equal(out[:at], clean[:at])


def test_causal_future_never_leaks_single_tokens():
    """The split form: two new tokens, the second one's value not finite."""
    t = make([2], [3000], 4, 1, seed=13)
    clean = call(t, causal=True)
    t["v"][2999] = float("nan")
    out = call(t, causal=True)
    tol = 2 * U16 * clean[0].float().abs().max() + 2 * U16
    assert (out[0].float() - clean[0].float()).abs().max() <= tol and out[1].isnan().all()


def test_strided_inputs():
    """Slices of one fused projection, head-major and broadcast tensors."""
    fused = torch.randn((140, 8, 128), device=DEV).to(torch.bfloat16)
    t = dict(q=fused[:, :4], k=fused[:, 4:6], v=fused[:, 6:8], qs=starts_of([100, 40]),
             ks=starts_of([100, 40]))
    want = call(t, causal=True)
    check(want, t, True)
    head_major = {x: t[x].transpose(0, 1).contiguous().transpose(0, 1) for x in "qkv"}
    assert torch.equal(call(dict(t, **head_major), causal=True), want)
    one = dict(t, k=fused[:, 4:5].expand(-1, 2, -1), v=fused[:, 6:7].expand(-1, 2, -1))
    check(call(one, causal=True), one, True)
    shifted = torch.randn(140 * 2 * 128 + 4, device=DEV).to(torch.bfloat16)[4:].view(140, 2, 128)
    off = dict(t, k=shifted)
    check(call(off, causal=True), off, True)


def test_streams_graph_and_repeats():
    t = make([300, 77], [300, 77], 8, 2, seed=15)
    want = call(t, causal=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outs = [kernels.packed_attention(t["q"], t["k"], t["v"], t["qs"], causal=True)
                for _ in range(4)]
    side.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = kernels.packed_attention(t["q"], t["k"], t["v"], t["qs"], causal=True)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(captured, want)


def test_no_keys_and_no_queries():
    t = make([5, 3], [0, 0], 2, 1)
    assert not call(t).any()
    t = make([0, 0], [4, 0], 2, 1)
    assert call(t).shape == (0, 2, 128)


def test_bad_offsets_are_reported():
    t = make([40, 25], [40, 25], 2, 1, seed=17)
    for key, bad in [("qs", [0, 40, 64]), ("qs", [1, 40, 65]), ("qs", [0, 90, 65]), ("qs", [0, -5, 65]),
                     ("ks", [0, 90, 65]), ("ks", [-1, 40, 65]), ("ks", [0, 40, 66])]:
        with pytest.raises(RuntimeError, match="out of range"):
            call(dict(t, **{key: torch.tensor(bad, dtype=torch.int32, device=DEV)}))


def test_wide_offsets_are_reported():
    """int64 offsets that an int32 would wrap onto valid rows."""
    t = make([40, 25], [40, 25], 2, 1, seed=17)
    for key, bad in [("qs", [0, 2 ** 32 + 40, 65]), ("qs", [0, 40, 2 ** 32 + 65]), ("ks", [0, 2 ** 32 + 40, 65]),
                     ("ks", [-2 ** 32, 40, 65])]:
        with pytest.raises(RuntimeError, match="out of range"):
            call(dict(t, **{key: torch.tensor(bad, dtype=torch.int64, device=DEV)}))


def test_refusals():
    t = make([4], [4], 4, 2)
    with pytest.raises(RuntimeError, match="CUDA"):
        kernels.packed_attention(t["q"].cpu(), t["k"], t["v"], t["qs"])
    for ch, match in [(dict(q=t["q"].float()), "bf16"), (dict(v=t["v"][:3]), "equal shapes"),
                      (dict(q=t["q"][:, :3]), "do not divide"),
                      (dict(ks=starts_of([2, 2])), "equal lengths"),
                      (dict(qs=t["qs"].float()), "integers")]:
        with pytest.raises(ValueError, match=match):
            call(dict(t, **ch))
    with pytest.raises(ValueError, match="same rows"):
        kernels.packed_attention(t["q"], t["k"][:3], t["v"][:3], t["qs"])
    with pytest.raises(NotImplementedError, match="head_dim"):
        kernels.packed_attention(t["q"][..., :64], t["k"][..., :64], t["v"][..., :64], t["qs"])
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(RuntimeError, match="scale"):
            call(t, scale=scale)
    wide = make([1], [1], 258, 2)
    with pytest.raises(RuntimeError, match="128 query heads"):
        call(wide)
