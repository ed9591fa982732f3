"""``kernels.residual_norm`` on a B200 against the float64 definition
(``oracle/packed.py``)."""

import numpy as np
import pytest
import torch

from dit_sparse_atten_b200 import _native, kernels
from oracle import packed as opacked

pytestmark = pytest.mark.gpu
DEV = "cuda"
U32 = 2.0 ** -24
# half a unit in the last place of a value in [1, 2): 8, 11 and 24 significant bits
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: U32}
# smallest normal: below it a 16-bit result keeps fewer bits
TINY = {torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -14, torch.float32: 2.0 ** -126}


def f64(t):
    return None if t is None else t.double().cpu().numpy()


def make(lengths, width, *, dtype=torch.bfloat16, ydtype=None, seed=0, mean=0.0, requests=None):
    g = torch.Generator().manual_seed(seed)
    rows, s = sum(lengths), len(lengths) if requests is None else requests

    def n(*shape, std=1.0, add=0.0, dt=torch.float32):
        return (torch.randn(shape, generator=g) * std + add).to(dt).to(DEV)
    return dict(x=n(rows, width, add=mean, dt=dtype),
                y=n(rows, width, std=0.7, dt=ydtype or dtype),
                gate=n(s, width, std=0.3), shift=n(s, width, std=0.3), scale=n(s, width, std=0.3),
                weight=n(width, std=0.1, add=1.0, dt=torch.bfloat16),
                bias=n(width, std=0.1, dt=torch.bfloat16),
                post_weight=n(width, std=0.1, add=1.0), post_bias=n(width, std=0.1),
                starts=torch.tensor(np.cumsum([0] + list(lengths)), dtype=torch.int32, device=DEV))


def check(got, t, keys, *, norm="layer", post_norm=None, eps=1e-6, row_request=None):
    """The kernel rounds once to the output type; before that every float32
    operation adds at most one unit of its operands' size.  A row's sum of C
    values by 8-value chains, a warp tree and a block loop has at most 8 * 4 +
    5 + 32 additions on any path, so its relative error is below 70 units of
    the sum of magnitudes; the mean enters h scaled by 1/std, the variance as
    half its relative error.  `size` bounds the magnitudes that h is made of."""
    rows = t["x"].shape[0]
    if row_request is None:
        starts = t["starts"].cpu().numpy()
        row_request = np.searchsorted(starts[1:], np.arange(rows), side="right")
    par = {k: f64(t[k]) for k in keys if k not in ("x", "y")}
    y = f64(t["y"]) if "y" in keys else None
    r, h = opacked.residual_norm(f64(t["x"]), y, row_request=row_request, norm=norm,
                                 post_norm=post_norm, eps=eps, **par)
    _native.check_device_errors()
    got_r, got_h = f64(got.residual), f64(got.normed)
    gain = 1.0 + (np.abs(par["gate"]).max() if "gate" in par else 1.0)
    post = 1.0
    if post_norm is not None:
        post = 80 * (1.0 + np.abs(opacked.standardise(y, post_norm, eps)).max())
    size_r = np.abs(r).max(-1, keepdims=True) + np.abs(f64(t["x"])).max(-1, keepdims=True)
    tol_r = 80 * U32 * size_r + gain * post * 4 * U32
    rt = t["x"].dtype
    if y is not None:
        assert (np.abs(got_r - r) <= 1.01 * UNIT[rt] * np.abs(r) + tol_r + TINY[rt] * UNIT[rt]).all()
    std = np.sqrt((r * r).mean(-1, keepdims=True) - (r.mean(-1, keepdims=True) ** 2 if norm == "layer" else 0)
                  + eps)
    amp = (np.abs(par["weight"]).max() if "weight" in par else 1.0)
    amp *= 1.0 + (np.abs(par["scale"]).max() if "scale" in par else 0.0)
    add = sum(np.abs(par[k]).max() for k in ("bias", "shift") if k in par)
    tol_h = 4 * (tol_r / std) * amp + 80 * U32 * (np.abs(h).max(-1, keepdims=True) + add * amp)
    ht = got.normed.dtype
    assert (np.abs(got_h - h) <= 1.01 * UNIT[ht] * np.abs(h) + tol_h + TINY[ht] * UNIT[ht]).all()


ALL = ("y", "gate", "shift", "scale")
AFFINE = ALL + ("weight", "bias")


def call(t, keys, **kw):
    kw.setdefault("row_starts", t["starts"])
    got = kernels.residual_norm(t["x"], t["y"] if "y" in keys else None,
                                **{k: t[k] for k in keys if k not in ("x", "y")}, **kw)
    torch.cuda.synchronize()
    return got


@pytest.mark.parametrize("width", [1, 2, 7, 8, 33, 256, 1000, 1536, 5120, 5128, 8191, 16392, 32768])
@pytest.mark.parametrize("norm", ["layer", "rms"])
def test_widths(width, norm):
    t = make([3, 0, 1, 4], width, seed=width)
    check(call(t, AFFINE, norm=norm), t, AFFINE, norm=norm)


@pytest.mark.parametrize("dtype,ydtype", [
    (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16),
    (torch.float32, torch.bfloat16), (torch.float32, torch.float16), (torch.float32, torch.float32)])
@pytest.mark.parametrize("width", [640, 1003])
def test_types(dtype, ydtype, width):
    t = make([5, 2], width, dtype=dtype, ydtype=ydtype, seed=3)
    got = call(t, AFFINE)
    assert got.residual.dtype == dtype and got.normed.dtype == ydtype
    check(got, t, AFFINE)


@pytest.mark.parametrize("keys", [(), ("y",), ("y", "gate"), ("shift", "scale"), ("weight",),
                                  ("y", "scale"), ("y", "shift", "bias")])
def test_parts_left_out(keys):
    t = make([4, 3], 512, seed=5)
    got = call(t, keys)
    check(got, t, keys)
    if "y" not in keys:
        assert got.residual is t["x"]


@pytest.mark.parametrize("post", ["layer", "rms"])
@pytest.mark.parametrize("width", [96, 5120, 12000])
def test_post_norm(post, width):
    t = make([2, 1, 6], width, seed=7)
    keys = AFFINE + ("post_weight", "post_bias")
    check(call(t, keys, norm="rms", post_norm=post), t, keys, norm="rms", post_norm=post)


@pytest.mark.parametrize("width", [8, 40, 256, 264, 512, 520, 1536, 2560, 5120, 5128, 8192, 10240])
@pytest.mark.parametrize("dtype,ydtype,norm,post", [
    (torch.bfloat16, torch.bfloat16, "layer", None), (torch.float16, torch.float16, "rms", "layer"),
    (torch.float32, torch.bfloat16, "rms", None), (torch.float32, torch.float32, "layer", "rms")])
def test_many_rows(width, dtype, ydtype, norm, post):
    """Enough rows for the resident blocks: several a block, requests that
    begin and end between a block's rows, some of a single row."""
    t = make([300, 0, 1, 2, 700, 149, 1], width, dtype=dtype, ydtype=ydtype, seed=width)
    keys = AFFINE + (("post_weight",) if post else ())
    check(call(t, keys, norm=norm, post_norm=post), t, keys, norm=norm, post_norm=post)
    if width == 520:
        for keys in ((), ("y",), ("shift", "scale"), ("y", "gate", "weight")):
            check(call(t, keys, norm=norm), t, keys, norm=norm)
        keys = AFFINE + ("post_weight", "post_bias")
        check(call(t, keys, norm=norm, post_norm="rms"), t, keys, norm=norm, post_norm="rms")
        rows = t["x"].shape[0]
        t = make([rows], width, dtype=dtype, ydtype=ydtype, seed=1, requests=rows)
        check(call(t, ALL, row_starts=None), t, ALL, row_request=np.arange(rows))
        bad = dict(t, starts=torch.tensor([0, 600, 900], dtype=torch.int32, device=DEV),
                   **{k: t[k][:2] for k in ("gate", "shift", "scale")})
        call(bad, ALL)
        with pytest.raises(RuntimeError, match="out of range"):
            _native.check_device_errors()


def test_many_requests_and_per_row_modulation():
    for s in (1, 2, 31, 32, 33, 64, 65, 200, 1024, 1025, 1500):
        lengths = [(i * 7) % 3 for i in range(s)]
        lengths[-1] += 1
        t = make(lengths, 64, seed=s)
        check(call(t, ALL), t, ALL)
    rows = 77
    t = make([rows], 64, seed=1, requests=rows)
    check(call(t, ALL, row_starts=None), t, ALL, row_request=np.arange(rows))
    t = make([rows], 64, seed=1, requests=1)
    check(call(t, ALL, row_starts=None), t, ALL, row_request=np.zeros(rows, int))


def test_large_mean_keeps_the_variance():
    t = make([16], 5120, dtype=torch.float32, ydtype=torch.float32, mean=1000.0, seed=9)
    check(call(t, AFFINE), t, AFFINE)


def test_constant_rows_and_poisoned_neighbours():
    t = make([3, 2], 320, seed=11)
    t["x"][0] = 2.0
    t["x"][1] = float("nan")
    t["x"][2, 5] = float("inf")
    got = call(t, ("shift", "scale"))
    h = got.normed.float()
    assert h[1].isnan().all() and not h[0].isnan().any() and not h[3:].isnan().any()
    assert torch.equal(h[0], t["shift"][0].to(torch.bfloat16).float())   # zero variance: h = 0


def test_strided_rows_and_modulation_views():
    base = make([6, 5], 3 * 256, seed=13)
    table = torch.randn((2, 6, 256), device=DEV)
    t = dict(base, x=base["x"][:, 256:512], y=base["y"][:, 1:257], gate=table[:, 2],
             shift=table[:, 0], scale=table[:, 1])
    assert not t["x"].is_contiguous()
    check(call(t, ALL), t, ALL)
    # three-dimensional rows and 16-byte alignment lost
    flat = torch.randn(2 * 3 * 64 + 1, device=DEV).to(torch.bfloat16)[1:].view(2, 3, 64)
    got = kernels.residual_norm(flat, flat.flip(0).contiguous())
    assert got.normed.shape == (2, 3, 64) and got.residual.shape == (2, 3, 64)
    d = flat.float() + flat.flip(0).float()
    ref = torch.nn.functional.layer_norm(d, (64,), eps=1e-6)
    assert (got.normed.float() - ref).abs().max() <= 2.0 ** -8 * ref.abs().max() + 1e-5


def test_another_stream_and_graph():
    t = make([40, 24], 1536, seed=17)
    want = call(t, AFFINE)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = kernels.residual_norm(t["x"], t["y"], row_starts=t["starts"],
                                    **{k: t[k] for k in AFFINE if k != "y"})
    side.synchronize()
    assert torch.equal(got.normed, want.normed) and torch.equal(got.residual, want.residual)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = kernels.residual_norm(t["x"], t["y"], row_starts=t["starts"],
                                         **{k: t[k] for k in AFFINE if k != "y"})
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(captured.normed, want.normed)


def test_empty_and_uncovered_rows():
    t = make([0, 0], 64)
    got = call(t, ALL)
    assert got.normed.shape == (0, 64)
    t = make([4, 4], 64, seed=19)
    for bad in ([0, 4, 7], [1, 4, 8], [0, 9, 7]):
        call(dict(t, starts=torch.tensor(bad, dtype=torch.int32, device=DEV)), ALL)
        with pytest.raises(RuntimeError, match="out of range"):
            _native.check_device_errors()


def test_refusals():
    t = make([4], 64)
    x, y = t["x"], t["y"]
    with pytest.raises(RuntimeError, match="CUDA"):
        kernels.residual_norm(x.cpu())
    for kw, match in [
            (dict(y=y[:3]), "equal shapes"), (dict(y=y.float()), "type"),
            (dict(gate=t["gate"]), "need y"), (dict(post_norm="rms"), "need y"),
            (dict(norm="group"), "norm must be"), (dict(norm=None), "norm must be"),
            (dict(y=y, post_weight=t["post_weight"]), "need post_norm"),
            (dict(shift=t["shift"][:, :32]), "requests, C"), (dict(shift=t["shift"][0, :1]), "requests, C"),
            (dict(shift=t["shift"], scale=t["scale"].half()), "share one type"),
            (dict(weight=t["weight"][:8]), "must be \\[C\\]"),
            (dict(shift=t["shift"].repeat(3, 1)), "number of rows"),
            (dict(row_starts=t["starts"].float()), "integers"),
            (dict(normed_dtype=torch.float32), "type"), (dict(normed_dtype=torch.int8), "normed_dtype")]:
        with pytest.raises(ValueError, match=match):
            kernels.residual_norm(x, **kw)
    with pytest.raises(ValueError, match="bf16, fp16 or float32"):
        kernels.residual_norm(x.int())
    with pytest.raises(RuntimeError, match="width"):
        kernels.residual_norm(torch.zeros((1, 32769), device=DEV))
