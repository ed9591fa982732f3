"""``kernels.lora_add`` on a B200 against the float64 definition (``oracle/packed.py``)."""

import numpy as np
import pytest
import torch

from dit_sparse_atten_b200 import _native, kernels
from oracle import packed as opacked

pytestmark = pytest.mark.gpu
DEV = "cuda"
U16 = 2.0 ** -8     # rounding to bf16, relative
U32 = 2.0 ** -24


def make(lengths, k, n, rank, count, ids, seed=0, scales=True):
    g = torch.Generator().manual_seed(seed)

    def rnd(*shape, std=1.0):
        return (torch.randn(shape, generator=g) * std).to(torch.bfloat16).to(DEV)
    rows = sum(lengths)
    return dict(y=rnd(rows, n), x=rnd(rows, k), a=rnd(count, rank, k, std=k ** -0.5),
                b=rnd(count, n, rank, std=0.5 * rank ** -0.5),
                scales=(torch.rand(count, generator=g) + 0.5).to(DEV) if scales else None,
                starts=torch.tensor(np.cumsum([0] + list(lengths)), dtype=torch.int32, device=DEV),
                ids=torch.tensor(ids, dtype=torch.int32, device=DEV))


def call(t, **kw):
    out = kernels.lora_add(t["y"], t["x"], t["a"], t["b"], row_starts=t["starts"],
                           adapters=t["ids"], scales=t["scales"], **kw)
    torch.cuda.synchronize()
    _native.check_device_errors()
    return out


def check(out, t, y=None):
    """The scaled x A^T is rounded to bf16 once (U16 of each of its entries),
    the result once (U16 of it); the float32 sums add at most one unit of
    their magnitudes for each of their K, then R + 1, terms."""
    f = {k: (None if v is None else v.double().cpu().numpy()) for k, v in t.items()}
    starts, ids = t["starts"].cpu().numpy(), t["ids"].cpu().numpy()
    ref = opacked.lora_add(f["y"] if y is None else y, f["x"], f["a"], f["b"], starts, ids, f["scales"])
    tol = 1.01 * U16 * np.abs(ref) + 1e-30
    k, r = f["x"].shape[1], f["a"].shape[1]
    for s, i in enumerate(ids):
        if i < 0:
            continue
        rows = slice(starts[s], starts[s + 1])
        sc = 1.0 if f["scales"] is None else f["scales"][i]
        u = sc * np.abs(f["x"][rows] @ f["a"][i].T)
        big = sc * np.abs(f["x"][rows]) @ np.abs(f["a"][i]).T
        tol[rows] += (1.01 * U16 * u + (k + 8) * U32 * big) @ np.abs(f["b"][i]).T
        tol[rows] += (r + 2) * U32 * (u @ np.abs(f["b"][i]).T + np.abs(f["y"][rows]))
    assert (np.abs(out.double().cpu().numpy() - ref) <= tol).all()


@pytest.mark.parametrize("rank", [8, 16, 24, 32, 40, 64, 72, 104, 128])
@pytest.mark.parametrize("lengths", [[1], [7, 0, 1, 9], [300, 129, 1, 64]])
def test_ranks(rank, lengths):
    t = make(lengths, 520, 264, rank, 3, [(2 * i) % 3 for i in range(len(lengths))], seed=rank)
    check(call(t), t)


@pytest.mark.parametrize("k,n", [(8, 8), (16, 1000), (40, 24), (4096, 64), (64, 4104), (5120, 256),
                                 (1032, 2056)])
def test_sizes(k, n):
    t = make([5, 130, 1, 0, 257], k, n, 16, 2, [1, 0, -1, 1, 1], seed=k + n)
    check(call(t), t)


@pytest.mark.parametrize("rank", [16, 64, 72, 128])
def test_many_tiles(rank):
    """Several tiles a CTA, requests with and without adapters between them,
    whole and partial row tiles, a last column tile of 8 columns."""
    t = make([700, 0, 128, 1, 515, 256, 40, 384], 192, 2056, rank, 3, [0, 1, 2, -1, 1, -1, 0, 2],
             seed=rank)
    want = call(t)
    check(want, t)
    y = t["y"].clone()
    assert torch.equal(call(dict(t, y=y), out=y), want)
    assert all(torch.equal(call(t), want) for _ in range(5))


def test_single_rows_and_many_requests():
    for s in (1, 31, 33, 200, 1030):
        t = make([1] * s, 256, 320, 16, 5, [(3 * i) % 6 - 1 for i in range(s)], seed=s)
        check(call(t), t)


def test_no_adapter_rows_pass_through():
    t = make([3, 200, 4], 128, 512, 32, 1, [-1, -1, -1], seed=4)
    assert torch.equal(call(t), t["y"])
    t = make([3, 200, 4], 128, 512, 32, 1, [-1, 0, -1], seed=4, scales=False)
    out = call(t)
    check(out, t)
    assert torch.equal(out[:3], t["y"][:3]) and torch.equal(out[203:], t["y"][203:])


def test_in_place_and_out():
    t = make([70, 3], 256, 520, 24, 2, [1, 0], seed=6)
    want = call(t)
    y = t["y"].clone()
    got = kernels.lora_add(y, t["x"], t["a"], t["b"], row_starts=t["starts"], adapters=t["ids"],
                           scales=t["scales"], out=y)
    assert got is y and torch.equal(y, want)
    wide = torch.zeros((73, 1040), dtype=torch.bfloat16, device=DEV)
    call(t, out=wide[:, 520:])
    assert torch.equal(wide[:, 520:], want) and not wide[:, :520].any()
    got = kernels.lora_add(t["y"][None], t["x"][None], t["a"], t["b"], row_starts=t["starts"],
                           adapters=t["ids"].long(), scales=t["scales"].double())
    assert got.shape == (1, 73, 520) and torch.equal(got[0], want)


def test_strided_inputs():
    t = make([33, 90], 3 * 256, 2 * 264, 16, 2, [1, 0], seed=8)
    t = dict(t, x=t["x"][:, 256:512], y=t["y"][:, 264:], a=t["a"][:, :, :256], b=t["b"][:, 264:])
    check(call(t), t)
    # columns that start off the 16-byte grid
    flat = torch.randn(123, 3 * 256 + 8, device=DEV).to(torch.bfloat16)
    t = dict(t, x=flat[:, 3:259])
    check(call(t), t)


@pytest.mark.parametrize("rows", [1, 2, 40])
def test_slices_of_odd_widths(rows):
    """Rows, and a single row, cut out of wider tensors of odd widths."""
    t = make([rows], 256, 264, 16, 1, [0], seed=20)
    want = call(t)
    wide = {k: torch.zeros((rows, t[k].shape[1] + 11), dtype=torch.bfloat16, device=DEV) for k in "xy"}
    for shift in (0, 3, 8):
        views = {k: wide[k][:, shift:shift + t[k].shape[1]] for k in "xy"}
        for k in "xy":
            views[k].copy_(t[k])
        assert torch.equal(call(dict(t, **views)), want)
        if rows == 1 and shift != 3:
            into = torch.zeros((1, 275), dtype=torch.bfloat16, device=DEV)[:, shift:shift + 264]
            assert torch.equal(call(dict(t, **views), out=into), want) and torch.equal(into, want)
            assert torch.equal(call(dict(t, **views), out=views["y"]), want)
            assert torch.equal(views["y"], want)


def test_factors_off_the_16_byte_grid():
    t = make([33, 90], 256, 264, 16, 2, [1, 0], seed=21)
    want = call(t)

    def shifted(f):
        return torch.cat([f.new_zeros(3), f.flatten()])[3:].view(f.shape)
    for keys in ("a", "b", "ab"):
        assert torch.equal(call(dict(t, **{k: shifted(t[k]) for k in keys})), want)


def test_poison_stays_in_its_request():
    t = make([40, 25, 3], 320, 264, 32, 2, [0, 1, 0], seed=10)
    clean = call(t)
    t["x"][40:65] = float("nan")
    t["a"][1] = float("inf")
    out = call(t)
    assert torch.equal(out[:40], clean[:40]) and torch.equal(out[65:], clean[65:])
    assert out[40:65].isnan().all()


@pytest.mark.parametrize("rank", [8, 24, 40, 72])
@pytest.mark.parametrize("lengths", [[3, 2, 1], [40, 25, 130]])
@pytest.mark.parametrize("where", ["x", "scales"])
def test_infinities_keep_their_sign_at_padded_ranks(rank, lengths, where):
    """Positive factors and an infinity in x, or as a scale: every result of
    those rows is +inf, also where the kernels pad the rank."""
    t = make(lengths, 72, 136, rank, 2, [0, 1, -1], seed=rank)
    t["x"], t["a"], t["b"] = t["x"].abs() + 0.1, t["a"].abs() + 0.01, t["b"].abs() + 0.01
    clean = call(t)
    if where == "x":
        t["x"][0, 5] = float("inf")
        bad = slice(0, 1)
    else:
        t["scales"][1] = float("inf")
        bad = slice(lengths[0], lengths[0] + lengths[1])
    out = call(t)
    assert torch.isposinf(out[bad]).all()
    keep = torch.ones(sum(lengths), dtype=torch.bool)
    keep[bad] = False
    assert torch.equal(out[keep], clean[keep])


def test_runs_are_identical_and_streams_agree():
    t = make([513, 100, 1], 1024, 768, 64, 3, [2, 0, 1], seed=12)
    want = call(t)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outs = [kernels.lora_add(t["y"], t["x"], t["a"], t["b"], row_starts=t["starts"],
                                 adapters=t["ids"], scales=t["scales"]) for _ in range(3)]
    side.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = kernels.lora_add(t["y"], t["x"], t["a"], t["b"], row_starts=t["starts"],
                                    adapters=t["ids"], scales=t["scales"])
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(captured, want)


def test_bad_offsets_and_ids_are_reported():
    t = make([40, 25], 64, 64, 8, 2, [0, 1], seed=14)
    for key, bad in [("starts", [0, 40, 64]), ("starts", [1, 40, 65]), ("starts", [0, 90, 65]),
                     ("starts", [0, -5, 65]), ("ids", [0, 2]), ("ids", [-2, 1])]:
        b = dict(t, **{key: torch.tensor(bad, dtype=torch.int32, device=DEV)})
        with pytest.raises(RuntimeError, match="out of range"):
            call(b)


def test_wide_ids_and_offsets_are_reported():
    """int64 values that an int32 would wrap onto a valid adapter or row."""
    t = make([40, 25], 64, 64, 8, 2, [0, 1], seed=14)
    for key, bad in [("ids", [2 ** 32, 1]), ("ids", [0, -2 ** 32 + 1]), ("starts", [0, 2 ** 32 + 40, 65]),
                     ("starts", [0, 40, 2 ** 32 + 65]), ("starts", [-2 ** 32, 40, 65])]:
        b = dict(t, **{key: torch.tensor(bad, dtype=torch.int64, device=DEV)})
        with pytest.raises(RuntimeError, match="out of range"):
            call(b)


def test_empty():
    t = make([0, 0], 64, 64, 8, 2, [0, 1])
    assert call(t).shape == (0, 64)


def test_refusals():
    t = make([4], 64, 64, 8, 1, [0])
    kw = dict(row_starts=t["starts"], adapters=t["ids"])
    with pytest.raises(RuntimeError, match="CUDA"):
        kernels.lora_add(t["y"].cpu(), t["x"], t["a"], t["b"], **kw)
    for args, match in [
            ((t["y"].float(), t["x"], t["a"], t["b"]), "bf16"),
            ((t["y"][:3], t["x"], t["a"], t["b"]), "same rows"),
            ((t["y"], t["x"], t["a"][:, :, :32], t["b"]), "lora_a must be"),
            ((t["y"], t["x"], t["a"], t["b"][:, :32]), "lora_b must be")]:
        with pytest.raises(ValueError, match=match):
            kernels.lora_add(*args, **kw)
    base = (t["y"], t["x"], t["a"], t["b"])
    with pytest.raises(ValueError, match="adapters must be"):
        kernels.lora_add(*base, row_starts=t["starts"], adapters=t["ids"].repeat(2))
    with pytest.raises(ValueError, match="scales must be"):
        kernels.lora_add(*base, **kw, scales=torch.ones(2, device=DEV))
    with pytest.raises(ValueError, match="out must have"):
        kernels.lora_add(*base, **kw, out=t["y"][:2])
    with pytest.raises(RuntimeError, match="overlap"):
        both = torch.zeros((4, 128), dtype=torch.bfloat16, device=DEV)
        kernels.lora_add(both[:, :64], t["x"], t["a"], t["b"], **kw, out=both[:, 8:72])
    for k, n, r in [(60, 64, 8), (64, 60, 8), (64, 64, 12), (64, 64, 136)]:
        b = make([4], k, n, r, 1, [0])
        with pytest.raises((RuntimeError, ValueError), match="multiple"):
            call(b)
