"""Argument checks of the packed-request entry points, and their definitions in
``oracle/packed.py``.  No call here reaches a kernel."""

import ctypes

import numpy as np
import pytest

from dit_sparse_atten_b200 import _native
from oracle import packed as opacked

F32, BF16, F16 = 0, 1, 2
NONE, LAYER, RMS = 0, 1, 2


def _err():
    return _native.load_library().bsa_last_error().decode()


def norm(**kw):
    a = dict(x=4096, x_dtype=BF16, x_stride=64, y=1 << 20, y_dtype=BF16, y_stride=64, rows=4, width=64,
             starts=16, requests=2, gate=16, gate_stride=64, shift=16, shift_stride=64, scale=16,
             scale_stride=64, mods=F32, weight=16, bias=16, affine=BF16, post_weight=None,
             post_bias=None, post_dtype=F32, norm=LAYER, post=NONE, eps=1e-6, residual=1 << 21,
             normed=1 << 22, err=16)
    a.update(kw)
    return _native.load_library().bsa_residual_norm(*a.values(), None)


@pytest.mark.parametrize("kw,code,text", [
    (dict(x_dtype=3), -1, "element type"), (dict(mods=-1), -1, "element type"),
    (dict(y_dtype=F32), -2, "16-bit x"), (dict(rows=-1), -1, "rows"), (dict(rows=1 << 31), -1, "rows"),
    (dict(width=0), -2, "width"), (dict(width=32769), -2, "width"), (dict(norm=NONE), -1, "norm"),
    (dict(post=3), -1, "post_norm"), (dict(eps=-1.0), -1, "eps"), (dict(eps=float("nan")), -1, "eps"),
    (dict(requests=0), -1, "requests"), (dict(starts=None), -1, "1 or rows"),
    (dict(y=None), -1, "need y"), (dict(y=None, gate=None, post=RMS), -1, "need y"),
    (dict(post_weight=16), -1, "need post_norm"), (dict(x=None), -1, "null"),
    (dict(normed=None), -1, "null"), (dict(residual=None), -1, "null"), (dict(err=None), -1, "null"),
    (dict(x=4097), -1, "aligned"), (dict(weight=17), -1, "aligned"), (dict(gate=18), -1, "aligned"),
    (dict(x_stride=-64), -1, "strides"), (dict(normed=4096), -1, "overlap"),
    (dict(residual=4096 + 256), -1, "overlap"), (dict(normed=(1 << 21) + 128), -1, "overlap")])
def test_residual_norm_refuses(kw, code, text):
    assert norm(**kw) == code and text in _err()


def test_residual_norm_without_rows_is_done():
    assert norm(rows=0, x=None, normed=None) == 0 and _err() == ""


def lora(**kw):
    a = dict(y=1 << 20, y_stride=64, x=4096, x_stride=32, a=16, b=16, scales=16, starts=16, ids=16, rows=4,
             requests=2, count=1, k=32, n=64, rank=8, work=1 << 23, bytes=1 << 20, out=1 << 22,
             out_stride=64, err=16)
    a.update(kw)
    return _native.load_library().bsa_lora_add(*a.values(), None)


@pytest.mark.parametrize("kw,code,text", [
    (dict(rows=-1), -1, "rows"), (dict(count=-1), -1, "count"), (dict(rank=0), -2, "rank"),
    (dict(rank=12), -2, "rank"), (dict(rank=136), -2, "rank"), (dict(k=36), -2, "multiples of 8"),
    (dict(n=0), -2, "multiples of 8"), (dict(x_stride=24), -1, "row strides"),
    (dict(y_stride=68), -1, "row strides"), (dict(out_stride=8), -1, "row strides"),
    (dict(requests=0), -1, "requests"), (dict(x=None), -1, "null"), (dict(ids=None), -1, "null"),
    (dict(work=None), -1, "null"), (dict(a=None), -1, "null"), (dict(x=4104), -1, "aligned"),
    (dict(bytes=63), -1, "workspace"), (dict(out=4096), -1, "overlap"),
    (dict(out=(1 << 20) + 128), -1, "overlap"), (dict(out=1 << 20, out_stride=128), -1, "overlap")])
def test_lora_add_refuses(kw, code, text):
    assert lora(**kw) == code and text in _err()


def test_lora_workspace():
    lib = _native.load_library()
    assert lib.bsa_lora_add_workspace_bytes(4, 2, 32, 8) == 4 * 32 * 2
    assert lib.bsa_lora_add_workspace_bytes(1000, 2, 5120, 72) == 1000 * 96 * 2
    assert lib.bsa_lora_add_workspace_bytes(0, 2, 5120, 72) == 0
    assert lora(rows=0, x=None) == 0


def attention(**kw):
    a = dict(q=4096, q_t=256, q_h=128, k=1 << 20, k_t=128, k_h=128, v=1 << 21, v_t=128, v_h=128, qs=16,
             ks=16, q_rows=4, k_rows=4, requests=1, heads=2, kv_heads=1, head_dim=128, causal=1,
             scale=0.1, work=None, bytes=0, out=1 << 22, err=16)
    a.update(kw)
    return _native.load_library().bsa_packed_attention(*a.values(), None)


@pytest.mark.parametrize("kw,code,text", [
    (dict(head_dim=64), -2, "head_dim"), (dict(q_rows=-1), -1, "q_rows"),
    (dict(k_rows=(1 << 31) - 256), -1, "k_rows"), (dict(kv_heads=3, heads=4), -1, "divide"),
    (dict(heads=0), -1, "divide"), (dict(heads=129), -2, "128 query heads"),
    (dict(scale=0.0), -1, "scale"), (dict(scale=float("inf")), -1, "scale"),
    (dict(scale=float("nan")), -1, "scale"), (dict(requests=0), -1, "requests"), (dict(q=None), -1, "null"),
    (dict(v=None), -1, "null"), (dict(qs=None), -1, "null"), (dict(k=(1 << 20) + 8), -1, "aligned"),
    (dict(q_t=252), -1, "strides"), (dict(q_h=64), -1, "strides"), (dict(q_t=128, q_h=256), -1, "strides"),
    (dict(out=4096), -1, "overlap"), (dict(out=(1 << 21) + 256), -1, "overlap"),
    (dict(k_rows=100000, out=1 << 28), -1, "workspace")])
def test_packed_attention_refuses(kw, code, text):
    assert attention(**kw) == code and text in _err()


def test_packed_attention_workspace():
    """One part where the tiles fill the GPU; otherwise parts x rows x heads x
    (128 + 2) floats."""
    lib = _native.load_library()
    bytes_of = lib.bsa_packed_attention_workspace_bytes
    assert bytes_of(57600, 57600, 1, 40, 40) == 0 and bytes_of(0, 10, 1, 2, 1) == 0
    need = bytes_of(16, 160000, 16, 40, 8)
    assert need > 0 and need % (16 * 40 * 130 * 4) == 0
    assert bytes_of(16, 160000, 16, 40, 7) == 0
    assert attention(q_rows=0, q=None) == 0


def test_binding_refuses_to_guess():
    """Without CUDA tensors the compiled front steps aside."""
    import torch
    binding = _native.load_binding()
    t = torch.zeros((4, 64), dtype=torch.bfloat16)
    none = [None] * 8
    assert binding.residual_norm(t, *none, None, LAYER, NONE, 1e-6, -1) is None
    assert binding.residual_norm(t) is None
    assert binding.lora_add(t, t, t, t, t, t, None, None) is None
    assert binding.packed_attention(t, t, t, t, t, False, 1.0) is None
    with pytest.raises(ValueError):
        binding.set_err_word(-1, 0)


def test_definitions():
    """The oracle's own formulas on values that can be checked by hand."""
    r, h = opacked.residual_norm(np.array([[1.0, 3.0]]), np.array([[2.0, -2.0]]), row_request=[0],
                                 gate=np.array([[1.0, 0.5]]), scale=np.array([[1.0, 0.0]]),
                                 shift=np.array([[0.0, 5.0]]), eps=0.0)
    assert np.allclose(r, [[3.0, 2.0]]) and np.allclose(h, [[2.0, 4.0]])
    y = opacked.lora_add(np.zeros((3, 1)), np.ones((3, 2)), np.array([[[1.0, 2.0]]]),
                         np.array([[[10.0]]]), [0, 1, 3], [-1, 0], np.array([0.5]))
    assert np.allclose(y, [[0.0], [15.0], [15.0]])
    q = np.zeros((2, 1, 1))
    v = np.array([[[1.0]], [[3.0]], [[8.0]]])
    out = opacked.packed_attention(q, np.zeros((3, 1, 1)), v, [0, 2], [0, 3], True)
    assert np.allclose(out[:, 0, 0], [2.0, 4.0])     # the first of two queries sees two of three keys
    out = opacked.packed_attention(q, np.zeros((1, 1, 1)), v[:1], [0, 2], [0, 1], True)
    assert np.allclose(out[:, 0, 0], [0.0, 1.0])     # no key: 0


def test_wide_integers_do_not_wrap():
    """int64 offsets and ids beyond int32 stay beyond every table, at its ends."""
    import torch
    from dit_sparse_atten_b200 import kernels
    wide = torch.tensor([0, 7, 2 ** 32 + 4, 2 ** 31, -2 ** 32, -2 ** 31 - 1], dtype=torch.int64)
    want = [0, 7, 2 ** 31 - 1, 2 ** 31 - 1, -2 ** 31, -2 ** 31]
    for t in (wide, torch.stack([wide, wide], 1)[:, 1]):
        got = kernels._starts_i32(t, "row_starts", torch.device("cpu"))
        assert got.dtype == torch.int32 and got.is_contiguous() and got.tolist() == want


def test_binding_of_another_torch_is_refused(monkeypatch):
    """The compiled front goes through torch's C++ types: one that was built for
    another version is not loaded, and not taken for up to date."""
    import torch
    from dit_sparse_atten_b200.csrc import build
    assert _native.binding_torch_version() == torch.__version__
    monkeypatch.setattr(_native, "_binding", None)
    monkeypatch.setattr(torch, "__version__", "0.0.1")
    assert not build.binding_up_to_date()
    with pytest.raises(RuntimeError, match="was built for torch"):
        _native.load_binding()
