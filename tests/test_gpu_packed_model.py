"""Several requests through ``packed_model.PackedWanTransformer`` against each
one alone through ``wan_model.WanTransformer`` with its adapter merged into the
weights."""

import math

import pytest
import torch

from dit_sparse_atten_b200 import _native, packed_model, wan_model
from test_wan_model import sdpa, torch_prologue

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
CFG = wan_model.WanConfig(dim=256, ffn=512, heads=2, layers=2, in_channels=4, out_channels=4,
                          text_dim=64, text_tokens=16, freq_dim=32)
GRIDS = [(2, 8, 16), (1, 5, 7), (3, 8, 8), (1, 1, 1)]
TEXT = [16, 3, 77, 129]
TIMES = [900.0, 37.5, 500.0, 1000.0]
IDS = [1, -1, 0, 1]
FEATURES = {"q": (256, 256), "k": (256, 256), "v": (256, 256), "o": (256, 256), "q2": (256, 256),
            "o2": (256, 256), "ffn1": (256, 512), "ffn2": (512, 256)}


def make_adapters(rank=16, count=2):
    g = torch.Generator(device=DEV)
    g.manual_seed(8)

    def factors(fan_in, fan_out):
        a = torch.randn((count, rank, fan_in), generator=g, device=DEV) / math.sqrt(fan_in)
        b = torch.randn((count, fan_out, rank), generator=g, device=DEV) / math.sqrt(rank) * 0.3
        return a.to(torch.bfloat16), b.to(torch.bfloat16)
    blocks = [{name: factors(*f) for name, f in FEATURES.items()} for _ in range(CFG.layers)]
    return packed_model.LoraAdapters(blocks, torch.tensor([0.5, 1.25], device=DEV),
                                     factors(256, 6 * 256))


def merged(weights, adapters, i, dtype):
    """A copy of ``weights`` in ``dtype`` with adapter ``i`` added in float32."""
    def copy(v):
        return tuple(t.to(dtype) for t in v) if isinstance(v, tuple) else v.to(dtype)

    def add(wb, factors):
        a, b = (f[i].float() for f in factors)
        return ((wb[0].float() + float(adapters.scales[i]) * b @ a).to(dtype), wb[1].to(dtype))
    out = object.__new__(wan_model.WanWeights)
    out.cfg = weights.cfg
    for name in ("patch", "time_1", "time_2", "time_proj", "text_1", "text_2", "proj_out"):
        setattr(out, name, copy(getattr(weights, name)))
    out.out_table = weights.out_table
    out.blocks = []
    for blk, factors in zip(weights.blocks, adapters.blocks):
        new = {k: (v if k == "table" else copy(v)) for k, v in blk.items()}
        if i >= 0:
            for name, f in factors.items():
                new[name] = add(blk[name], f)
        out.blocks.append(new)
    if i >= 0:
        out.time_proj = add(weights.time_proj, adapters.time_proj)
    return out


def alone(weights, adapters, patches, texts, dtype, prologue):
    outs = []
    for s, grid in enumerate(GRIDS):
        w = merged(weights, adapters, IDS[s], dtype)
        model = wan_model.WanTransformer(w, grid, wan_model.SequenceShard(), prologue)
        ctx = model.context(texts[s].to(dtype)[None])
        outs.append(model.forward(patches[s], TIMES[s], ctx, sdpa, 0, 0))
    return torch.cat(outs)


def build():
    weights = wan_model.WanWeights(CFG, DEV, seed=4)
    g = torch.Generator(device=DEV)
    g.manual_seed(5)
    patches = [torch.randn((math.prod(grid), 16), generator=g, device=DEV) for grid in GRIDS]
    texts = [torch.randn((n, CFG.text_dim), generator=g, device=DEV).to(torch.bfloat16) for n in TEXT]
    return weights, make_adapters(), patches, texts


def test_requests_together_match_each_alone():
    """Both run in bf16 with different roundings; the packed path may be no
    further from the float32 result than twice the path of one request."""
    weights, adapters, patches, texts = build()
    model = packed_model.PackedWanTransformer(weights, GRIDS, TEXT, adapters, IDS)
    out = model.forward(torch.cat(patches), TIMES, model.context(torch.cat(texts)))
    torch.cuda.synchronize()
    _native.check_device_errors()
    exact = alone(weights, adapters, patches, texts, torch.float32, torch_prologue(CFG.heads, CFG.eps))
    one = alone(weights, adapters, patches, texts, torch.bfloat16,
                wan_model.fused_prologue(CFG.heads, CFG.eps))
    begin = 0
    for grid in GRIDS:
        rows = slice(begin, begin + math.prod(grid))
        begin = rows.stop
        err = (out[rows].float() - exact[rows]).norm()
        ref = (one[rows].float() - exact[rows]).norm()
        assert err <= 2 * ref, (grid, float(err), float(ref), float(exact[rows].norm()))


def test_requests_do_not_see_each_other():
    weights, adapters, patches, texts = build()
    model = packed_model.PackedWanTransformer(weights, GRIDS, TEXT, adapters, IDS)
    want = model.forward(torch.cat(patches), TIMES, model.context(torch.cat(texts)))
    patches[1] = torch.full_like(patches[1], float("nan"))
    texts[1] = torch.full_like(texts[1], float("inf"))
    got = model.forward(torch.cat(patches), TIMES, model.context(torch.cat(texts)))
    a, b = 256, 256 + 35
    assert torch.equal(got[:a], want[:a]) and torch.equal(got[b:], want[b:])


def test_custom_self_attention_and_no_adapters():
    weights, _, patches, texts = build()
    model = packed_model.PackedWanTransformer(weights, GRIDS, TEXT)
    ctx = model.context(torch.cat(texts))
    seen = []

    def attention(request, layer, q, k, v):
        seen.append((request, layer, q.shape[1]))
        return sdpa(q, k, v)
    got = model.forward(torch.cat(patches), TIMES, ctx, attention)
    want = model.forward(torch.cat(patches), TIMES, ctx)
    assert seen == [(r, layer, math.prod(g)) for layer in range(2) for r, g in enumerate(GRIDS)]
    # two bf16 attentions of the same rows: their roundings apart
    assert (got.float() - want.float()).norm() <= 0.02 * want.float().norm()


def test_refusals():
    weights, adapters, _, _ = build()
    with pytest.raises(ValueError, match="text length"):
        packed_model.PackedWanTransformer(weights, GRIDS, TEXT[:2])
    with pytest.raises(ValueError, match="adapter id"):
        packed_model.PackedWanTransformer(weights, GRIDS, TEXT, adapters, IDS[:2])
    with pytest.raises(ValueError, match="number of blocks"):
        packed_model.PackedWanTransformer(
            weights, GRIDS, TEXT, packed_model.LoraAdapters([{}], adapters.scales), IDS)
    with pytest.raises(ValueError, match="unknown projections"):
        packed_model.LoraAdapters([{"gate": ()}], adapters.scales)
    model = packed_model.PackedWanTransformer(weights, GRIDS, TEXT)
    with pytest.raises(ValueError, match="one timestep"):
        model.forward(torch.zeros((1, 16), device=DEV), [1.0], None)
