"""A routed backend under ``packed_model.PackedWanTransformer``: each request's
self-attention goes through ``FlexReuseBackend``, which keeps its routes by
branch (here: one for each request)."""

import math

import pytest
import torch

from dit_sparse_atten_b200 import _native, packed_model, wan_model
from dit_sparse_atten_b200.context import reset_runtime_state, set_routing_context
from dit_sparse_atten_b200.flex import FlexReuseBackend, FlexReuseConfig

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
CFG = wan_model.WanConfig(dim=256, ffn=512, heads=2, layers=2, in_channels=4, out_channels=4,
                          text_dim=64, text_tokens=16, freq_dim=32)
GRIDS, TEXT, STEPS = [(2, 16, 32), (4, 16, 16), (2, 16, 32)], [16, 3, 77], 3


def generate(backend):
    weights = wan_model.WanWeights(CFG, DEV, seed=4)
    model = packed_model.PackedWanTransformer(weights, GRIDS, TEXT)
    g = torch.Generator(device=DEV)
    g.manual_seed(6)
    x = torch.randn((sum(math.prod(grid) for grid in GRIDS), 16), generator=g, device=DEV)
    ctx = model.context(torch.randn((sum(TEXT), CFG.text_dim), generator=g, device=DEV).to(torch.bfloat16))
    reset_runtime_state()
    sigmas = wan_model.flow_sigmas(STEPS)
    for step in range(STEPS):
        def attention(request, layer, q, k, v):
            set_routing_context(attention_id=layer, step=step, branch=request, grid=GRIDS[request])
            return backend(q, k, v)
        noise = model.forward(x, [sigmas[step] * 1000.0] * len(GRIDS), ctx, backend and attention)
        x = x + (sigmas[step + 1] - sigmas[step]) * noise.float()
    torch.cuda.synchronize()
    _native.check_device_errors()
    return x


def backend(**kw):
    return FlexReuseBackend(FlexReuseConfig(bootstrap_mode="sampled", route_samples=16, sampled_update_interval=2,
                                            prefetch_sampled_update=False, spatial_reorder=True,
                                            total_steps=STEPS, **kw))


def test_full_routes_match_the_packed_attention():
    """Routes that keep every block are full attention: the packed kernel's, up
    to the bf16 roundings of three steps (the bound of test_gpu_wan_model.py)."""
    routed = backend(keep=1.0, mass_target=1.0)
    sparse, dense = generate(routed), generate(None)
    requests = len(GRIDS)
    assert routed.phase_counts["sparse_reuse"] == requests * 2            # layer 1, steps 1 and 2
    assert routed.phase_counts["first_layer_dense"] == requests * STEPS
    err = (sparse - dense).abs()
    assert err.max() <= 0.05 * dense.abs().max() and err.mean() <= 0.02 * dense.abs().mean()


def test_each_request_keeps_its_own_routes():
    routed = backend(keep=0.625, mass_target=0.95, dense_route_threshold=0.58)
    assert generate(routed).isfinite().all()
    counts, requests = routed.phase_counts, len(GRIDS)
    assert counts["sampled_bootstrap"] == requests
    assert counts["sparse_reuse"] + counts["dense_dispatch"] == requests * 2
    assert routed.profile_summary()["released_routes"] == requests
