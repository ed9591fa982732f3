"""Argument checks of ``packed_model.PackedWanTransformer``; nothing here reaches a kernel."""

import pytest
import torch

from dit_sparse_atten_b200 import packed_model, wan_model

CFG = wan_model.WanConfig(dim=256, ffn=64, heads=2, layers=1, in_channels=4, out_channels=4,
                          text_dim=16, text_tokens=4, freq_dim=32)
GRIDS, TEXT = [(1, 2, 3), (2, 2, 2)], [5, 0]


@pytest.fixture(scope="module")
def weights():
    return wan_model.WanWeights(CFG, torch.device("cpu"), seed=1)


def adapters(count):
    return packed_model.LoraAdapters([{}], torch.ones(count))


def test_rows_must_be_those_of_the_requests(weights):
    """Rows that the requests do not cover would come back as whatever the memory held."""
    model = packed_model.PackedWanTransformer(weights, GRIDS, TEXT)
    patches, ctx = torch.zeros((14, 16)), torch.zeros((5, 256), dtype=torch.bfloat16)
    for bad in (torch.zeros((13, 16)), torch.zeros((15, 16)), torch.zeros((14, 12)), patches[None]):
        with pytest.raises(ValueError, match="patches must be"):
            model.forward(bad, [1.0, 2.0], ctx)
    for bad in (ctx[:4], ctx.repeat(2, 1), ctx[:, :128], ctx[None]):
        with pytest.raises(ValueError, match="ctx must be"):
            model.forward(patches, [1.0, 2.0], bad)


@pytest.mark.parametrize("ids", [[0, 2], [-2, 0], [1, 7]])
def test_adapter_ids_must_exist(weights, ids):
    with pytest.raises(ValueError, match="adapter ids must be in"):
        packed_model.PackedWanTransformer(weights, GRIDS, TEXT, adapters(2), ids)
    model = packed_model.PackedWanTransformer(weights, GRIDS, TEXT, adapters(2), torch.tensor([1, -1]))
    assert model.adapter_ids.tolist() == [1, -1]


def test_adapter_ids_need_adapters(weights):
    """A request is not served without the adapter that it asks for."""
    with pytest.raises(ValueError, match="adapter ids must be in"):
        packed_model.PackedWanTransformer(weights, GRIDS, TEXT, None, [0, -1])
    assert packed_model.PackedWanTransformer(weights, GRIDS, TEXT, None, [-1, -1]).adapters is None


def test_negative_lengths(weights):
    with pytest.raises(ValueError, match="negative"):
        packed_model.PackedWanTransformer(weights, GRIDS, [5, -1])
