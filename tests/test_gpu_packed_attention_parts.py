"""Requests of few tokens over long keys (``kernels.packed_attention``): parts of
the keys whose blocks two tiles take in turn, against ``oracle/packed.py``."""

import numpy as np
import pytest
import torch

from oracle import packed as opacked
from test_gpu_packed_attention import U16, call, check, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (5, 1), (16, 2), (3, 3)])
def test_ends_of_blocks_and_parts(heads, kv_heads, causal):
    k_lengths = [4096 + d for d in (-1, 0, 1, 63, 64, 65, 127, 128, 129, 192, 256, 320)]
    t = make([1, 2, 1, 3, 1, 1, 7, 1, 1, 4, 1, 1], k_lengths, heads, kv_heads, seed=heads)
    check(call(t, causal=causal), t, causal)


def test_few_and_many_tokens_beside_each_other():
    """Requests whose tokens fill one tile, both, and several items."""
    q = [1, 16, 17, 32, 33, 70]
    t = make(q, [5000, 3000, 9000, 2049, 1500, 4000], 16, 2, seed=2)
    for causal in (False, True):
        check(call(t, causal=causal), t, causal)


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("keys", [1024, 1100, 1153, 1281, 1409, 2700, 2900, 3000, 5003, 5130])
def test_hidden_values_that_are_not_finite(keys, value):
    """The last key's value is not finite and only the last token sees it: the
    block that holds it is either tile's, and the other tile's keys count once."""
    t = make([4], [keys], 4, 1, seed=keys)
    ref = opacked.packed_attention(*(t[x].double().cpu().numpy() for x in "qkv"), [0, 4], [0, keys], True)
    t["v"][keys - 1] = value
    for _ in range(3):
        out = call(t, causal=True)
        tol = 2 * U16 * np.abs(ref[:3]).max()
        assert np.abs(out[:3].double().cpu().numpy() - ref[:3]).max() <= tol
        assert not out[3].isfinite().any()
