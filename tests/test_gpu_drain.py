"""The kernels' wait for what they have in flight (``mbar_drain``): an earlier
timeout, which ends their other waits after a few polls, does not cut it short,
and its own limit does.  A barrier that nothing arrives on, and a short limit."""

import pytest
import torch

from dit_sparse_atten_b200 import _native

pytestmark = pytest.mark.gpu

LIMIT_NS = 200_000_000          # 200 ms


def test_drain_waits_to_its_own_limit():
    import diag

    device = torch.device("cuda", torch.cuda.current_device())
    word = _native.err_word(device)
    _native.check_device_errors()
    for earlier in (1, 0):
        word.fill_(earlier)
        completed, elapsed_ns, late = diag.unarmed_wait(LIMIT_NS, word, drain=True)
        assert completed == 0 and late == 1
        assert LIMIT_NS <= elapsed_ns < 5 * LIMIT_NS
        with pytest.raises(RuntimeError, match="timed out"):       # reported as any other
            _native.check_device_errors()
    word.fill_(1)
    _, elapsed_ns, _ = diag.unarmed_wait(LIMIT_NS, word)
    assert elapsed_ns < LIMIT_NS                                   # an ordinary wait ends early
    with pytest.raises(RuntimeError, match="timed out"):
        _native.check_device_errors()
