"""Float64 restatement of the packed-request operators, request by request.

The definitions that ``kernels.residual_norm``, ``kernels.lora_add`` and
``kernels.packed_attention`` are tested against; numpy float64 throughout.
"""

from __future__ import annotations

import numpy as np


def standardise(v, kind, eps):
    """``(v - mean) / sqrt(var + eps)`` ("layer") or ``v / sqrt(mean(v^2) + eps)`` ("rms")."""
    if kind == "layer":
        v = v - v.mean(-1, keepdims=True)
    return v / np.sqrt((v * v).mean(-1, keepdims=True) + eps)


def residual_norm(x, y=None, *, row_request, gate=None, shift=None, scale=None, weight=None,
                  bias=None, norm="layer", post_norm=None, post_weight=None, post_bias=None,
                  eps=1e-6):
    """``(residual, normed)`` of rows ``x``; ``row_request[t]`` indexes the modulation rows."""
    r = x
    if y is not None:
        p = y
        if post_norm is not None:
            p = standardise(p, post_norm, eps)
            p = p * (1.0 if post_weight is None else post_weight)
            p = p + (0.0 if post_bias is None else post_bias)
        r = x + p * (1.0 if gate is None else gate[row_request])
    h = standardise(r, norm, eps)
    h = h * (1.0 if weight is None else weight) + (0.0 if bias is None else bias)
    if scale is not None:
        h = h * (1.0 + scale[row_request])
    return r, h + (0.0 if shift is None else shift[row_request])


def lora_add(y, x, a, b, starts, adapters, scales=None):
    """``y + scales[i] * (x a_i^T) b_i^T`` with adapter ``i = adapters[s]`` for request s's rows."""
    out = y.copy()
    for s, i in enumerate(adapters):
        if i < 0:
            continue
        rows = slice(starts[s], starts[s + 1])
        out[rows] += (1.0 if scales is None else scales[i]) * (x[rows] @ a[i].T) @ b[i].T
    return out


def packed_attention(q, k, v, q_starts, k_starts, causal, scale=None):
    """Softmax attention of each request's queries over its own keys; causal: query i of
    q_len sees keys j <= i + k_len - q_len.  A query without a key gives 0."""
    heads, kv_heads = q.shape[1], k.shape[1]
    scale = q.shape[2] ** -0.5 if scale is None else scale
    out = np.zeros(q.shape)
    for s in range(len(q_starts) - 1):
        n, m = q_starts[s + 1] - q_starts[s], k_starts[s + 1] - k_starts[s]
        qr, kr = slice(q_starts[s], q_starts[s + 1]), slice(k_starts[s], k_starts[s + 1])
        seen = np.ones((n, m), bool)
        if causal:
            seen = np.arange(m)[None] <= np.arange(n)[:, None] + (m - n)
        for h in range(heads):
            g = h * kv_heads // heads
            for i in range(n):
                at = np.flatnonzero(seen[i])
                if not at.size:
                    continue
                w = k[kr, g][at] @ q[qr, h][i] * scale
                w = np.exp(w - w.max())
                out[qr.start + i, h] = (w @ v[kr, g][at]) / w.sum()
    return out
