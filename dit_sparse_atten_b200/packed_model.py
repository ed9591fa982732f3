"""Wan transformer forward for several requests at once.

``wan_model.WanTransformer`` runs one request: one token grid, one timestep,
one text, the base weights.  A server has several -- clips of different sizes,
CFG branches, prompts of different lengths, each with its own timestep and
perhaps its own low-rank adapter.  Here their tokens lie one after the other on
one row axis, so every projection is one product over all of them, and three
operators keep the requests apart (``kernels``):

* ``residual_norm``: a sub-block's gate, the residual and the next sub-block's
  modulated norm in one pass, the modulation rows picked by request;
* ``lora_add``: each request's adapter beside a shared projection;
* ``packed_attention``: self-attention within each request and cross-attention
  to its own text.

Same block as ``wan_model`` (reference ``wan_diffusers.py:75-191``), on one
GPU.  A request's routed self-attention can be kept: pass ``self_attention``.
"""

from __future__ import annotations

import itertools
import math

import torch
import torch.nn.functional as F

from . import kernels
from .wan_model import WanWeights, _linear, fused_prologue, rotary_tables, timestep_embedding

# projections that an adapter may have, per block; TIME_PROJ is the model's own
BLOCK_PROJECTIONS = ("q", "k", "v", "o", "q2", "o2", "ffn1", "ffn2")
TIME_PROJ = "time_proj"


def row_starts(lengths, device) -> torch.Tensor:
    """Offsets of packed requests: int32 ``[len(lengths) + 1]`` on ``device``."""
    return torch.tensor([0, *itertools.accumulate(lengths)], dtype=torch.int32, device=device)


class LoraAdapters:
    """Low-rank adapters of one model: ``blocks[i][name] = (a, b)`` with ``a``
    bf16 ``[count, R, in]`` and ``b`` bf16 ``[count, out, R]`` for block i's
    projection ``name`` (``BLOCK_PROJECTIONS``; absent: no adapter has one),
    ``time_proj`` the same for the timestep projection, ``scales`` float32
    ``[count]``."""

    def __init__(self, blocks, scales, time_proj=None):
        for factors in blocks:
            unknown = set(factors) - set(BLOCK_PROJECTIONS)
            if unknown:
                raise ValueError(f"unknown projections {sorted(unknown)}")
        self.blocks = list(blocks)
        self.scales = scales
        self.time_proj = time_proj


class PackedWanTransformer:
    """Forward of several requests: ``grids`` their token grids, ``text_lengths``
    their numbers of text tokens, ``adapter_ids`` which adapter of ``adapters``
    each uses (-1: none)."""

    def __init__(self, weights: WanWeights, grids, text_lengths, adapters: LoraAdapters | None = None,
                 adapter_ids=None):
        device = weights.patch[0].device
        self.w, self.cfg = weights, weights.cfg
        self.grids = [tuple(g) for g in grids]
        if len(self.grids) != len(text_lengths):
            raise ValueError("one text length for each grid")
        if adapters is not None and len(adapters.blocks) != self.cfg.layers:
            raise ValueError("adapters must have the model's number of blocks")
        self.lengths = [math.prod(g) for g in self.grids]
        self.text_lengths = [int(n) for n in text_lengths]
        if min(self.lengths + self.text_lengths, default=0) < 0:
            raise ValueError("grids and text lengths must not be negative")
        self.starts = row_starts(self.lengths, device)
        self.text_starts = row_starts(self.text_lengths, device)
        self.adapters = adapters
        ids = [-1] * len(self.grids) if adapter_ids is None else [int(i) for i in adapter_ids]
        if len(ids) != len(self.grids):
            raise ValueError("one adapter id for each grid")
        count = adapters.scales.numel() if adapters is not None else 0
        if any(not -1 <= i < count for i in ids):
            raise ValueError(f"adapter ids must be in [-1, {count})")
        self.adapter_ids = torch.tensor(ids, dtype=torch.int32, device=device)
        self.request_starts = row_starts([1] * len(ids), device)   # a row for each request
        tables = [rotary_tables(self.cfg, g) for g in self.grids]
        self.rope = tuple(torch.cat(t).to(device) for t in zip(*tables))
        self.prologue = fused_prologue(self.cfg.heads, self.cfg.eps)

    def context(self, text):
        """Packed text conditioning ``[sum(text_lengths), text_dim]`` -> ``[.., dim]``."""
        return _linear(F.gelu(_linear(text, self.w.text_1), approximate="tanh"), self.w.text_2)

    def _adapted(self, x, weight, factors, starts):
        """Shared projection of the packed rows ``x`` plus each request's adapter, in place."""
        y = _linear(x, weight)
        if factors is None:
            return y
        return kernels.lora_add(y, x, *factors, row_starts=starts, adapters=self.adapter_ids,
                                scales=self.adapters.scales, out=y)

    def forward(self, patches, timesteps, ctx, self_attention=None):
        """Noise prediction ``[T, out * 4]`` of the packed ``patches [T, C * 4]``
        at one timestep for each request.  ``self_attention(request, layer, q, k, v)``
        replaces the dense self-attention of one request (``[1, n, H, D]``
        tensors, as an attention backend takes them)."""
        cfg, w = self.cfg, self.w
        dtype, device = w.patch[0].dtype, patches.device
        if len(timesteps) != len(self.grids):
            raise ValueError("one timestep for each request")
        rows, text_rows = sum(self.lengths), sum(self.text_lengths)
        if tuple(patches.shape) != (rows, w.patch[0].shape[1]):
            raise ValueError(f"patches must be {(rows, w.patch[0].shape[1])}, a row for each token")
        if tuple(ctx.shape) != (text_rows, cfg.dim):
            raise ValueError(f"ctx must be {(text_rows, cfg.dim)}, the context of the packed texts")
        emb = torch.cat([timestep_embedding(t, cfg.freq_dim) for t in timesteps]).to(device, dtype)
        temb = _linear(F.silu(_linear(emb, w.time_1)), w.time_2)         # [requests, dim]
        time_factors = self.adapters.time_proj if self.adapters is not None else None
        tproj = self._adapted(F.silu(temb), w.time_proj, time_factors, self.request_starts)
        tproj = tproj.unflatten(1, (6, cfg.dim)).float()
        mods = [blk["table"] + tproj for blk in w.blocks]                # [requests, 6, dim]
        out_mod = w.out_table + temb.float()[:, None]                    # [requests, 2, dim]
        x = _linear(patches.to(dtype), w.patch)                          # [T, dim]
        h = self._norm(x, None, shift=mods[0][:, 0], scale=mods[0][:, 1]).normed
        for layer, (blk, mod) in enumerate(zip(w.blocks, mods)):
            lora = self.adapters.blocks[layer] if self.adapters is not None else {}

            def linear(t, name):
                return self._adapted(t, blk[name], lora.get(name), self.starts)

            q, k, v = self.prologue(linear(h, "q"), linear(h, "k"), linear(h, "v"), blk, *self.rope)
            a = self._self_attention(q[0], k[0], v[0], layer, self_attention)
            x, h = self._norm(x, linear(a.flatten(1), "o"), gate=mod[:, 2], weight=blk["norm2_w"],
                              bias=blk["norm2_b"])
            a = self._cross_attention(linear(h, "q2"), ctx, blk)
            x, h = self._norm(x, linear(a.flatten(1), "o2"), shift=mod[:, 3], scale=mod[:, 4])
            f = linear(F.gelu(linear(h, "ffn1"), approximate="tanh"), "ffn2")
            after = mods[layer + 1] if layer + 1 < cfg.layers else out_mod
            x, h = self._norm(x, f, gate=mod[:, 5], shift=after[:, 0], scale=after[:, 1])
        return _linear(h, w.proj_out)

    def _norm(self, x, y, **kw):
        return kernels.residual_norm(x, y, eps=self.cfg.eps, row_starts=self.starts, **kw)

    def _self_attention(self, q, k, v, layer, custom):
        if custom is None:
            return kernels.packed_attention(q, k, v, self.starts)
        out = torch.empty_like(q)
        begin = 0
        for request, n in enumerate(self.lengths):
            rows = slice(begin, begin + n)
            out[rows] = custom(request, layer, q[None, rows], k[None, rows], v[None, rows])[0]
            begin += n
        return out

    def _cross_attention(self, q, ctx, blk):
        heads, eps = self.cfg.heads, self.cfg.eps
        q = kernels.residual_norm(q, weight=blk["norm_q2"], norm="rms", eps=eps).normed
        k = kernels.residual_norm(_linear(ctx, blk["k2"]), weight=blk["norm_k2"], norm="rms",
                                  eps=eps).normed
        v = _linear(ctx, blk["v2"])
        return kernels.packed_attention(*(t.unflatten(1, (heads, -1)) for t in (q, k, v)),
                                        self.starts, self.text_starts)
