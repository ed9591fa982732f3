"""Cases of the packed-request operators: the fused residual norm, the low-rank
adapters and the packed attention.

A packed batch is one row axis that holds the tokens of several requests one
after the other; ``row_starts`` (int32, on the device, one more entry than
requests) says where each begins.  ``own`` selects between the plain form of
each operator (elementary torch operations in 32 bits) and the framework's
entry points.
"""

import math

import torch

own = False

DEVICE = "cuda"
EPS = 1e-6


# ----------------------------------------------------------------------------
# cases
# ----------------------------------------------------------------------------

def listed():
    return [
        # A block boundary of the 57,600-token layer: both CFG branches, each with its own timestep modulation.
        dict(name="norm_two_branches", op="norm", lengths="28800,28800", width=5120, norm="layer", post="none",
             affine=False, stream="bf16"),
        # Clips of different sizes in one batch, float32 residual stream, affine norm.
        dict(name="norm_ragged_float32", op="norm", lengths="4680,1,2197,0,1560,777,33", width=5120, norm="layer",
             post="none", affine=True, stream="fp32"),
        # A sandwich block (norm of the sub-block's output too) of a narrow model.
        dict(name="norm_sandwich_rms", op="norm", lengths="4095,4095", width=1536, norm="rms", post="rms",
             affine=True, stream="bf16"),
        # One row per request: the latency of a step on single tokens.
        dict(name="norm_single_rows", op="norm", lengths="1,1,1,1,1,1,1,1", width=5120, norm="layer", post="none",
             affine=False, stream="bf16"),
        # Output projection of the 57,600-token layer, one adapter per branch.
        dict(name="lora_two_branches", op="lora", lengths="28800,28800", k=5120, n=5120, rank=32, count=2,
             ids="0,1"),
        # Feed-forward input projection, ragged clips, one request without an adapter.
        dict(name="lora_ffn_ragged", op="lora", lengths="4680,1,2197,0,1560,777,33,512,247", k=5120, n=13824,
             rank=64, count=4, ids="0,1,2,3,-1,1,0,3,2"),
        # Text projection of eight prompts.
        dict(name="lora_text", op="lora", lengths="512,77,130,511,9,256,64,300", k=4096, n=5120, rank=128, count=8,
             ids="0,1,2,3,4,5,6,7"),
        # The timestep projection: one row per request, 16 adapters among 32 requests.
        dict(name="lora_single_rows", op="lora", lengths=",".join(["1"] * 32), k=5120, n=30720, rank=16, count=16,
             ids=",".join(str((7 * i) % 16) for i in range(32))),
        # Cross-attention of four clips to prompts of different lengths.
        dict(name="attention_text", op="attention", q_lengths="7200,7200,6007,1560", k_lengths="512,77,300,129",
             heads=40, kv_heads=40, causal=False),
        # A batch of prompts, causal, five query heads to a key head.
        dict(name="attention_prompts", op="attention",
             q_lengths="512,77,130,511,9,256,64,300,1,899,640,33,450,128,200,721", k_lengths="same", heads=40,
             kv_heads=8, causal=True),
        # One long causal sequence.
        dict(name="attention_long_causal", op="attention", q_lengths="16380", k_lengths="same", heads=16,
             kv_heads=4, causal=True),
        # One new token per request over its long past.
        dict(name="attention_single_tokens", op="attention", q_lengths=",".join(["1"] * 16),
             k_lengths="32760,1560,20001,8192,4680,14040,127,30000,9360,25000,513,18720,1,16384,28080,12345",
             heads=40, kv_heads=8, causal=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _text(values):
    return ",".join(str(v) for v in values)


def _split(rng, total, parts):
    """``parts`` lengths with the given sum: some near-equal, some ragged, a few zero."""
    cuts = sorted(rng.randint(0, total) for _ in range(parts - 1))
    return [b - a for a, b in zip([0] + cuts, cuts + [total])]


def draw(rng):
    op = rng.choice(("norm", "lora", "attention"))
    if op == "norm":
        requests = _log(rng, 1, 64)
        rows = max(requests, _log(rng, 1, 57600))
        return dict(op=op, lengths=_text(_split(rng, rows, requests)),
                    width=rng.choice((256, 1000, 1536, 2048, 4096, 5120, 5120, _log(rng, 64, 5120))),
                    norm=rng.choice(("layer", "rms")), post=rng.choice(("none", "none", "layer", "rms")),
                    affine=rng.random() < 0.5, stream=rng.choice(("bf16", "bf16", "fp32")))
    if op == "lora":
        requests = _log(rng, 1, 48)
        rows = max(requests, _log(rng, 1, 28800))
        lengths = [1] * requests if rng.random() < 0.3 else _split(rng, rows, requests)
        count = _log(rng, 1, 16)
        return dict(op=op, lengths=_text(lengths), k=8 * _log(rng, 8, 640), n=8 * _log(rng, 8, 1728),
                    rank=rng.choice((8, 16, 24, 32, 64, 128)), count=count,
                    ids=_text(rng.choice([-1] + list(range(count)) * 3) for _ in range(requests)))
    kv_heads = rng.choice((1, 2, 4, 8, 40))
    heads = kv_heads * (1 if kv_heads == 40 else rng.choice((1, 2, 3, 4, 5, 8)))
    form = rng.choice(("text", "prompts", "past", "past"))
    if form == "text":
        requests = _log(rng, 1, 8)
        q = _split(rng, max(requests, _log(rng, 64, 14400)), requests)
        k = [_log(rng, 1, 512) for _ in q]
        return dict(op="attention", q_lengths=_text(q), k_lengths=_text(k), heads=heads, kv_heads=kv_heads,
                    causal=False)
    if form == "prompts":
        requests = _log(rng, 1, 24)
        q = _split(rng, max(requests, _log(rng, 64, 4096)), requests)
        return dict(op="attention", q_lengths=_text(q), k_lengths="same", heads=heads, kv_heads=kv_heads,
                    causal=rng.random() < 0.7)
    # new tokens (one, or a few) over a past
    requests = _log(rng, 1, 24)
    q = [rng.choice((1, 1, 1, 1, 2, 5, 17)) for _ in range(requests)]
    k = [n + _log(rng, 1, 16384) - 1 for n in q]
    return dict(op="attention", q_lengths=_text(q), k_lengths=_text(k), heads=heads, kv_heads=kv_heads, causal=True)


def _lengths(text):
    return [int(t) for t in text.split(",")]


def _kv_lengths(case):
    return _lengths(case["q_lengths"] if case["k_lengths"] == "same" else case["k_lengths"])


# ----------------------------------------------------------------------------
# inputs
# ----------------------------------------------------------------------------

def _starts(lengths):
    total, out = 0, [0]
    for n in lengths:
        total += n
        out.append(total)
    return torch.tensor(out, dtype=torch.int32, device=DEVICE)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)

    def normal(*shape, std=1.0, dtype=torch.bfloat16, mean=0.0):
        return torch.randn(shape, generator=g, device=DEVICE).mul_(std).add_(mean).to(dtype)

    s = dict(case)
    if case["op"] == "norm":
        lengths = _lengths(case["lengths"])
        rows, c, requests = sum(lengths), case["width"], len(lengths)
        stream = torch.float32 if case["stream"] == "fp32" else torch.bfloat16
        # hidden states have a few channels far larger than the rest
        loud = torch.where(torch.rand(c, generator=g, device=DEVICE) < 0.01, 12.0, 1.0)
        s["starts"] = _starts(lengths)
        s["x"] = (torch.randn((rows, c), generator=g, device=DEVICE) * loud).to(stream)
        s["y"] = normal(rows, c, std=0.7)
        # [requests, 6, c]: the modulation table plus the projected timestep, as a block splits it
        table = normal(requests, 6, c, std=0.3, dtype=torch.float32)
        s["shift"], s["scale"], s["gate"] = table[:, 0], table[:, 1], table[:, 5]
        s["weight"] = normal(c, std=0.1, mean=1.0) if case["affine"] else None
        s["bias"] = normal(c, std=0.1) if case["affine"] and case["norm"] == "layer" else None
        s["post_weight"] = normal(c, std=0.1, mean=1.0) if case["affine"] and case["post"] != "none" else None
    elif case["op"] == "lora":
        lengths = _lengths(case["lengths"])
        rows = sum(lengths)
        s["starts"] = _starts(lengths)
        s["adapters"] = torch.tensor(_lengths(case["ids"]), dtype=torch.int32, device=DEVICE)
        s["x"] = normal(rows, case["k"])
        s["y"] = normal(rows, case["n"])
        s["a"] = normal(case["count"], case["rank"], case["k"], std=1.0 / math.sqrt(case["k"]))
        s["b"] = normal(case["count"], case["n"], case["rank"], std=0.5 / math.sqrt(case["rank"]))
        s["scales"] = torch.rand(case["count"], generator=g, device=DEVICE) + 0.5
    else:
        q_len, k_len = _lengths(case["q_lengths"]), _kv_lengths(case)
        s["q_starts"], s["k_starts"] = _starts(q_len), _starts(k_len)
        s["q_longest"], s["k_longest"] = max(q_len), max(k_len)
        s["q"] = normal(sum(q_len), case["heads"], 128, std=1.5)
        s["k"] = normal(sum(k_len), case["kv_heads"], 128)
        s["v"] = normal(sum(k_len), case["kv_heads"], 128)
    return s


# ----------------------------------------------------------------------------
# passes
# ----------------------------------------------------------------------------

def _request_of_row(starts, rows):
    return torch.searchsorted(starts[1:], torch.arange(rows, device=starts.device, dtype=starts.dtype), right=True)


def _plain_normalise(v, kind, weight, bias):
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    v = v * torch.rsqrt((v * v).mean(-1, keepdim=True) + EPS)
    if weight is not None:
        v = v * weight.float()
    return v if bias is None else v + bias.float()


def _plain_norm(s):
    at = _request_of_row(s["starts"], s["x"].shape[0])
    p = s["y"].float()
    if s["post"] != "none":
        p = _plain_normalise(p, s["post"], s["post_weight"], None)
    r = s["x"].float() + s["gate"][at] * p
    h = _plain_normalise(r, s["norm"], s["weight"], s["bias"])
    h = h * (1 + s["scale"][at]) + s["shift"][at]
    return {"residual": r.to(s["x"].dtype), "normed": h.to(torch.bfloat16)}


def _plain_lora(s):
    count, rank = s["count"], s["rank"]
    row_adapter = s["adapters"][_request_of_row(s["starts"], s["x"].shape[0])]
    column_adapter = torch.arange(count, device=row_adapter.device).repeat_interleave(rank)
    t = s["x"].float() @ s["a"].float().reshape(count * rank, -1).t()
    t = t * (row_adapter[:, None] == column_adapter[None]) * s["scales"].repeat_interleave(rank)
    delta = t @ s["b"].float().transpose(1, 2).reshape(count * rank, -1)
    return {"out": (s["y"].float() + delta).to(s["y"].dtype)}


def _padded(x, starts, longest):
    """``[requests, heads, longest, D]`` float32 of packed ``[rows, heads, D]``."""
    at = starts[:-1, None] + torch.arange(longest, device=starts.device)
    return x[at.clamp_(max=x.shape[0] - 1)].float().transpose(1, 2)


def _plain_attention(s):
    q_starts, k_starts, kv = s["q_starts"], s["k_starts"], s["kv_heads"]
    requests, group = q_starts.numel() - 1, s["heads"] // kv
    q = _padded(s["q"], q_starts, s["q_longest"]).reshape(requests, kv, group * s["q_longest"], 128)
    k = _padded(s["k"], k_starts, s["k_longest"])
    v = _padded(s["v"], k_starts, s["k_longest"])
    q_len = (q_starts[1:] - q_starts[:-1])[:, None, None]
    k_len = (k_starts[1:] - k_starts[:-1])[:, None, None]
    i = torch.arange(s["q_longest"], device=q.device)[None, :, None]
    j = torch.arange(s["k_longest"], device=q.device)[None, None]
    hidden = (j >= k_len) | (j > i + k_len - q_len if s["causal"] else False)
    w = (q @ k.transpose(2, 3)).mul_(1 / math.sqrt(128))
    w = w.view(requests, kv, group, s["q_longest"], s["k_longest"])
    w.masked_fill_(hidden[:, None, None], -math.inf)
    top = w.amax(-1, keepdim=True)
    w.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = w.sum(-1, keepdim=True)
    o = (w.view(requests, kv, group * s["q_longest"], s["k_longest"]) @ v).view(*w.shape[:4], 128)
    o = torch.where(total > 0, o / total, 0.0)
    o = o.reshape(requests, s["heads"], s["q_longest"], 128)
    row = torch.arange(s["q"].shape[0], device=q.device)
    at = _request_of_row(q_starts, row.numel())
    return {"out": o[at, :, row - q_starts[at]].to(s["q"].dtype)}


def _own_norm(s):
    from dit_sparse_atten_b200 import kernels
    residual, normed = kernels.residual_norm(
        s["x"], s["y"], gate=s["gate"], shift=s["shift"], scale=s["scale"], weight=s["weight"], bias=s["bias"],
        norm=s["norm"], post_norm=None if s["post"] == "none" else s["post"], post_weight=s["post_weight"], eps=EPS,
        row_starts=s["starts"], normed_dtype=torch.bfloat16)
    return {"residual": residual, "normed": normed}


def _own_lora(s):
    from dit_sparse_atten_b200 import kernels
    return {"out": kernels.lora_add(s["y"], s["x"], s["a"], s["b"], row_starts=s["starts"], adapters=s["adapters"],
                                    scales=s["scales"])}


def _own_attention(s):
    from dit_sparse_atten_b200 import kernels
    return {"out": kernels.packed_attention(s["q"], s["k"], s["v"], s["q_starts"], s["k_starts"],
                                            causal=s["causal"])}


def run(state):
    if own:
        return {"norm": _own_norm, "lora": _own_lora, "attention": _own_attention}[state["op"]](state)
    return {"norm": _plain_norm, "lora": _plain_lora, "attention": _plain_attention}[state["op"]](state)


# ----------------------------------------------------------------------------
# what a pass cannot do without
# ----------------------------------------------------------------------------

def work(case):
    if case["op"] == "norm":
        lengths = _lengths(case["lengths"])
        rows, c = sum(lengths), case["width"]
        stream = 4 if case["stream"] == "fp32" else 2
        tables = 3 * 4 * c * sum(1 for n in lengths if n) + (6 * c if case["affine"] else 0)
        return {"bytes": rows * c * (2 * stream + 4) + tables, "flops": rows * c * 12}
    if case["op"] == "lora":
        lengths, ids = _lengths(case["lengths"]), _lengths(case["ids"])
        rows, k, n, rank = sum(lengths), case["k"], case["n"], case["rank"]
        with_adapter = sum(m for m, a in zip(lengths, ids) if a >= 0)
        used = len({a for m, a in zip(lengths, ids) if m and a >= 0})
        return {"bytes": 2 * (with_adapter * k + 2 * rows * n + used * rank * (k + n)),
                "flops": 2 * with_adapter * rank * (k + n)}
    q_len, k_len = _lengths(case["q_lengths"]), _kv_lengths(case)
    pairs = 0
    for a, b in zip(q_len, k_len):
        if not case["causal"]:
            pairs += a * b
        else:  # query i sees min(b, max(0, i + 1 + b - a)) keys
            first = max(0, a - b)
            pairs += (a - first) * (b - a + 1) + (first + a - 1) * (a - first) // 2 if a > first else 0
    rows = 2 * sum(q_len) * case["heads"] + 2 * sum(k_len) * case["kv_heads"]
    return {"bytes": rows * 128 * 2, "flops": 4 * 128 * case["heads"] * pairs}


# ----------------------------------------------------------------------------
# the definitions in 64 bits, request by request
# ----------------------------------------------------------------------------

def _exact_standardised(v, kind):
    mean = v.sum(-1, keepdim=True) / v.shape[-1] if kind == "layer" else 0.0
    centred = v - mean
    return centred / (centred.pow(2).sum(-1, keepdim=True) / v.shape[-1] + EPS).sqrt()


def _exact_norm(s, lengths):
    residual, normed, begin = [], [], 0
    for r, n in enumerate(lengths):
        x, y = s["x"][begin:begin + n].double(), s["y"][begin:begin + n].double()
        begin += n
        if s["post"] != "none":
            y = _exact_standardised(y, s["post"]) * (s["post_weight"].double() if s["affine"] else 1.0)
        x = x + y * s["gate"][r].double()
        h = _exact_standardised(x, s["norm"])
        if s["weight"] is not None:
            h = h * s["weight"].double()
        if s["bias"] is not None:
            h = h + s["bias"].double()
        residual.append(x)
        normed.append(h + h * s["scale"][r].double() + s["shift"][r].double())
    return {"residual": torch.cat(residual), "normed": torch.cat(normed)}


def _exact_lora(s, lengths, ids):
    out, begin = [], 0
    for n, a in zip(lengths, ids):
        y = s["y"][begin:begin + n].double()
        if a >= 0 and n:
            low = torch.einsum("tk,rk->tr", s["x"][begin:begin + n].double(), s["a"][a].double())
            y = y + torch.einsum("tr,nr->tn", low, s["b"][a].double()) * float(s["scales"][a])
        out.append(y)
        begin += n
    return {"out": torch.cat(out)}


def _exact_attention(s, q_len, k_len):
    heads, group = s["heads"], s["heads"] // s["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEVICE)
    q0 = k0 = 0
    for a, b in zip(q_len, k_len):
        for h in range(heads if a and b else 0):
            k = s["k"][k0:k0 + b, h // group].double()
            v = s["v"][k0:k0 + b, h // group].double()
            for at in range(0, a, 8192):
                q = s["q"][q0 + at:q0 + min(a, at + 8192), h].double()
                score = torch.einsum("id,jd->ij", q, k) / math.sqrt(128)
                if s["causal"]:
                    last = torch.arange(at, at + q.shape[0], device=DEVICE) + (b - a)
                    score[torch.arange(b, device=DEVICE)[None] > last[:, None]] = -math.inf
                weight = torch.softmax(score, -1).nan_to_num_(0.0)
                out[q0 + at:q0 + at + q.shape[0], h] = torch.einsum("ij,jd->id", weight, v)
        q0 += a
        k0 += b
    return {"out": out}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        return _exact_norm(s, _lengths(case["lengths"]))
    if case["op"] == "lora":
        return _exact_lora(s, _lengths(case["lengths"]), _lengths(case["ids"]))
    return _exact_attention(s, _lengths(case["q_lengths"]), _kv_lengths(case))
