"""Cases of the INT8 head path, from the last hidden state to the next token, for timing and comparison:

  norm     residual addition, RMS norm and quantisation of each row to int8 with one scale
           (pollux_b200.int8.add_rms_norm_int8), read back by dequantize_rows_int8
  linear   product of int8 rows with an INT8 layer, scales for each token and each output channel
           (pollux_b200.int8.int8_linear)
  sample   one token a row under temperature, top-k, top-p and min-p from given uniform numbers
           (pollux_b200.sampling.sample_tokens)

With ``own`` false, ``run`` computes the same things with elementary torch operations in 32 bits.
"""
from __future__ import annotations

import torch

own = False

EPS = 1e-6
FLOOR = 1e-8            # smallest largest-magnitude of a quantised row
WEIGHT_ONE = 2.0 ** 40  # fixed-point weight of the most probable token
DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"fp32": 4, "fp16": 2, "bf16": 2}


def listed():
    return [
        # One token of the d=1920 model on its way to the head: latency.
        {"name": "norm 1x1920 bf16", "op": "norm", "tokens": 1, "cols": 1920, "dtype": "bf16", "residual": True},
        # Four prompts of 1024 tokens.
        {"name": "norm 4096x1920 bf16", "op": "norm", "tokens": 4096, "cols": 1920, "dtype": "bf16", "residual": True},
        # A ragged batch in a width that is no multiple of a vector, fp32, the first norm (no residual yet).
        {"name": "norm 531x1153 fp32", "op": "norm", "tokens": 531, "cols": 1153, "dtype": "fp32", "residual": False},
        # One decoding step of one sequence through the d=1920 head: the head's bytes.
        {"name": "linear 1x50688x1920 fp32", "op": "linear", "tokens": 1, "out": 50688, "in": 1920, "dtype": "fp32", "bias": False},
        # A decoding step of 32 sequences through an MLP's first layer.
        {"name": "linear 32x7680x1920 bf16", "op": "linear", "tokens": 32, "out": 7680, "in": 1920, "dtype": "bf16", "bias": False},
        # A ragged prompt through an MLP's second layer, with a bias: few output tiles, a long sum.
        {"name": "linear 333x1920x7680 fp16", "op": "linear", "tokens": 333, "out": 1920, "in": 7680, "dtype": "fp16", "bias": True},
        # Four prompts of 1024 tokens through an MLP's first layer: arithmetic.
        {"name": "linear 4096x7680x1920 bf16", "op": "linear", "tokens": 4096, "out": 7680, "in": 1920, "dtype": "bf16", "bias": False},
        # Scoring every position of one 1024-token sequence: fp32 logits of the whole vocabulary.
        {"name": "linear 1024x50688x1920 fp32", "op": "linear", "tokens": 1024, "out": 50688, "in": 1920, "dtype": "fp32", "bias": False},
        # One sequence, the usual settings: latency.
        {"name": "sample 1x50688 fp32", "op": "sample", "rows": 1, "vocab": 50688, "dtype": "fp32", "params": "scalar",
         "temperature": 0.8, "top_k": 50, "top_p": 0.9, "min_p": 0.0},
        # A few sequences over a small odd vocabulary.
        {"name": "sample 9x1009 fp16", "op": "sample", "rows": 9, "vocab": 1009, "dtype": "fp16", "params": "scalar",
         "temperature": 1.0, "top_k": 0, "top_p": 0.9, "min_p": 0.0},
        # A batch with a wide nucleus and min-p, 16-bit logits (many exact ties).
        {"name": "sample 64x50688 bf16", "op": "sample", "rows": 64, "vocab": 50688, "dtype": "bf16", "params": "scalar",
         "temperature": 1.0, "top_k": 0, "top_p": 0.95, "min_p": 0.02},
        # A large batch in which every sequence has settings of its own, greedy ones among them.
        {"name": "sample 512x50688 fp32", "op": "sample", "rows": 512, "vocab": 50688, "dtype": "fp32", "params": "rows",
         "temperature": 0.0, "top_k": 0, "top_p": 0.0, "min_p": 0.0},
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], even over the logarithm."""
    return max(lo, min(hi, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    op = rng.choice(["norm", "linear", "sample"])
    dtype = rng.choice(["fp32", "fp16", "bf16"])
    if op == "norm":
        cols = _spread(rng, 24, 8192)
        if rng.random() < 0.6:
            cols = -(-cols // 24) * 24
        tokens = min(_spread(rng, 1, 4096), 4096 * 1920 // cols)
        return {"op": op, "tokens": max(1, tokens), "cols": cols, "dtype": dtype, "residual": rng.random() < 0.7}
    if op == "linear":
        out, k = _spread(rng, 24, 50688), _spread(rng, 24, 7680)
        if rng.random() < 0.75:
            k = -(-k // 48) * 48
        tokens = min(_spread(rng, 1, 4096), 4096 * 7680 * 1920 // (out * k), 1024 * 50688 // out)
        return {"op": op, "tokens": max(1, tokens), "out": out, "in": k, "dtype": dtype, "bias": rng.random() < 0.3}
    vocab = _spread(rng, 200, 131072)
    rows = max(1, min(_spread(rng, 1, 512), 512 * 50688 // vocab))
    if rng.random() < 0.3:
        return {"op": op, "rows": rows, "vocab": vocab, "dtype": dtype, "params": "rows",
                "temperature": 0.0, "top_k": 0, "top_p": 0.0, "min_p": 0.0}
    return {"op": op, "rows": rows, "vocab": vocab, "dtype": dtype, "params": "scalar",
            "temperature": rng.choice([0.0, 0.5, 0.7, 0.8, 1.0, 1.3]), "top_k": rng.choice([0, 0, 1, 20, 50, 100]),
            "top_p": rng.choice([1.0, 0.8, 0.9, 0.95, 0.99]), "min_p": rng.choice([0.0, 0.0, 0.02, 0.1])}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dev = "cuda"
    if case["op"] == "norm":
        t, c, dt = case["tokens"], case["cols"], DTYPES[case["dtype"]]
        # A residual stream with a few channels much larger than the rest.
        channel = torch.where(torch.rand(c, generator=g, device=dev) < 0.005, 12.0, 1.0)
        x = (torch.randn(t, c, generator=g, device=dev) * 0.7).to(dt)
        r = (torch.randn(t, c, generator=g, device=dev) * 2.0 * channel).to(dt) if case["residual"] else None
        w = (1.0 + 0.2 * torch.randn(c, generator=g, device=dev)).to(dt)
        return {"case": case, "x": x, "residual": r, "weight": w}
    if case["op"] == "linear":
        t, o, k = case["tokens"], case["out"], case["in"]
        # Normed activations and N(0, 0.02^2) weights, quantised row by row.
        x = torch.randn(t, k, generator=g, device=dev)
        a = x.abs().amax(dim=1, keepdim=True).clamp_min(FLOOR)
        q = torch.round(x / a * 127.0).to(torch.int8)
        scale = (a / 127.0).reshape(t)
        del x
        w = torch.randn(o, k, generator=g, device=dev)
        m = w.abs().amax(dim=1, keepdim=True).clamp_min(FLOOR)
        w8 = torch.round(w / m * 127.0).to(torch.int8)
        mu = (m * 0.02).reshape(o).to(torch.float16)
        bias = torch.randn(o, generator=g, device=dev) * 0.1 if case["bias"] else None
        return {"case": case, "q": q, "scale": scale, "weight_int8": w8, "mu_rows": mu, "bias": bias}
    b, v = case["rows"], case["vocab"]
    # A next-token distribution: probabilities that fall off with the rank, in
    # a shuffled order, with noise; one token in a hundred is banned.
    rank = torch.rand(b, v, generator=g, device=dev) * v + 1.0
    logits = 12.0 - 1.3 * torch.log(rank) + 0.8 * torch.randn(b, v, generator=g, device=dev)
    logits = logits.masked_fill(torch.rand(b, v, generator=g, device=dev) < 0.01, float("-inf"))
    logits = logits.to(DTYPES[case["dtype"]])
    u = torch.rand(b, generator=g, device=dev)
    par = {k: case[k] for k in ("temperature", "top_k", "top_p", "min_p")}
    if case["params"] == "rows":
        pick = torch.rand(4, b, generator=g, device=dev)
        par["temperature"] = torch.where(pick[0] < 0.2, 0.0, 0.3 + pick[0])
        par["top_k"] = torch.where(pick[1] < 0.5, 0.0, pick[1] * 100).to(torch.int32)
        par["top_p"] = torch.where(pick[2] < 0.4, 1.0, 0.4 + 0.6 * pick[2])
        par["min_p"] = torch.where(pick[3] < 0.7, 0.0, 0.1 * pick[3])
    return {"case": case, "logits": logits, "u": u, "params": par}


def run(state):
    op = state["case"]["op"]
    if op == "norm":
        return _norm_own(state) if own else _norm_plain(state)
    if op == "linear":
        return _linear_own(state) if own else _linear_plain(state)
    return _sample_own(state) if own else _sample_plain(state)


def _norm_own(s):
    from pollux_b200 import int8
    q, scale, residual = int8.add_rms_norm_int8(s["x"], s["weight"], residual=s["residual"], eps=EPS)
    values = int8.dequantize_rows_int8(q, scale, dtype=torch.bfloat16)
    return {"values": values} if residual is None else {"values": values, "residual": residual}


def _norm_plain(s):
    x = s["x"].float()
    if s["residual"] is not None:
        x = x + s["residual"].float()
    y = x * torch.rsqrt(x.square().mean(dim=-1, keepdim=True) + EPS) * s["weight"].float()
    mu = y.abs().amax(dim=-1, keepdim=True).clamp_min(FLOOR)
    q = torch.round(y / mu * 127.0).clamp(-128.0, 127.0)
    values = (q * (mu / 127.0)).to(torch.bfloat16)
    return {"values": values} if s["residual"] is None else {"values": values, "residual": x.to(s["x"].dtype)}


def _linear_own(s):
    from pollux_b200 import int8
    return int8.int8_linear(s["q"], s["scale"], s["weight_int8"], s["mu_rows"], bias=s["bias"],
                            out_dtype=DTYPES[s["case"]["dtype"]])


def _linear_plain(s):
    y = torch.matmul(s["q"].float(), s["weight_int8"].float().t())
    # The layer's reconstruction scale is fp16(mu / 127).
    y = y * s["scale"].unsqueeze(1) * (s["mu_rows"].float() / 127.0).half().float()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(DTYPES[s["case"]["dtype"]])


def _sample_own(s):
    from pollux_b200 import sampling
    token, logprob = sampling.sample_tokens(s["logits"], s["u"], return_logprob=True, **s["params"])
    return {"token": token, "logprob": logprob}


def _column(v, b, dtype, device):
    return (v.to(dtype) if isinstance(v, torch.Tensor) else torch.full((b,), v, dtype=dtype, device=device)).unsqueeze(1)


def _sample_plain(s):
    """The operator's definition: tokens ordered by scaled logit (ties: lowest
    index), fixed-point weights so that sums do not depend on their order."""
    logits, p, dev = s["logits"].float(), s["params"], s["logits"].device
    b, v = logits.shape
    t = _column(p["temperature"], b, torch.float32, dev)
    k = _column(p["top_k"], b, torch.int64, dev)
    top_p = _column(p["top_p"], b, torch.float32, dev)
    min_p = _column(p["min_p"], b, torch.float32, dev)
    k = torch.where(t > 0, torch.where(k > 0, k, v), 1)
    z = (logits - logits.amax(dim=1, keepdim=True)) * (1.0 / torch.where(t > 0, t, 1.0))
    w = torch.round(torch.exp(z) * WEIGHT_ONE).to(torch.int64)
    total = w.sum(dim=1, keepdim=True)
    order = torch.sort(z, dim=1, descending=True, stable=True).indices
    ws = w.gather(1, order)
    ws = torch.where(torch.arange(v, device=dev) < k, ws, 0)
    before = ws.cumsum(dim=1) - ws
    limit = torch.ceil(top_p.double() * ws.sum(dim=1, keepdim=True).double()).to(torch.int64)
    keep = (before < limit.clamp_min(1)) | (top_p >= 1.0)
    keep &= ws >= torch.ceil(min_p.double().clamp(0.0, 1.0) * WEIGHT_ONE).to(torch.int64)
    wk = torch.zeros_like(w).scatter_(1, order, torch.where(keep, ws, 0))
    run_sum = wk.cumsum(dim=1)
    mass = run_sum[:, -1:]
    target = torch.minimum(torch.floor(s["u"].double().unsqueeze(1) * mass.double()).to(torch.int64), mass - 1)
    token = (run_sum <= target).sum(dim=1)
    logprob = z.gather(1, token.unsqueeze(1)) - torch.log((total.double() / WEIGHT_ONE).float())
    return {"token": token, "logprob": logprob.squeeze(1)}


def work(case):
    if case["op"] == "norm":
        n, s = case["tokens"] * case["cols"], SIZE[case["dtype"]]
        # x (and the residual in and out), the gains, the bf16 values.
        return {"bytes": n * (s * (3 if case["residual"] else 1) + 2) + case["cols"] * s, "flops": 8 * n}
    if case["op"] == "linear":
        t, o, k = case["tokens"], case["out"], case["in"]
        return {"bytes": t * k + o * k + t * 4 + o * 2 + (o * 4 if case["bias"] else 0) + t * o * SIZE[case["dtype"]],
                "flops": 2 * t * o * k}
    return {"bytes": case["rows"] * (case["vocab"] * SIZE[case["dtype"]] + 4 + 8 + 4),
            "flops": 8 * case["rows"] * case["vocab"]}


def exact(case, seed):
    """The definitions in 64 bits."""
    s = prepare(case, seed)
    if case["op"] == "norm":
        x = s["x"].double()
        if s["residual"] is not None:
            x = x + s["residual"].double()
        y = x / torch.sqrt((x * x).sum(dim=-1, keepdim=True) / x.shape[-1] + EPS) * s["weight"].double()
        step = torch.maximum(y.abs().max(dim=-1, keepdim=True).values, torch.full_like(y[:, :1], FLOOR)) / 127.0
        values = torch.round(y / step) * step
        return {"values": values} if s["residual"] is None else {"values": values, "residual": x}
    if case["op"] == "linear":
        y = torch.einsum("tk,ok->to", s["q"].double(), s["weight_int8"].double())
        y = y * s["scale"].double()[:, None] * (s["mu_rows"].float() / 127.0).half().double()[None, :]
        return y if s["bias"] is None else y + s["bias"].double()[None, :]
    out = torch.empty(case["rows"], dtype=torch.float64, device="cuda")
    full = {k: _column(v, case["rows"], torch.float64, "cuda").squeeze(1).tolist() for k, v in s["params"].items()}
    for i in range(case["rows"]):
        z = s["logits"][i].double()
        z = (z - z.max()) / (full["temperature"][i] if full["temperature"][i] > 0 else 1.0)
        e = torch.exp(z)
        order = torch.argsort(z, descending=True, stable=True)
        k = 1 if full["temperature"][i] <= 0 else int(full["top_k"][i]) or z.numel()
        top = e[order[:k]]
        keep = torch.ones_like(top, dtype=torch.bool)
        if full["top_p"][i] < 1.0:
            keep = top.cumsum(0) - top < full["top_p"][i] * top.sum()
            keep[0] = True
        keep &= top >= full["min_p"][i]
        kept = torch.zeros_like(e)
        kept[order[:k][keep]] = top[keep]
        c = kept.cumsum(0)
        token = int((c <= s["u"][i].double() * c[-1]).sum().clamp_max(z.numel() - 1))
        out[i] = z[token] - torch.log(e.sum())
    return {"token": None, "logprob": out}
