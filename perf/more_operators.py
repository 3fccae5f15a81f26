"""Cases of the training head path, from the residual stream to the loss and back, for timing and comparison:

  norm   residual addition and RMS or layer norm, forward alone or with the gradients of both outputs
         (pollux_b200.norm.add_rms_norm, add_layer_norm)
  loss   softmax cross entropy of a head's product, without its logits: each token's loss alone ("score") or
         the loss with the gradients of the states and of the head (pollux_b200.loss.linear_cross_entropy)

With ``own`` false, ``run`` computes the same things with elementary torch operations in 32 bits.
"""
from __future__ import annotations

import torch

own = False

IGNORE = -100
DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"fp32": 4, "fp16": 2, "bf16": 2}
EPS = {"rms": 1e-6, "layer": 1e-5}


def listed():
    return [
        # One token of the d=1920 model on its way to an unquantised head: latency.
        {"name": "norm rms 1x1920 bf16", "op": "norm", "kind": "rms", "tokens": 1, "cols": 1920, "dtype": "bf16",
         "residual": True, "train": False},
        # A training step's norm over 16 sequences of 1024 tokens, with the gradient that comes down the residual.
        {"name": "norm rms 16384x1920 bf16 train", "op": "norm", "kind": "rms", "tokens": 16384, "cols": 1920,
         "dtype": "bf16", "residual": True, "train": True},
        # The widest rows of the d=1920 model (its MLP's inner width).
        {"name": "norm layer 8192x7680 bf16 train", "op": "norm", "kind": "layer", "tokens": 8192, "cols": 7680,
         "dtype": "bf16", "residual": True, "train": True},
        # Four sequences of the d=1152 model in fp32, the first norm (no residual yet).
        {"name": "norm layer 4096x1152 fp32 train", "op": "norm", "kind": "layer", "tokens": 4096, "cols": 1152,
         "dtype": "fp32", "residual": False, "train": True},
        # A ragged batch in a width that is no multiple of a vector.
        {"name": "norm layer 777x1153 fp16 train", "op": "norm", "kind": "layer", "tokens": 777, "cols": 1153,
         "dtype": "fp16", "residual": True, "train": True},
        # A few tokens over a small odd vocabulary: latency.
        {"name": "loss 9x1009x240 fp16 score", "op": "loss", "tokens": 9, "vocab": 1009, "in": 240, "dtype": "fp16",
         "train": False, "reduction": "none", "masked": 0.0},
        # The log-likelihood of one more token under the d=1920 model: the head's bytes.
        {"name": "loss 1x50688x1920 bf16 score", "op": "loss", "tokens": 1, "vocab": 50688, "in": 1920,
         "dtype": "bf16", "train": False, "reduction": "none", "masked": 0.0},
        # Scoring every position of one 1024-token sequence.
        {"name": "loss 1024x50688x1920 bf16 score", "op": "loss", "tokens": 1024, "vocab": 50688, "in": 1920,
         "dtype": "bf16", "train": False, "reduction": "none", "masked": 0.0},
        # A ragged micro-batch over an odd vocabulary and width, some of it padding; fp16 with a scaled loss.
        {"name": "loss 333x50257x1153 fp16 train", "op": "loss", "tokens": 333, "vocab": 50257, "in": 1153,
         "dtype": "fp16", "train": True, "reduction": "mean", "masked": 0.1},
        # One sequence through the d=1152 model's head.
        {"name": "loss 1024x50688x1152 bf16 train", "op": "loss", "tokens": 1024, "vocab": 50688, "in": 1152,
         "dtype": "bf16", "train": True, "reduction": "mean", "masked": 0.0},
        # Answers learnt after their questions: half of the tokens have no loss, each other one its own weight.
        {"name": "loss 4096x50688x1920 bf16 train", "op": "loss", "tokens": 4096, "vocab": 50688, "in": 1920,
         "dtype": "bf16", "train": True, "reduction": "none", "masked": 0.5},
        # A training step's micro-batch of eight sequences through the d=1920 model's head: arithmetic.
        {"name": "loss 8192x50688x1920 bf16 train", "op": "loss", "tokens": 8192, "vocab": 50688, "in": 1920,
         "dtype": "bf16", "train": True, "reduction": "mean", "masked": 0.0},
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], even over the logarithm."""
    return max(lo, min(hi, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    if rng.random() < 0.5:
        cols = _spread(rng, 24, 8192)
        if rng.random() < 0.6:
            cols = -(-cols // 24) * 24
        tokens = min(_spread(rng, 1, 16384), 8192 * 7680 // cols)
        return {"op": "norm", "kind": rng.choice(["rms", "layer"]), "tokens": max(1, tokens), "cols": cols,
                "dtype": rng.choice(["fp32", "fp16", "bf16"]), "residual": rng.random() < 0.7,
                "train": rng.random() < 0.7}
    vocab, k = _spread(rng, 200, 131072), _spread(rng, 24, 7680)
    if rng.random() < 0.75:
        k = -(-k // 24) * 24
    train = rng.random() < 0.6
    tokens = min(_spread(rng, 1, 8192), 8192 * 50688 * 1920 // (vocab * k), 8192 * 50688 // vocab)
    return {"op": "loss", "tokens": max(1, tokens), "vocab": vocab, "in": k, "dtype": rng.choice(["fp16", "bf16"]),
            "train": train, "reduction": rng.choice(["mean", "sum", "none"]) if train else "none",
            "masked": rng.choice([0.0, 0.1, 0.5])}


def _kept(case):
    """Tokens that have a loss: never none."""
    return max(1, case["tokens"] - int(case["masked"] * case["tokens"]))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dev, dt = "cuda", DTYPES[case["dtype"]]
    if case["op"] == "norm":
        t, c = case["tokens"], case["cols"]
        # A residual stream with a few channels much larger than the rest.
        channel = torch.where(torch.rand(c, generator=g, device=dev) < 0.005, 12.0, 1.0)
        s = {"case": case, "bias": None, "residual": None}
        s["x"] = (torch.randn(t, c, generator=g, device=dev) * 0.7).to(dt)
        if case["residual"]:
            s["residual"] = (torch.randn(t, c, generator=g, device=dev) * 2.0 * channel).to(dt)
        s["weight"] = (1.0 + 0.2 * torch.randn(c, generator=g, device=dev)).to(dt)
        if case["kind"] == "layer":
            s["bias"] = (0.1 * torch.randn(c, generator=g, device=dev)).to(dt)
        if case["train"]:
            s["dy"] = torch.randn(t, c, generator=g, device=dev).to(dt)
            if case["residual"]:
                s["dsummed"] = torch.randn(t, c, generator=g, device=dev).to(dt)
            for name in ("x", "residual", "weight", "bias"):
                if s[name] is not None:
                    s[name].requires_grad_(True)
        return s
    t, v, k = case["tokens"], case["vocab"], case["in"]
    # Normed states and a head whose logits spread by 2.2; six tokens of ten lean to their target.
    w = torch.randn(v, k, generator=g, device=dev) * (2.2 / k ** 0.5)
    target = torch.randint(0, v, (t,), generator=g, device=dev)
    lean = torch.where(torch.rand(t, generator=g, device=dev) < 0.6, 1.6, 0.0)
    x = torch.randn(t, k, generator=g, device=dev) + lean[:, None] * w[target]
    out = torch.randperm(t, generator=g, device=dev)[: t - _kept(case)]
    target[out] = IGNORE
    s = {"case": case, "x": x.to(dt), "weight": w.to(dt), "target": target, "dloss": None}
    if case["train"]:
        s["x"].requires_grad_(True)
        s["weight"].requires_grad_(True)
        if case["reduction"] == "none":
            s["dloss"] = torch.rand(t, generator=g, device=dev) / t
        elif case["reduction"] == "mean" and case["dtype"] == "fp16":
            s["dloss"] = torch.tensor(4096.0, device=dev)  # the loss's scale
    return s


def run(state):
    if state["case"]["op"] == "norm":
        return _norm_own(state) if own else _norm_plain(state)
    return _loss_own(state) if own else _loss_plain(state)


def _norm_own(s):
    from pollux_b200 import norm
    case = s["case"]
    if case["kind"] == "rms":
        y, summed = norm.add_rms_norm(s["x"], s["weight"], residual=s["residual"], eps=EPS["rms"])
    else:
        y, summed = norm.add_layer_norm(s["x"], s["weight"], s["bias"], residual=s["residual"], eps=EPS["layer"])
    out = {"y": y} if summed is None else {"y": y, "summed": summed}
    if case["train"]:
        leaves = {n: s[n] for n in ("x", "residual", "weight", "bias") if s[n] is not None}
        grads = torch.autograd.grad(list(out.values()), list(leaves.values()),
                                    [s["dy"]] if summed is None else [s["dy"], s["dsummed"]])
        out = {n: t.detach() for n, t in out.items()}
        out.update({"d" + n: d for n, d in zip(leaves, grads)})
    return out


@torch.no_grad()
def _norm_plain(s):
    case = s["case"]
    dt = DTYPES[case["dtype"]]
    x, w = s["x"].float(), s["weight"].float()
    # The norm is taken of the residual stream as it is handed on, in x's type.
    h = x if s["residual"] is None else (x + s["residual"].float()).to(dt).float()
    c = h if case["kind"] == "rms" else h - h.mean(dim=1, keepdim=True)
    inv = 1.0 / torch.sqrt((c * c).mean(dim=1, keepdim=True) + EPS[case["kind"]])
    n = c * inv
    y = n * w
    if s["bias"] is not None:
        y = y + s["bias"].float()
    out = {"y": y.to(dt)}
    if s["residual"] is not None:
        out["summed"] = h.to(dt)
    if case["train"]:
        dy = s["dy"].float()
        v = dy * w
        d = v - n * (v * n).mean(dim=1, keepdim=True)
        if case["kind"] == "layer":
            d = d - v.mean(dim=1, keepdim=True)
        d = d * inv
        if s["residual"] is not None:
            d = d + s["dsummed"].float()
        out["dx"] = d.to(dt)
        if s["residual"] is not None:
            out["dresidual"] = out["dx"]
        out["dweight"] = (dy * n).sum(dim=0).to(dt)
        if s["bias"] is not None:
            out["dbias"] = dy.sum(dim=0).to(dt)
    return out


def _loss_own(s):
    from pollux_b200 import loss
    case = s["case"]
    value = loss.linear_cross_entropy(s["x"], s["weight"], s["target"], ignore_index=IGNORE,
                                      reduction=case["reduction"])
    if not case["train"]:
        return {"loss": value}
    dx, dw = torch.autograd.grad(value, (s["x"], s["weight"]), s["dloss"])
    return {"loss": value.detach(), "dx": dx, "dweight": dw}


@torch.no_grad()
def _loss_plain(s):
    case = s["case"]
    dt = DTYPES[case["dtype"]]
    rows = torch.nonzero(s["target"] != IGNORE).squeeze(1)
    at = s["target"][rows].unsqueeze(1)
    x, w = s["x"][rows].float(), s["weight"].float()
    z = torch.matmul(x, w.t())
    top = z.amax(dim=1, keepdim=True)
    lse = top + torch.log(torch.exp(z - top).sum(dim=1, keepdim=True))
    each = torch.zeros(case["tokens"], device=x.device)
    each[rows] = (lse - z.gather(1, at)).squeeze(1)
    n = rows.numel()
    value = {"none": each, "sum": each.sum(), "mean": each.sum() / n}[case["reduction"]]
    if not case["train"]:
        return {"loss": value}
    if case["reduction"] == "none":
        g = s["dloss"][rows].unsqueeze(1)
    else:
        g = torch.ones((), device=x.device) if s["dloss"] is None else s["dloss"]
        if case["reduction"] == "mean":
            g = g / n
    d = torch.exp(z - lse)
    d.scatter_add_(1, at, torch.full_like(at, -1.0, dtype=torch.float32))
    d *= g
    dx = torch.zeros(case["tokens"], case["in"], device=x.device)
    dx[rows] = torch.matmul(d, w)
    return {"loss": value, "dx": dx.to(dt), "dweight": torch.matmul(d.t(), x).to(dt)}


def work(case):
    s = SIZE[case["dtype"]]
    if case["op"] == "norm":
        t, c = case["tokens"], case["cols"]
        # x and y, with a residual that and the sum; back: dy and dx, with a residual the sum's gradient.
        planes = 4 if case["residual"] else 2
        if case["train"]:
            planes += 3 if case["residual"] else 2
        params = 1 if case["kind"] == "rms" else 2
        return {"bytes": s * (planes * t * c + params * c * (2 if case["train"] else 1)),
                "flops": t * c * (20 if case["train"] else 8)}
    t, v, k, n = case["tokens"], case["vocab"], case["in"], _kept(case)
    loss = 4 * t if case["reduction"] == "none" else 4
    if not case["train"]:
        return {"bytes": s * (n * k + v * k) + 8 * t + loss, "flops": 2 * n * v * k}
    # Back: the gradients of all states and of the head; the logits' product and one for each gradient.
    return {"bytes": s * (n * k + t * k + 2 * v * k) + 8 * t + 2 * loss, "flops": 6 * n * v * k}


def exact(case, seed):
    """The definitions in 64 bits."""
    s = prepare(case, seed)
    with torch.no_grad():
        return _norm_exact(case, s) if case["op"] == "norm" else _loss_exact(case, s)


def _norm_exact(case, s):
    h = s["x"].double()
    if s["residual"] is not None:
        # (The sum of two values of a 16-bit type, or of fp32, is rounded once to that type.)
        h = (h + s["residual"].double()).to(DTYPES[case["dtype"]]).double()
    w = s["weight"].double()
    size = case["cols"]
    mu = h.sum(1, keepdim=True) / size if case["kind"] == "layer" else torch.zeros_like(h[:, :1])
    sigma = torch.sqrt(((h - mu) ** 2).sum(1, keepdim=True) / size + EPS[case["kind"]])
    unit = (h - mu) / sigma
    out = {"y": unit * w + (0.0 if s["bias"] is None else s["bias"].double())}
    if s["residual"] is not None:
        out["summed"] = h
    if case["train"]:
        dy = s["dy"].double()
        dn = dy * w
        along = (dn * unit).sum(1, keepdim=True) / size
        flat = dn.sum(1, keepdim=True) / size if case["kind"] == "layer" else 0.0
        dh = (dn - flat - unit * along) / sigma
        if s["residual"] is not None:
            dh = dh + s["dsummed"].double()
        out["dx"] = dh
        if s["residual"] is not None:
            out["dresidual"] = dh
        out["dweight"] = torch.einsum("tc,tc->c", dy, unit)
        if s["bias"] is not None:
            out["dbias"] = dy.sum(0)
    return out


def _loss_exact(case, s):
    target, w = s["target"], s["weight"].double()
    t, v, k = case["tokens"], case["vocab"], case["in"]
    kept = target != IGNORE
    n = int(kept.sum())
    each = torch.zeros(t, dtype=torch.float64, device=w.device)
    weights = kept.double()  # what a token's loss adds to the value that is differentiated
    if case["train"]:
        if case["reduction"] == "none":
            weights = weights * s["dloss"].double()
        else:
            weights = weights * (1.0 if s["dloss"] is None else float(s["dloss"]))
            if case["reduction"] == "mean":
                weights = weights / n
        dx = torch.zeros(t, k, dtype=torch.float64, device=w.device)
        dw = torch.zeros(v, k, dtype=torch.float64, device=w.device)
    step = max(1, (1 << 27) // v)  # rows at once, 1 GB of logits
    for a in range(0, t, step):
        rows = slice(a, min(t, a + step))
        x = s["x"][rows].double()
        z = torch.einsum("tk,vk->tv", x, w)
        lse = torch.logsumexp(z, dim=1)
        at = target[rows].clamp_min(0)
        own_z = z[torch.arange(at.numel(), device=z.device), at]
        each[rows] = torch.where(kept[rows], lse - own_z, 0.0)
        if case["train"]:
            z = torch.softmax(z, dim=1)
            z[torch.arange(at.numel(), device=z.device), at] -= 1.0
            z *= weights[rows, None]
            dx[rows] = torch.einsum("tv,vk->tk", z, w)
            dw += torch.einsum("tv,tk->vk", z, x)
    value = {"none": each, "sum": each.sum(), "mean": each.sum() / n}[case["reduction"]]
    return {"loss": value, "dx": dx, "dweight": dw} if case["train"] else {"loss": value}
