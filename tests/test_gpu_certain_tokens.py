"""Losses of tokens that are nearly certain (loss.linear_cross_entropy): never below 0, and right to the roundings of a
sum of exponentials, however large the logits.

States and head hold whole sixteenths, and every logit is below 2^11, so products and their sums are exact in fp32 and in
a tensor core in whatever order, and only what follows them is seen.

Bounds, u = 2^-24.  Of s = sum exp(z - max): the largest term is 1 exactly; a chain has at most 32 additions in a tile, 4
of its parts, 8 + 3 + 7 joins of two roundings each, 100 u of s in all; each other term is off by 2^-22 of ex2 and
2 u (log2 e) |z - max| of its exponent, below 2^-20 of itself while |z - max| e^-|z - max| is below 1.  log adds 2 u, its
sum with max - z_target one more rounding: |loss - got| <= 100 u + 2^-20 min(1, s - 1) + 4 u loss."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DTYPES = [torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def ce(lib):
    from pollux_b200 import loss
    return loss.linear_cross_entropy


def _certain(tokens, vocab, top, dtype, k=64, kinds=32):
    """Token t has the logit `top` at one place, elsewhere sixteenths between -8 and 8."""
    g = torch.Generator(device="cuda").manual_seed(vocab + tokens)
    w = torch.randint(-16, 17, (vocab, k), generator=g, device="cuda") / 16
    x = torch.randint(0, 2, (tokens, k), generator=g, device="cuda").float()
    x[:, kinds + 8:] = 0
    places = torch.arange(kinds, device="cuda") * (vocab // kinds) + 3
    w[:, :kinds] = 0
    w[places] = 0
    w[places, torch.arange(kinds, device="cuda")] = 1
    x[:, :kinds] = 0
    which = torch.arange(tokens, device="cuda") % kinds
    x[torch.arange(tokens, device="cuda"), which] = float(top)
    x, w = x.to(dtype), w.to(dtype)
    z = x.double() @ w.double().t()
    assert float(z.abs().max()) < 2 ** 11 and float(z.max()) == top
    return x, w, places[which], z


@pytest.mark.parametrize("top", [12, 20, 30, 100, 1000])
@pytest.mark.parametrize("tokens,vocab", [(1, 1009), (20, 50688), (128, 12672), (129, 12672), (700, 50257)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_certain_tokens(ce, tokens, vocab, top, dtype):
    x, w, right, z = _certain(tokens, vocab, top, dtype)
    s = torch.exp(z - z.amax(1, keepdim=True)).sum(1)
    wrong = (right + 1) % vocab
    for target in (right, wrong):
        want = torch.log(s) + (z.amax(1) - z.gather(1, target[:, None])[:, 0])
        bound = 100 * U + 2.0 ** -20 * (s - 1).clamp(max=1) + 4 * U * want
        got = ce(x, w, target, reduction="none")
        assert bool((got >= 0).all()), float(got.min())
        assert bool(((got.double() - want).abs() <= bound).all()), float(((got.double() - want).abs() / bound).max())
        # Each token's error once, and the last rounding.
        for reduction, n in (("sum", 1), ("mean", tokens)):
            value = ce(x, w, target, reduction=reduction)
            assert float(value) >= 0
            assert abs(float(value) - float(want.sum()) / n) <= float(bound.sum()) / n + U * float(want.sum()) / n


# Gradients.  Where k is long, the forward pass's z may be off by ez and the backward pass's by eb: d of another token v is
# p (1 + ez + eb), rounded to 16 bits; the target's is -(1 - e^-loss), whose error is that of the loss.
def _long(tokens, vocab, k, dtype, top, seed=0):
    """Near-certain tokens whose logit is a sum of one sign over all of k."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    kinds = min(tokens, 32)
    places = torch.arange(kinds, device="cuda") * (vocab // kinds) + 3
    sign = torch.where(torch.rand(kinds, k, generator=g, device="cuda") < 0.5, -1.0, 1.0)
    w = torch.randn(vocab, k, generator=g, device="cuda") * (0.3 / k ** 0.5)
    size = (0.5 + torch.rand(kinds, k, generator=g, device="cuda")) * (top / k) ** 0.5
    w[places] = sign * size
    which = torch.arange(tokens, device="cuda") % kinds
    x = (sign * size)[which] * (0.8 + 0.25 * torch.rand(tokens, 1, generator=g, device="cuda"))
    return x.to(dtype), w.to(dtype), places[which]


@pytest.mark.parametrize("tokens,vocab,k,top", [(20, 5003, 7680, 18), (200, 5003, 7680, 18), (200, 9001, 1920, 22),
                                                (64, 9001, 1153, 16), (300, 1009, 4097, 14), (40, 1009, 12000, 14)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_gradients_of_certain_tokens(ce, tokens, vocab, k, top, dtype):
    """The target's entry of d is right relative to 1 - p, and the others to p."""
    x, w, target = _long(tokens, vocab, k, dtype, top)
    half, tiny = torch.finfo(dtype).eps / 2, (2.0 ** -134 if dtype == torch.bfloat16 else 2.0 ** -25)
    z = x.double() @ w.double().t()
    lse = torch.logsumexp(z, 1)
    rest = z.scatter(1, target[:, None], float("-inf"))
    loss = torch.nn.functional.softplus(torch.logsumexp(rest, 1) - z.gather(1, target[:, None])[:, 0])
    assert 1e-7 < float(loss.min()) and float(loss.max()) < 0.5
    # Truncated sums: 2^-23 of the sum of magnitudes for each 16 k of a slice (1,024 k, in fp16 512), and its additions.
    mags = x.double().abs() @ w.double().abs().t()
    ez = ((1024 / 16 + k / 512 + 8) * 2.0 ** -23 * mags.amax(1))
    # ... and of what the backward pass sums at once (4,096 and 1,408).
    eb = ((min(k, 4096) / 16 + k / 1408 + 8) * 2.0 ** -23 * mags.amax(1))
    eloss = (1 - torch.exp(-loss)) * (torch.expm1(2 * ez) + 2.0 ** -18) + 100 * U
    xs, ws = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    scale = 256.0
    value = ce(xs, ws, target, reduction="none")
    assert bool(((value.detach().double() - loss).abs() <= eloss).all())
    dx, dw = torch.autograd.grad(value, (xs, ws), torch.full((tokens,), scale, device="cuda"))
    own = torch.expm1(-loss)
    ed_own = own.abs() * half + eloss * (1 + half)
    p = torch.exp(rest - lse[:, None])
    ed = (p * (half + torch.expm1(ez + eb) + 2.0 ** -18)[:, None] + 2.0 ** -40).scatter(1, target[:, None], ed_own[:, None])
    d = p.scatter(1, target[:, None], own[:, None])
    for got, want, err in ((dx, d @ w.double(), ed @ w.double().abs() + (vocab / 16 + 16) * 2.0 ** -23 * (d.abs() @ w.double().abs())),
                           (dw, d.t() @ x.double(), ed.t() @ x.double().abs() + (tokens / 16 + 16) * 2.0 ** -23 * (d.abs().t() @ x.double().abs()))):
        want, err = scale * want, scale * err
        err = err + half * (want.abs() + err) + tiny
        assert bool(((got.double() - want).abs() <= err).all()), float(((got.double() - want).abs() / err).max())


@pytest.mark.parametrize("top", [30, 100, 1000])
@pytest.mark.parametrize("tokens", [33, 300])
@pytest.mark.parametrize("dtype", DTYPES)
def test_entry_of_d_at_the_target(ce, tokens, top, dtype):
    """Exact logits, one other token 9 below the largest: 1 - p = 1.2e-4.  One state is there in one token alone, so that
    an element of the target's row of dW is that token's d times powers of two: half a step of d, half a step of dW, and
    100 u of the loss's sum."""
    k, vocab = 64, 515
    x = torch.zeros(tokens, k, device="cuda")
    w = torch.zeros(vocab, k, device="cuda")
    t = torch.arange(tokens, device="cuda")
    x[:, 0] = float(top)
    x[:, 1] = 1
    x[:, 2] = (t == 5).float() * 0.5  # one token alone
    w[7, 0], w[9, 0], w[9, 1] = 1, 1, -9
    target = torch.full((tokens,), 7, device="cuda")
    z = torch.zeros(tokens, vocab, dtype=torch.float64, device="cuda")
    z[:, 7], z[:, 9] = top, top - 9
    loss = torch.log1p(torch.exp(z.scatter(1, target[:, None], float("-inf")) - top).sum(1))
    xs, ws = x.to(dtype).requires_grad_(True), w.to(dtype).requires_grad_(True)
    value = ce(xs, ws, target, reduction="none")
    dx, dw = torch.autograd.grad(value, (xs, ws), torch.full((tokens,), 1024.0, device="cuda"))
    half = torch.finfo(dtype).eps / 2
    assert bool(((value.detach().double() - loss).abs() <= 100 * U).all())
    want = 1024.0 * 0.5 * torch.expm1(-loss[5])
    bound = abs(float(want)) * 2.01 * half + 1024 * 0.5 * 100 * U
    assert abs(float(dw[7, 2]) - float(want)) <= bound, (float(dw[7, 2]), float(want))


@pytest.mark.parametrize("tokens", [20, 200])
@pytest.mark.parametrize("factor", [1.9989, -1.9985, 1.0, 0.99951, 3.9978])
@pytest.mark.parametrize("dtype", DTYPES)
def test_a_certain_wrong_token(ce, tokens, factor, dtype):
    """All logits far below 0 and one of them certain: its sum loses magnitude in the tensor cores, so p comes out above 1,
    and times a factor just below 2 it stays finite.  dx = g (W[7] - W[target]) up to e^-140: half a step of each entry of
    d, with what z[7] was cut off in p (an addition in a tensor core may truncate, by up to 2^-23 of the sum: that for each
    16 k, of |z[7]| since all products have one sign), and half a step of the result."""
    k, vocab = 1400, 300
    g = torch.Generator(device="cuda").manual_seed(5)
    size = (0.5 + torch.rand(k, generator=g, device="cuda")) * (150.0 / k) ** 0.5
    w = -2 * size.expand(vocab, k) * (1 + 0.01 * torch.rand(vocab, k, generator=g, device="cuda"))
    w[7] = -size
    x = size.expand(tokens, k) * (0.95 + 0.05 * torch.rand(tokens, 1, generator=g, device="cuda"))
    target = torch.arange(tokens, device="cuda") % 5 + 20
    xs, ws = x.to(dtype).requires_grad_(True), w.to(dtype).requires_grad_(True)
    value = ce(xs, ws, target, reduction="none")
    z = xs.detach().double() @ ws.detach().double().t()
    assert bool(((value.detach().double() - (z[:, 7] - z.gather(1, target[:, None])[:, 0])).abs() <= 1e-2).all())
    dx, dw = torch.autograd.grad(value, (xs, ws), torch.full((tokens,), factor, device="cuda"))
    half = torch.finfo(dtype).eps / 2
    wd = ws.detach().double()
    want = factor * (wd[7] - wd[target])
    cut = torch.expm1(z[:, 7:8].abs() * (k / 16 + 8) * 2.0 ** -23)
    err = abs(factor) * (wd[7].abs() * (half + cut + 2.0 ** -18) + wd[target].abs() * half)
    err = err + half * (want.abs() + err) + 2.0 ** -25
    assert bool(((dx.double() - want).abs() <= err).all())
    assert bool(torch.isfinite(dw).all())
