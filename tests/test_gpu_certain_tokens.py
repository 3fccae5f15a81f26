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
