"""Gradients of tokens whose factors lie far apart (loss.linear_cross_entropy, reduction "none").

Bounds, h half a step of the operands' type relative to the value, u = 2^-23.  An element of dW is sum_t g d x: each d is
off by h |d| (its rounding with the factor's part), 2^-18 p of the exponentials and 2^-40 (fp16's smallest steps of d times
2^15); each scaled state in fp16 by half a smallest step where the largest |g x| lies at 2^14 or above, 2^-39 of that; and
the result by half a step and half the type's smallest."""
from __future__ import annotations

import pytest
import torch

from test_gpu_linear_ce import _check, _inputs

pytestmark = pytest.mark.gpu
U = 2.0 ** -23


@pytest.fixture(scope="module")
def ce(lib):
    from pollux_b200 import loss
    return loss.linear_cross_entropy


@pytest.mark.parametrize("powers", [(14, -2), (14, -6), (14, -10), (14, -12), (10, -16), (-3, -30), (0, -24)])
@pytest.mark.parametrize("tokens", [40, 300])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_rows_that_one_small_factor_feeds(ce, tokens, powers, dtype):
    """Half of the tokens, with large factors, are nearly sure of their targets; the others' targets are rows of the head
    that nothing else reaches (logits 40 below)."""
    k, vocab = 72, 700
    g = torch.Generator(device="cuda").manual_seed(tokens)
    x = torch.randn(tokens, k, generator=g, device="cuda")
    w = torch.randn(vocab, k, generator=g, device="cuda") * 0.05
    small = torch.arange(tokens, device="cuda") % 2 == 1
    x[:, 0], x[:, 1] = (~small) * 8.0, small * 8.0
    w[:, 0] = w[:, 1] = 0
    rows = torch.arange(tokens, device="cuda") + 50
    w[rows[small], 0] = -5  # out of the others' reach
    target = torch.where(small, rows, 3)
    w[3, 0], w[3, 1] = 1.7, -5
    x, w = x.to(dtype), w.to(dtype)
    f = 2.0 ** torch.where(small, powers[1], powers[0]).float() * (1 + torch.rand(tokens, generator=g, device="cuda"))
    f = f * torch.where(torch.rand(tokens, generator=g, device="cuda") < 0.5, -1.0, 1.0)
    f[4], f[5] = 0.0, 0.0
    xs, ws = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    dx, dw = torch.autograd.grad(ce(xs, ws, target, reduction="none"), (xs, ws), f)
    xd, wd, fd = x.double(), w.double(), f.double()[:, None]
    p = torch.softmax(xd @ wd.t(), 1)
    d = p.scatter_add(1, target[:, None], torch.full((tokens, 1), -1.0, dtype=torch.float64, device="cuda"))
    half, tiny = torch.finfo(dtype).eps / 2, (2.0 ** -134 if dtype == torch.bfloat16 else 2.0 ** -25)
    ed = half * d.abs() + 2.0 ** -18 * p + 2.0 ** -40
    gx = (fd * xd).abs()
    step = 2.0 ** -39 * float(gx.max()) if dtype == torch.float16 else 0.0
    for got, want, err in ((dw, d.t() @ (fd * xd), ed.t() @ gx + (tokens / 16 + 16) * U * (d.abs().t() @ gx)
                            + step * d.abs().sum(0)[:, None]),
                           (dx, fd * (d @ wd), fd.abs() * (ed @ wd.abs() + (vocab / 16 + 16) * U * (d.abs() @ wd.abs())))):
        err = err + half * (want.abs() + err) + tiny
        assert bool(((got.double() - want).abs() <= err).all()), float(((got.double() - want).abs() / err).max())
    # (They are there, but token 5's: not below what the type holds.)
    if powers[1] >= -12:
        assert bool((dw[rows[small][3:]].abs().amax(1) > 2.0 ** -14).all())


@pytest.mark.parametrize("tokens,vocab,k", [(16385, 33, 40), (40001, 70, 113), (300, 500, 1153), (9, 40, 7)])
def test_many_tokens_in_fp16(ce, tokens, vocab, k):
    """Sizes of states and factors by blocks of tokens; the largest product is the last kept token's."""
    x, w, target = _inputs(tokens, vocab, k, torch.float16, seed=29, masked=0.3)
    target[-1] = 1
    dloss = torch.rand(tokens, device="cuda") * 0.02
    dloss[-1] = -3.0
    _check(ce, x, w, target, "none", dloss)


@pytest.mark.parametrize("tokens", [50, 500])
def test_sizes_at_the_ends_of_the_types(ce, tokens):
    """Products from far below fp32's smallest to near its largest set the scale; ignored rows and zeros do not."""
    x, w, target = _inputs(tokens, 90, 48, torch.float16, seed=31)
    target[::5] = -100
    x[0], x[5] = float("inf"), 60000.0
    for f in (2.0 ** -140, 2.0 ** -100, 2.0 ** -40, 2.0 ** 10, 2.0 ** 126):
        dloss = torch.full((tokens,), f, device="cuda")
        dloss[0], dloss[5], dloss[10] = float("inf"), float("nan"), 2.0 ** 127
        dloss[1] = 0.0
        xs, ws = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        dx, dw = torch.autograd.grad(ce(xs, ws, target, reduction="none"), (xs, ws), dloss)
        ones = torch.ones(tokens, device="cuda")
        ones[1] = 0.0
        bx, bw = torch.autograd.grad(ce(xs, ws, target, reduction="none"), (xs, ws), ones)
        if f == 2.0 ** 10:  # powers of two: the same digits where neither end cuts them
            for a, b in ((dx, bx), (dw, bw)):
                far = (b.abs() > 2.0 ** -13) & (b.abs() < 60)
                assert torch.equal(a[far], (b[far].double() * f).half())
        elif f <= 2.0 ** -40:
            assert not bool(dx.any()) and not bool(dw.any())
        else:
            assert not bool(dx.isnan().any()) and not bool(dw.isnan().any())
            assert bool((dw[bw.abs() > 2.0 ** -13].isinf()).all())


@pytest.mark.parametrize("tokens", [40, 300])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_a_state_of_zeros_with_a_large_factor(ce, tokens, dtype):
    """It adds nothing to dW, however far its factor lies above the others'."""
    x, w, target = _inputs(tokens, 90, 48, dtype, seed=47)
    x[3] = 0
    dloss = torch.full((tokens,), 2.0 ** -70, device="cuda")
    dloss[3] = 2.0 ** 120
    xs, ws = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    dw = torch.autograd.grad(ce(xs, ws, target, reduction="none"), ws, dloss)[0]
    assert bool(torch.isfinite(dw).all())
    if dtype == torch.float16:
        assert not bool(dw.any())
