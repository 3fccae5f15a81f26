"""Cross entropy of a head's product (loss.linear_cross_entropy) against its formula in 64 bits.

Bounds.  h is half a step of the operands' type relative to the value (eps / 2: 2^-8 in bf16, 2^-11 in fp16), u = 2^-23 (a tensor core may truncate where it adds).
  z       products are exact; sums run over in/16 groups of 16: |dz| <= ez = (in/16 + 16) u max sum|x w|
  loss    log-sum-exp and logit carry ez each, exponentials and their sum 2^-20, the last roundings
          of lse, logit and loss 4 * 2^-24 of the largest magnitude
  d       |dd| <= h |d| + p (2 ez + 2^-20) + 2^-40 (fp16 holds d in steps of 2^-24 * 2^-15)
  dx, dW  the sum of |dd| times the other factor's magnitude, (length/16 + 16) u of the sum of magnitudes
          for the additions, h of the value at the end and half the type's smallest step;
          a token's own factor is exact in dW, but where it takes a state below the type's range: half a smallest
          step of the largest factor."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -23
HALF = {t: torch.finfo(t).eps / 2 for t in (torch.bfloat16, torch.float16)}  # 8 bits: 2^-8; 11 bits: 2^-11
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}
DTYPES = [torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def ce(lib):
    from pollux_b200 import loss
    return loss.linear_cross_entropy


def _inputs(tokens, vocab, k, dtype, seed=0, masked=0.0, lean=0.6):
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + tokens * 31 + vocab * 17 + k)
    w = torch.randn(vocab, k, generator=g, device="cuda") * (2.2 / k ** 0.5)
    target = torch.randint(0, vocab, (tokens,), generator=g, device="cuda")
    on = (torch.rand(tokens, generator=g, device="cuda") < lean).float()
    x = torch.randn(tokens, k, generator=g, device="cuda") + 1.6 * on[:, None] * w[target]
    if masked:
        target[torch.rand(tokens, generator=g, device="cuda") < masked] = -100
    return x.to(dtype), w.to(dtype), target


def _reference(x, w, target, factor):
    """loss of each token and the gradients of sum(factor * loss), with their bounds.  (In steps of rows.)"""
    dtype, half = x.dtype, HALF[x.dtype]
    x, w = x.double(), w.double()
    t, k = x.shape
    v = w.shape[0]
    keep = target != -100
    loss = torch.zeros(t, dtype=torch.float64, device=x.device)
    eloss = torch.zeros_like(loss)
    dx, edx = torch.zeros_like(x), torch.zeros_like(x)
    dw, edw, mag = torch.zeros_like(w), torch.zeros_like(w), torch.zeros_like(w)
    top = factor[keep].abs().max() if bool(keep.any()) else factor.new_zeros(())
    step = max(1, (1 << 25) // v)
    for a in range(0, t, step):
        r = torch.arange(a, min(t, a + step), device=x.device)
        r = r[keep[r]]
        if r.numel() == 0:
            continue
        z = x[r] @ w.t()
        ez = (k / 16 + 16) * U * (x[r].abs() @ w.abs().t()).amax(1)
        lse = torch.logsumexp(z, 1)
        zt = z.gather(1, target[r][:, None])[:, 0]
        loss[r] = lse - zt
        eloss[r] = 2 * ez + 2.0 ** -20 + 4 * 2.0 ** -24 * torch.maximum(lse.abs(), zt.abs())
        p = torch.exp(z - lse[:, None])
        d = p.scatter_add(1, target[r][:, None], torch.full_like(zt, -1.0)[:, None])
        ed = half * d.abs() + p * (2 * ez + 2.0 ** -20)[:, None] + 2.0 ** -40
        f = factor[r][:, None]
        dx[r] = f * (d @ w)
        edx[r] = f.abs() * (ed @ w.abs() + (v / 16 + 16) * U * (d.abs() @ w.abs()))
        dw += d.t() @ (f * x[r])
        edw += ed.t() @ (f * x[r]).abs()
        mag += d.abs().t() @ (f * x[r]).abs()
        edw += d.abs().t() @ torch.full_like(x[r], float(top) * TINY[dtype])
    edw += (t / 16 + 16) * U * mag
    edx += half * (dx.abs() + edx) + TINY[dtype]
    edw += half * (dw.abs() + edw) + TINY[dtype]
    return loss, eloss, dx, edx, dw, edw


def _close(got, want, bound, what):
    bad = ~((got.double() - want).abs() <= bound)
    assert not bool(bad.any()), (what, int(bad.sum()), float((got.double() - want).abs().max()), float(bound.max()))


def _factor(target, reduction, scale=1.0):
    keep = target != -100
    n = int(keep.sum())
    return torch.full(target.shape, scale / (n if reduction == "mean" and n else 1), dtype=torch.float64,
                      device=target.device)


def _check(ce, x, w, target, reduction, dloss=None):
    xs, ws = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    value = ce(xs, ws, target, reduction=reduction)
    assert value.dtype == torch.float32
    dx, dw = torch.autograd.grad(value, (xs, ws), dloss)
    assert dx.dtype == x.dtype and dw.dtype == w.dtype and dx.shape == x.shape and dw.shape == w.shape
    factor = dloss.double() if reduction == "none" else _factor(target, reduction, 1.0 if dloss is None else float(dloss))
    loss, eloss, rdx, edx, rdw, edw = _reference(x, w, target, factor)
    n = max(1, int((target != -100).sum()))
    if reduction == "none":
        _close(value, loss, eloss, "loss")
    elif reduction == "sum":
        _close(value, loss.sum(), eloss.sum() + 2.0 ** -23 * loss.sum().abs(), "loss")
    else:
        _close(value, loss.sum() / n, eloss.sum() / n + 2.0 ** -23 * loss.sum().abs() / n, "loss")
    _close(dx, rdx, edx, "dx")
    _close(dw, rdw, edw, "dw")
    assert bool((dx[target == -100] == 0).all())
    with torch.no_grad():
        assert torch.equal(ce(x, w, target, reduction=reduction), value.detach())


SIZES = [(1, 1, 1), (1, 2, 8), (3, 200, 24), (9, 1009, 240), (33, 257, 1153), (130, 300, 65), (257, 1000, 96),
         (64, 64, 64), (65, 511, 7), (520, 131, 1920), (300, 50257, 40), (1, 50688, 128), (256, 256, 256)]


@pytest.mark.parametrize("tokens,vocab,k", SIZES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_loss_and_gradients(ce, tokens, vocab, k, dtype):
    x, w, target = _inputs(tokens, vocab, k, dtype)
    _check(ce, x, w, target, "mean", torch.tensor(64.0, device="cuda"))


@pytest.mark.parametrize("reduction", ["sum", "none", "mean"])
@pytest.mark.parametrize("masked", [0.1, 0.6])
@pytest.mark.parametrize("dtype", DTYPES)
def test_masks_and_reductions(ce, reduction, masked, dtype):
    for tokens, vocab, k in ((70, 515, 120), (700, 300, 33), (1500, 77, 200)):
        x, w, target = _inputs(tokens, vocab, k, dtype, seed=3, masked=masked)
        dloss = torch.rand(tokens, device="cuda") if reduction == "none" else None
        _check(ce, x, w, target, reduction, dloss)


@pytest.mark.parametrize("tokens,vocab,k", [(16385, 33, 40), (200001, 17, 24)])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_many_tokens(ce, reduction, tokens, vocab, k):
    """Tokens counted by blocks; the largest factor is the last kept token's."""
    x, w, target = _inputs(tokens, vocab, k, torch.bfloat16, seed=23, masked=0.3)
    target[-1] = 1
    dloss = None
    if reduction == "none":
        dloss = torch.rand(tokens, device="cuda")
        dloss[-1] = -37.0
    _check(ce, x, w, target, reduction, dloss)


@pytest.mark.parametrize("tokens", [40, 300])
@pytest.mark.parametrize("dtype", DTYPES)
def test_factors_of_all_sizes(ce, tokens, dtype):
    """A gradient for each token: zeros, signs, 1e-30 to 1e6, parts around 1.999; and one that is no number."""
    x, w, target = _inputs(tokens, 700, 72, dtype, seed=13, masked=0.2)
    x[1] *= 40.0  # (d of nearly one in magnitude)
    target[1] = 5
    g = torch.Generator().manual_seed(17)
    # fp16's results end at 65,504.
    most = 6.0 if dtype == torch.bfloat16 else 0.0
    dloss = 10.0 ** (torch.rand(tokens, generator=g) * (6.0 + most) - 6.0)
    dloss = dloss * torch.where(torch.rand(tokens, generator=g) < 0.5, -1.0, 1.0)
    dloss[::7] = 0.0
    dloss[1], dloss[2], dloss[3], dloss[4] = 1.99951, -1.9989, 0.99976, 1e-30
    dloss[5] = 1e-38
    dloss = dloss.cuda()
    target[2:7] = 9
    _check(ce, x, w, target, "none", dloss)
    _check(ce, x, w, target, "none", torch.zeros_like(dloss))
    xs, ws = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    want = torch.autograd.grad(ce(xs, ws, target, reduction="none"), xs, dloss)[0]
    for bad in (float("nan"), float("inf")):
        dloss[3] = bad
        dx, dw = torch.autograd.grad(ce(xs, ws, target, reduction="none"), (xs, ws), dloss)
        rest = torch.arange(tokens, device="cuda") != 3
        assert torch.equal(dx[rest], want[rest]) and not bool(dx[3].isfinite().any()) and bool(dw.isnan().any())


@pytest.mark.parametrize("tokens,vocab,k", [(96, 1025, 1160), (97, 2049, 520), (128, 3001, 264), (129, 3001, 264),
                                            (20, 20011, 1920)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_few_tokens(ce, tokens, vocab, k, dtype):
    """Around the 128 tokens up to which they are the tiles' columns."""
    for masked, reduction in ((0.0, "mean"), (0.3, "sum")):
        x, w, target = _inputs(tokens, vocab, k, dtype, seed=7, masked=masked)
        _check(ce, x, w, target, reduction, torch.tensor(8.0, device="cuda"))


@pytest.mark.parametrize("tokens,vocab,k", [(1000, 50257, 48), (4100, 30001, 40), (40, 400003, 24)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_several_pieces(ce, tokens, vocab, k, dtype):
    x, w, target = _inputs(tokens, vocab, k, dtype, seed=5, masked=0.2)
    _check(ce, x, w, target, "mean")
