"""Gradients that are sums over very many tokens, or over a very large vocabulary, of terms of one sign
(loss.linear_cross_entropy): a sum in the tensor cores loses what falls below its last place at every addition, so long
ones are cut.

The head is 0 where dW is looked at, the states are 0 where dx is: all logits are 0 and a probability is 1 / vocab, a power
of two that d holds exactly.  Bounds, relative to the sum: 2^-23 for each 16 terms of a slice (131,072 terms, in fp16
32,768) and 2^-24 for each slice, 2^-18 of the exponentials, and half a step of the result; half the type's smallest.  In
the target's row d is 1 - 1 / vocab, which bf16's 8 bits do not hold from a vocabulary of 512 on: half a step more."""
from __future__ import annotations

import pytest
import torch

from test_gpu_linear_ce import _check, _inputs

pytestmark = pytest.mark.gpu
SLICE = {torch.bfloat16: 131072, torch.float16: 32768}
DTYPES = [torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def ce(lib):
    from pollux_b200 import loss
    return loss.linear_cross_entropy


def _bound(dtype, terms):
    n = min(terms, SLICE[dtype])
    return (n / 16 + 8) * 2.0 ** -23 + (terms / SLICE[dtype] + 1) * 2.0 ** -24 + 2.0 ** -18 + torch.finfo(dtype).eps / 2


@pytest.mark.parametrize("tokens,vocab,k", [(1048576, 64, 64), (1000003, 256, 49), (20000, 64, 300), (32769, 512, 24),
                                            (140000, 1024, 16)])
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_dw_over_many_tokens(ce, tokens, vocab, k, masked, dtype):
    g = torch.Generator(device="cuda").manual_seed(tokens)
    x = (0.5 + torch.rand(tokens, k, generator=g, device="cuda")).to(dtype).requires_grad_(True)
    w = torch.zeros(vocab, k, device="cuda", dtype=dtype, requires_grad=True)
    target = torch.full((tokens,), 3, device="cuda")
    if masked:
        target[torch.rand(tokens, generator=g, device="cuda") < 0.3] = -100
    keep = (target != -100).double()
    dx, dw = torch.autograd.grad(ce(x, w, target), (x, w), torch.tensor(float(vocab), device="cuda"))
    mean = (x.detach().double() * keep[:, None]).sum(0) / keep.sum()
    want = mean.expand(vocab, k).clone()
    want[3] = mean * (1 - vocab)
    bound = torch.full((vocab, 1), _bound(dtype, tokens), dtype=torch.float64, device="cuda")
    bound[3] += torch.finfo(dtype).eps / 2
    assert bool(((dw.double() - want).abs() <= want.abs() * bound).all()), float(((dw.double() - want).abs() / want.abs()).max())
    assert not bool(dx.any())  # (a head of zeros)


@pytest.mark.parametrize("tokens,vocab,k", [(3, 262144, 1024), (200, 131072, 48), (130, 65536, 1536), (1, 524288, 24)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_dx_over_a_large_vocabulary(ce, tokens, vocab, k, dtype):
    g = torch.Generator(device="cuda").manual_seed(vocab)
    w = torch.empty(vocab, k, device="cuda", dtype=dtype)
    for a in range(0, vocab, 65536):
        w[a:a + 65536] = (0.5 + torch.rand(min(65536, vocab - a), k, generator=g, device="cuda")).to(dtype)
    target = torch.full((tokens,), 3, device="cuda")
    w[3] = 0
    mean = sum(w[a:a + 16384].double().sum(0) for a in range(0, vocab, 16384)) / vocab
    x = torch.zeros(tokens, k, device="cuda", dtype=dtype, requires_grad=True)
    (dx,) = torch.autograd.grad(ce(x, w, target, reduction="sum"), x)
    bound = mean * _bound(dtype, vocab) + (2.0 ** -134 if dtype == torch.bfloat16 else 2.0 ** -25)
    assert bool(((dx.double() - mean).abs() <= bound).all())


@pytest.mark.parametrize("tokens,vocab,k", [(24577, 8200, 40), (25000, 9001, 24), (40000, 4097, 33)])
@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_several_pieces_of_many_tokens(ce, tokens, vocab, k, reduction, dtype):
    """From 24,577 tokens on a piece of the vocabulary is 4,096 columns at least, whatever its bytes: two and three of them,
    the last one short, against the formulas."""
    x, w, target = _inputs(tokens, vocab, k, dtype, seed=37, masked=0.2)
    dloss = torch.rand(tokens, device="cuda") * 0.05 if reduction == "none" else None
    _check(ce, x, w, target, reduction, dloss)


@pytest.mark.parametrize("tokens,vocab,k,dtype", [(33000, 300, 1500, torch.float16), (132000, 260, 4200, torch.bfloat16)])
def test_long_in_both(ce, tokens, vocab, k, dtype):
    """Tokens and k longer than a slice, in one kernel."""
    x, w, target = _inputs(tokens, vocab, k, dtype, seed=41, masked=0.1)
    _check(ce, x, w, target, "mean", torch.tensor(512.0, device="cuda"))


def test_captured_with_factors_in_fp16(ce):
    """Scratch of the sizes and counts by blocks, new values at each replay."""
    for tokens, vocab, k in ((60, 300, 72), (700, 900, 113), (17000, 40, 24)):
        x, w, target = _inputs(tokens, vocab, k, torch.float16, seed=43, masked=0.2)
        x, w = x.requires_grad_(True), w.requires_grad_(True)
        dloss = torch.rand(tokens, device="cuda")

        def step():
            value = ce(x, w, target, reduction="none")
            return (value, *torch.autograd.grad(value, (x, w), dloss))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        for seed in range(3):
            with torch.no_grad():
                x.normal_()
                dloss.copy_(2.0 ** (torch.rand(tokens, device="cuda") * 20 - 18 + seed))
                target.random_(0, vocab)
                target[seed::4] = -100
            graph.replay()
            assert all(torch.equal(a, b) for a, b in zip(out, step()))
