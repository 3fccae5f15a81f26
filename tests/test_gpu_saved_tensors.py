"""Norms and loss of the training head path under hooks on saved tensors: checkpoints, tensors kept elsewhere, hooks that
raise and hooks that give something else back."""
from __future__ import annotations

import pytest
import torch
from torch.autograd.graph import saved_tensors_hooks
from torch.utils.checkpoint import checkpoint

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.fixture(scope="module")
def calls(lib):
    """name -> (function of the leaves, leaves)"""
    from pollux_b200 import loss, norm
    g = torch.Generator(device="cuda").manual_seed(0)

    def leaf(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(BF).requires_grad_(True)
    x, r, gain, bias, w = leaf(70, 96), leaf(70, 96), leaf(96), leaf(96), leaf(500, 96, scale=0.2)
    t = torch.randint(0, 500, (70,), generator=g, device="cuda")
    return {
        "rms": (lambda x, w: norm.add_rms_norm(x * 2, w)[0], (x, gain)),
        "residual": (lambda x, r, w: sum(norm.add_rms_norm(x * 2, w, residual=r * 3)), (x, r, gain)),
        "layer": (lambda x, r, w, b: norm.add_layer_norm(x * 2, w, b, residual=r)[0], (x, r, gain, bias)),
        "loss": (lambda x, w: loss.linear_cross_entropy(x * 2, w, t), (x, w)),
        "together": (lambda x, g, w: loss.linear_cross_entropy(norm.add_rms_norm(x * 2, g)[0], w, t), (x, gain, w)),
    }


NAMES = ["rms", "residual", "layer", "loss", "together"]


@pytest.fixture(params=[True, False], ids=["direct", "general"])
def path(request, lib):
    """With the torch module and without it."""
    from pollux_b200 import _native as N
    before = N.torch_calls()
    if not request.param:
        N._torch_calls = N._GeneralPath()
    yield request.param
    N._torch_calls = before


def _grads(fn, leaves):
    return torch.autograd.grad(fn(*leaves).float().square().sum(), leaves)


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("reentrant", [False, True])
def test_checkpointed(calls, path, name, reentrant):
    """The same gradients with the call computed again in the backward pass, which ends it inside a hook."""
    fn, leaves = calls[name]
    want = _grads(fn, leaves)
    for p in leaves:
        p.grad = None
    checkpoint(fn, *leaves, use_reentrant=reentrant).float().square().sum().backward()
    for p, g in zip(leaves, want):
        assert torch.equal(p.grad, g)
        p.grad = None


class Stop(Exception):
    pass


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("which", [1, 2, 3])
def test_a_hook_that_raises(calls, path, name, which):
    """Its exception arrives, whichever tensor it is, and the next call is as ever."""
    fn, leaves = calls[name]
    want = _grads(fn, leaves)
    seen = []

    def pack(t):
        seen.append(t)
        if len(seen) == which + 1:  # (the first belongs to the product before the call)
            raise Stop
        return t
    with saved_tensors_hooks(pack, lambda t: t):
        try:
            fn(*leaves)
            assert len(seen) <= which
        except Stop:
            pass
    assert all(torch.equal(a, b) for a, b in zip(_grads(fn, leaves), want))


@pytest.mark.parametrize("name", NAMES)
def test_kept_on_the_host(calls, path, name):
    fn, leaves = calls[name]
    want = _grads(fn, leaves)
    with torch.autograd.graph.save_on_cpu():
        value = fn(*leaves).float().square().sum()
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(value, leaves), want))


def _other_strides(t):
    """The same values: a matrix by columns, a vector by every second element, another view of the same rows."""
    if t.dim() == 2:
        return t.t().contiguous().t()
    if t.dim() == 1:
        wide = t.new_zeros(2 * t.numel())
        wide[::2] = t
        return wide[::2]
    return t


@pytest.mark.parametrize("name", NAMES)
def test_a_hook_that_gives_other_strides(calls, path, name):
    fn, leaves = calls[name]
    want = _grads(fn, leaves)
    with saved_tensors_hooks(lambda t: t, _other_strides):
        value = fn(*leaves).float().square().sum()
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(value, leaves), want))


@pytest.mark.parametrize("name", ["rms", "residual", "layer", "loss"])
@pytest.mark.parametrize("change", [lambda t: t.float() if t.dtype == BF else t.double(), lambda t: t[..., :-1], lambda t: t.cpu(),
                                    lambda t: t[None]], ids=["type", "shorter", "device", "shape"])
def test_a_hook_that_gives_something_else(calls, path, name, change):
    """What is saved by the call itself comes back changed, and is refused before a kernel sees it."""
    fn, leaves = calls[name]
    want = _grads(fn, leaves)
    inside = []

    def unpack(t):
        return change(t) if inside else t
    with saved_tensors_hooks(lambda t: t, unpack):
        out = fn(*leaves)
    inside.append(1)
    with pytest.raises(RuntimeError, match="hook on saved tensors"):
        torch.autograd.grad(out, leaves, torch.ones_like(out))
    assert all(torch.equal(a, b) for a, b in zip(_grads(fn, leaves), want))
