"""The INT8 head path records no gradient, and says so: a backward pass that reaches it raises."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def m(lib):
    from pollux_b200 import int8, sampling
    return int8, sampling


def _layer(bias=False):
    from pollux_b200 import packed_linear as pl
    lin = pl.PackedInt8Linear(48, 100, bias=bias).cuda()
    lin.weight_int8.copy_(torch.randint(-127, 128, (100, 48), device="cuda", dtype=torch.int8))
    lin.mu_rows.fill_(0.1)
    return lin


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_model_with_a_trainable_backbone(m, bias, dtype):
    """The head's loss must not lose its gradient silently beside another loss."""
    body, head = torch.nn.Linear(48, 48).cuda().to(dtype), _layer(bias)
    assert m[0].enable_int8_forward(head) == 1
    hidden = body(torch.randn(6, 48, device="cuda", dtype=dtype))
    y = head(hidden)
    assert y.requires_grad
    with pytest.raises(NotImplementedError, match="gradient"):
        (y.float().square().mean() + hidden.float().square().mean()).backward()
    # Where nothing asks for a gradient, the same outputs without one.
    with torch.no_grad():
        z = head(hidden)
    assert not z.requires_grad and torch.equal(z, y.detach())
    if not bias:
        assert not head(hidden.detach()).requires_grad
    with torch.inference_mode():
        assert torch.equal(head(hidden.detach()), z)


def test_the_entries(m):
    int8, sampling = m
    x = torch.randn(4, 48, device="cuda", requires_grad=True)
    r = torch.randn(4, 48, device="cuda")
    w = torch.ones(48, device="cuda")
    for args in ((x, w, r), (r, w, x), (r, w.clone().requires_grad_(), r), (x, w, None)):
        want = int8.add_rms_norm_int8(*(None if a is None else a.detach() for a in args))
        q, scale, summed = int8.add_rms_norm_int8(*args)
        assert not q.requires_grad and scale.requires_grad and torch.equal(q, want[0]) and torch.equal(scale, want[1])
        for out in (scale,) if summed is None else (scale, summed):
            with pytest.raises(NotImplementedError, match="add_rms_norm_int8"):
                out.sum().backward(retain_graph=True)
    assert x.grad is None
    q, scale = int8.quantize_rows_int8(x)
    assert not q.requires_grad
    y = int8.dequantize_rows_int8(q, scale)
    with pytest.raises(NotImplementedError, match="gradient"):
        y.sum().backward(retain_graph=True)
    w8, mu = torch.ones(7, 48, device="cuda", dtype=torch.int8), torch.ones(7, device="cuda").half()
    y = int8.int8_linear(q, scale.detach(), w8, mu, torch.ones(7, device="cuda", requires_grad=True))
    with pytest.raises(NotImplementedError, match="int8_linear"):
        y.sum().backward()
    logits = torch.randn(4, 100, device="cuda", requires_grad=True)
    u = torch.rand(4, device="cuda")
    tok, lp = sampling.sample_tokens(logits, u, return_logprob=True)
    assert not tok.requires_grad and lp.requires_grad
    with pytest.raises(NotImplementedError, match="sample_tokens"):
        lp.sum().backward()
    assert not sampling.sample_tokens(logits, u).requires_grad
    assert torch.equal(sampling.sample_tokens(logits.detach(), u), tok)


def test_in_place_on_an_output(m):
    """What comes back is a tensor of its own, not a view."""
    int8 = m[0]
    y = int8.quantize_rows_int8(torch.randn(4, 48, device="cuda", requires_grad=True))[1]
    y.mul_(2)
    assert y.requires_grad
