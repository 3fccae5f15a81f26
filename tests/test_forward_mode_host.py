"""A tangent (forward-mode derivative) is not lost: every call that would have to carry one on raises.  The general path,
with the kernels' calls left out."""
from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwAD


@pytest.fixture
def general(lib, monkeypatch):
    from pollux_b200 import _native as N
    from pollux_b200 import int8, loss, norm, sampling
    monkeypatch.setattr(N, "_torch_calls", N._GeneralPath())
    for m in (int8, loss, norm, sampling):
        monkeypatch.setattr(m, "_call", lambda *a: None)
        monkeypatch.setattr(m, "_stream", lambda dev: 0)
        monkeypatch.setattr(m, "_work_device", lambda t: t.device)
    return int8, loss, norm, sampling


def _calls(int8, loss, norm, sampling):
    w, mu = torch.zeros(5, 8, dtype=torch.int8), torch.ones(5, dtype=torch.float16)
    t = torch.zeros(3, dtype=torch.int64)
    q = torch.zeros(3, 8, dtype=torch.int8)
    return {
        "rms": (lambda x, g: norm.add_rms_norm(x, g), (torch.randn(3, 8), torch.ones(8))),
        "residual": (lambda x, r, g: norm.add_rms_norm(x, g, residual=r), (torch.randn(3, 8), torch.randn(3, 8), torch.ones(8))),
        "layer": (lambda x, g, b: norm.add_layer_norm(x, g, b), (torch.randn(3, 8), torch.ones(8), torch.zeros(8))),
        "loss": (lambda x, w: loss.linear_cross_entropy(x, w, t), (torch.randn(3, 8).half(), torch.randn(5, 8).half())),
        "norm to int8": (lambda x, g: int8.add_rms_norm_int8(x, g), (torch.randn(3, 8), torch.ones(8))),
        "quantize": (lambda x: int8.quantize_rows_int8(x), (torch.randn(3, 8),)),
        "dequantize": (lambda s: int8.dequantize_rows_int8(q, s), (torch.rand(3),)),
        "int8 product": (lambda s: int8.int8_linear(q, s, w, mu), (torch.rand(3),)),
        "log-probability": (lambda z: sampling.sample_tokens(z, torch.rand(3), return_logprob=True), (torch.randn(3, 5),)),
    }


NAMES = ["rms", "residual", "layer", "loss", "norm to int8", "quantize", "dequantize", "int8 product", "log-probability"]


@pytest.mark.parametrize("name", NAMES)
def test_a_tangent_raises(general, name):
    fn, args = _calls(*general)[name]
    fn(*args)
    with fwAD.dual_level():
        fn(*args)  # no tangent among them
        for i, a in enumerate(args):
            for leaf in (a, a.detach().requires_grad_(True)):
                dual = [*args[:i], fwAD.make_dual(leaf, torch.ones_like(a)), *args[i + 1:]]
                with pytest.raises(NotImplementedError):
                    fn(*dual)
                with torch.no_grad(), pytest.raises(NotImplementedError):
                    fn(*dual)
    fn(*args)


def test_tokens_have_no_tangent(general):
    """Whole numbers carry none, so a sample of dual logits is one."""
    with fwAD.dual_level():
        z = fwAD.make_dual(torch.randn(3, 5), torch.ones(3, 5))
        assert general[3].sample_tokens(z, torch.rand(3)).dtype == torch.int64
