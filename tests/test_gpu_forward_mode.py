"""A tangent (forward-mode derivative) is not lost on the way past the general path either."""
from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwAD

pytestmark = pytest.mark.gpu


def test_a_tangent_raises(lib):
    from pollux_b200 import int8, loss, norm, sampling
    x = torch.randn(30, 48, device="cuda").half()
    g, b, w = torch.ones(48, device="cuda").half(), torch.zeros(48, device="cuda").half(), torch.randn(70, 48, device="cuda").half()
    t, u = torch.zeros(30, dtype=torch.int64, device="cuda"), torch.rand(30, device="cuda")
    q, s = int8.quantize_rows_int8(x)
    w8, mu = torch.zeros(70, 48, dtype=torch.int8, device="cuda"), torch.ones(70, device="cuda").half()
    calls = [(norm.add_rms_norm, (x, g)), (lambda x, r, g: norm.add_rms_norm(x, g, residual=r), (x, x, g)),
             (norm.add_layer_norm, (x, g, b)), (lambda x, w: loss.linear_cross_entropy(x, w, t), (x, w)),
             (int8.add_rms_norm_int8, (x, g)), (int8.quantize_rows_int8, (x,)),
             (lambda s: int8.dequantize_rows_int8(q, s), (s,)), (lambda s: int8.int8_linear(q, s, w8, mu), (s,)),
             (lambda z: sampling.sample_tokens(z, u, return_logprob=True), (x,))]
    for fn, args in calls:
        want = fn(*args)
        with fwAD.dual_level():
            for i, a in enumerate(args):
                for leaf in (a, a.detach().requires_grad_(True)):
                    dual = [*args[:i], fwAD.make_dual(leaf, torch.ones_like(a)), *args[i + 1:]]
                    with pytest.raises(NotImplementedError):
                        fn(*dual)
        again = fn(*args)
        for p, r in zip(want if isinstance(want, tuple) else (want,), again if isinstance(again, tuple) else (again,)):
            assert (p is None and r is None) or torch.equal(p, r)
