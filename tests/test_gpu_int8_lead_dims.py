"""Leading dimensions in every number and size, an empty last dimension among them."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
LEAD = [(), (3,), (2, 3), (2, 0), (1, 2, 3)]


@pytest.mark.parametrize("lead", LEAD)
@pytest.mark.parametrize("cols", [0, 1, 24])
def test_shapes(lib, lead, cols):
    from pollux_b200 import int8
    x = torch.randn(*lead, cols, device="cuda")
    q, scale = int8.quantize_rows_int8(x)
    assert q.shape == x.shape and scale.shape == lead
    assert int8.dequantize_rows_int8(q, scale).shape == x.shape
    q, scale, summed = int8.add_rms_norm_int8(x, torch.ones(cols, device="cuda"), residual=x)
    assert q.shape == x.shape and scale.shape == lead and summed.shape == x.shape
    w = torch.ones(5, cols, device="cuda", dtype=torch.int8)
    mu, b = torch.ones(5, device="cuda").half(), torch.randn(5, device="cuda")
    y = int8.int8_linear(q, scale, w, mu, b)
    assert y.shape == lead + (5,)
    if cols == 0:
        assert torch.equal(y, b.expand(*lead, 5))
    # The same of a view that is not contiguous.
    wide = torch.zeros(*lead, cols + 3, device="cuda", dtype=torch.int8)[..., 1:cols + 1]
    wide.copy_(q)
    assert torch.equal(int8.int8_linear(wide, scale, w, mu, b), y)
    assert torch.equal(int8.dequantize_rows_int8(wide, scale), int8.dequantize_rows_int8(q, scale))
