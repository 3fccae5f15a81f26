"""What stands in for a call without a gradient (int8._NoGradient): its outputs are in the graph, going back raises."""
from __future__ import annotations

import pytest
import torch


def some_call(x, w, flag):
    return x.detach().round().to(torch.int8), x.detach() * 2, None if flag else w


def test_outputs_and_backward():
    from pollux_b200.int8 import _NoGradient, _tracked
    x, w = torch.randn(3, requires_grad=True), torch.ones(3)
    assert _tracked(None, x) and _tracked(w, x) and not _tracked(w, None) and not _tracked(x.detach())
    with torch.no_grad():
        assert not _tracked(x)
    q, y, none = _NoGradient.apply(some_call, x, w, True)
    assert none is None and not q.requires_grad and y.requires_grad
    with pytest.raises(NotImplementedError, match="some_call"):
        (y.sum() + x.sum()).backward()
    assert x.grad is None
