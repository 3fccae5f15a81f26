"""Tensors as rows, without a GPU: every number of leading dimensions, empty ones and an empty last one among them."""
from __future__ import annotations

import pytest
import torch


@pytest.mark.parametrize("shape,rows", [((2, 3, 0), 6), ((0,), 1), ((5,), 1), ((2, 0, 4), 0), ((2, 0, 0), 0), ((3, 0), 3),
                                        ((2, 3, 4), 6), ((1, 2, 3, 0), 6)])
def test_rows(shape, rows):
    from pollux_b200.int8 import _rows
    t = _rows(torch.zeros(shape), torch.device("cpu"))
    assert t.shape == (rows, shape[-1])
