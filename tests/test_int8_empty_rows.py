"""Rows without elements: their scale is that of a row of zeros, and a product with them is the bias."""
from __future__ import annotations

import pytest
import torch


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_scale_of_rows_without_elements(lib, dtype):
    from pollux_b200 import int8
    want = int8.quantize_rows_int8(torch.zeros(1, 8, device="cuda", dtype=dtype))[1]
    for rows in (1, 5, 3000):
        for fill in (float("nan"), 7.0):  # what a scale would hold that nothing writes
            junk = torch.full((rows,), fill, device="cuda")
            del junk
            x = torch.zeros(rows, 0, device="cuda", dtype=dtype)
            q, scale = int8.quantize_rows_int8(x)
            assert q.shape == (rows, 0) and torch.equal(scale, want.expand(rows))
            junk = torch.full((rows,), fill, device="cuda")
            del junk
            for r in (None, x):
                q, scale, summed = int8.add_rms_norm_int8(x, x[0], r)
                assert q.shape == (rows, 0) and torch.equal(scale, want.expand(rows))
                assert (summed is None) if r is None else summed.shape == (rows, 0)
    w = torch.zeros(50, 0, device="cuda", dtype=torch.int8)
    y = int8.int8_linear(q, scale, w, torch.ones(50, device="cuda").half())
    assert y.shape == (3000, 50) and (y == 0).all()


def test_c_entries_ask_for_the_scale(lib):
    """A call with rows but no elements has one output, the scales."""
    from pollux_b200 import _native as N
    assert lib.h24_add_rms_norm_int8(None, None, None, 0, 3, 0, 0, 0, 0, 1e-6, None, None, None, None) == N.H24_ERR_INVALID
    assert lib.h24_rows_int8_quantize(None, 3, 0, 0, 0, None, None, None) == N.H24_ERR_INVALID
    assert lib.h24_add_rms_norm_int8(None, None, None, 0, 0, 0, 0, 0, 0, 1e-6, None, None, None, None) == N.H24_OK
    assert lib.h24_rows_int8_quantize(None, 0, 0, 0, 0, None, None, None) == N.H24_OK
