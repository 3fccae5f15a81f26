"""Refusals of the INT8 head path that need no GPU: wrong types, sizes and
settings raise before anything is launched, in Python and at the C entries."""
from __future__ import annotations

import pytest
import torch


def test_norm_refusals(lib):
    from pollux_b200 import int8
    x, w = torch.zeros(2, 8), torch.ones(8)
    with pytest.raises(TypeError):
        int8.add_rms_norm_int8(x.double(), w)
    with pytest.raises(TypeError):
        int8.add_rms_norm_int8(x, w.to(torch.int32))
    with pytest.raises(ValueError, match="residual"):
        int8.add_rms_norm_int8(x, w, torch.zeros(2, 7))
    with pytest.raises(ValueError, match="residual"):
        int8.add_rms_norm_int8(x, w, x.half())
    with pytest.raises(ValueError, match="eps"):
        int8.add_rms_norm_int8(x, w, eps=-1.0)
    with pytest.raises(ValueError):
        int8.add_rms_norm_int8(torch.tensor(1.0), w)
    with pytest.raises(TypeError):
        int8.quantize_rows_int8(torch.zeros(2, 8, dtype=torch.int8))
    with pytest.raises(TypeError):
        int8.dequantize_rows_int8(x, torch.ones(2))
    with pytest.raises(TypeError):
        int8.dequantize_rows_int8(x.to(torch.int8), torch.ones(2), torch.int32)


def test_linear_refusals(lib):
    from pollux_b200 import int8
    q, s = torch.zeros(2, 8, dtype=torch.int8), torch.ones(2)
    w, mu = torch.zeros(3, 8, dtype=torch.int8), torch.ones(3).half()
    with pytest.raises(TypeError):
        int8.int8_linear(q.float(), s, w, mu)
    with pytest.raises(TypeError):
        int8.int8_linear(q, s, w, mu.float())
    with pytest.raises(ValueError):
        int8.int8_linear(q, s, w.view(1, 3, 8), mu)
    with pytest.raises(RuntimeError, match="shapes"):
        int8.int8_linear(q[:, :7], s, w, mu)
    with pytest.raises(TypeError):
        int8.int8_linear(q, s, w, mu, out_dtype=torch.int32)
    big = torch.zeros(1, 131_001, dtype=torch.int8)
    with pytest.raises(ValueError, match="in_features"):
        int8.int8_linear(big, s[:1], big, mu[:1])


def test_sampling_refusals(lib):
    from pollux_b200 import sampling
    l, u = torch.zeros(2, 8), torch.zeros(2)
    with pytest.raises(TypeError):
        sampling.sample_tokens(l.double(), u)
    with pytest.raises(ValueError, match="vocabulary"):
        sampling.sample_tokens(l[:, :0], u)
    for kw in (dict(temperature=-1.0), dict(temperature=float("nan")), dict(top_k=-1), dict(top_p=1.5),
               dict(top_p=-0.1), dict(min_p=2.0), dict(min_p=float("nan"))):
        with pytest.raises(ValueError, match="out of range"):
            sampling.sample_tokens(l, u, **kw)


def test_c_entries_refuse(lib):
    from pollux_b200 import _native as N
    bad = N.H24_ERR_INVALID
    p = 4096  # never dereferenced: every call is refused before a launch
    assert lib.h24_add_rms_norm_int8(p, None, p, 0, -1, 8, 8, 0, 0, 1e-6, p, p, None, None) == bad
    assert lib.h24_add_rms_norm_int8(p, None, p, 0, 1, 8, 8, 0, 7, 1e-6, p, p, None, None) == bad
    assert lib.h24_add_rms_norm_int8(p, None, p, 2, 1, 8, 8, 0, 1, 1e-6, p, p, None, None) == bad
    assert lib.h24_add_rms_norm_int8(p, None, None, 0, 1, 8, 8, 0, 0, 1e-6, p, p, None, None) == bad
    assert lib.h24_add_rms_norm_int8(p, None, p, 0, 1, 8, -8, 0, 0, 1e-6, p, p, None, None) == bad
    assert lib.h24_add_rms_norm_int8(p, None, p, 0, 1, 8, 8, 0, 0, -1.0, p, p, None, None) == bad
    assert lib.h24_add_rms_norm_int8(None, None, None, 0, 0, 8, 8, 0, 0, 1e-6, None, None, None, None) == N.H24_OK
    assert lib.h24_rows_int8_quantize(p, 1, -8, 8, 0, p, p, None) == bad
    assert lib.h24_rows_int8_quantize(None, 1, 8, 8, 0, p, p, None) == bad
    assert lib.h24_rows_int8_dequant(p, p, 1, 8, 5, p, None) == bad
    assert lib.h24_rows_int8_dequant(p, None, 1, 8, 0, p, None) == bad
    assert lib.h24_int8_linear(p, p, 1, 8, p, p, 8, 131001, None, 0, p, None) == bad
    assert b"131000" in lib.h24_last_error()
    assert lib.h24_int8_linear(p, p, -1, 8, p, p, 8, 8, None, 0, p, None) == bad
    assert lib.h24_int8_linear(p, p, 1, 8, p, p, 8, 8, None, 9, p, None) == bad
    assert lib.h24_int8_linear(p, p, 1, 8, p, None, 8, 8, None, 0, p, None) == bad
    assert lib.h24_int8_linear(None, None, 0, 8, None, None, 8, 8, None, 0, None, None) == N.H24_OK
    args = (1.0, None, 0, None, 1.0, None, 0.0)
    assert lib.h24_sample_tokens(p, 0, 1, (1 << 22) + 1, 8, p, None, *args, p, None, None) == bad
    assert lib.h24_sample_tokens(p, 0, 1, 0, 8, p, None, *args, p, None, None) == bad
    assert lib.h24_sample_tokens(p, 3, 1, 8, 8, p, None, *args, p, None, None) == bad
    assert lib.h24_sample_tokens(p, 0, 1, 8, 8, None, None, *args, p, None, None) == bad
    assert lib.h24_sample_tokens(None, 0, 0, 8, 8, None, None, *args, None, None, None) == N.H24_OK


def test_no_gpu_no_answer(lib):
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    from pollux_b200 import int8, sampling
    with pytest.raises(RuntimeError, match="CUDA"):
        int8.add_rms_norm_int8(torch.zeros(2, 8), torch.ones(8))
    with pytest.raises(RuntimeError, match="CUDA"):
        sampling.sample_tokens(torch.zeros(2, 8), torch.zeros(2))
