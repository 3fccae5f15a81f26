"""Activations in 8 bits (int8.add_rms_norm_int8, quantize_rows_int8,
dequantize_rows_int8) against their formulas in 64 bits.

Bounds.  u = 2^-24.  s, v carry one rounding each, so q differs from the exact
v/max|v| * 127 by at most 1/2 plus 127 * 8u (the roundings of s, v, max, the
two factors and their product).  The scale carries those, the square root and
division, and half the error of a sum of cols positive squares, taken in
chains of at most cols/32 + 32 additions."""
from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def m(lib):
    from pollux_b200 import int8
    return int8


def _inputs(rows, cols, dtype, seed, residual=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, cols, generator=g, device="cuda").to(dtype)
    r = (3 * torch.randn(rows, cols, generator=g, device="cuda")).to(dtype) if residual else None
    w = (1 + 0.3 * torch.randn(cols, generator=g, device="cuda")).to(dtype)
    return x, r, w


def _check(q, scale, v, inv, cols):
    """q, scale against v (64 bits) and the factor inv."""
    mu = torch.clamp_min(v.abs().amax(-1) * inv, 1e-8)
    tol = (16 + (cols / 32 + 32) / 2) * U
    assert ((scale.double() - mu / 127).abs() <= tol * mu / 127).all()
    err = (q.double() - v * (inv / mu * 127)[..., None]).abs()
    assert err.max() <= 0.5 + 127 * 8 * U, err.max()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 24), (3, 7), (1, 1920), (5, 1152), (130, 1920), (33, 1153),
                                       (2, 4099), (7, 8192), (3, 8200), (2, 20001), (2, 65536), (1000, 48)])
@pytest.mark.parametrize("residual", [True, False])
def test_norm_matches_formula(m, dtype, rows, cols, residual):
    x, r, w = _inputs(rows, cols, dtype, rows * 100003 + cols, residual)
    q, scale, summed = m.add_rms_norm_int8(x, w, r, eps=1e-5)
    s = x.double() + (r.double() if residual else 0)
    inv = 1 / torch.sqrt((s * s).mean(-1) + 1e-5)
    _check(q, scale, s * w.double(), inv, cols)
    if residual:
        assert torch.equal(summed, (x.float() + r.float()).to(dtype))
    else:
        assert summed is None


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (64, 7680), (9, 1921), (2, 30000)])
def test_quantize_and_back(m, dtype, rows, cols):
    x, _, _ = _inputs(rows, cols, dtype, cols, False)
    q, scale = m.quantize_rows_int8(x)
    _check(q, scale, x.double(), torch.ones(rows, device="cuda", dtype=torch.float64), cols)
    for out in DTYPES:
        y = m.dequantize_rows_int8(q, scale, out)
        assert y.dtype == out and torch.equal(y, (q.float() * scale[:, None]).to(out))


def test_gain_types(m):
    x, r, w = _inputs(17, 1920, torch.bfloat16, 5)
    base = m.add_rms_norm_int8(x, w, r)
    for wt in (w.float(), w.half().to(torch.bfloat16), w.float().double().float()):
        got = m.add_rms_norm_int8(x, wt, r)
        assert torch.equal(got[0], base[0]) and torch.equal(got[1], base[1])
    # A gain in the other 16-bit type is widened, not rounded to x's type.
    wh = (1 + 0.3 * torch.randn(1920, device="cuda")).half()
    assert torch.equal(m.add_rms_norm_int8(x, wh, r)[0], m.add_rms_norm_int8(x, wh.float(), r)[0])


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_offsets_and_shapes(m, dtype):
    base = torch.randn(40, 2 * 96 + 5, device="cuda").to(dtype)
    w = torch.randn(96, device="cuda").to(dtype)
    views = [base[:, :96], base[:, 1:97], base[:, 3:99], base[::2, 8:104], base[1:2, 5:101], base.t()[:96].t(),
             base[3, 7:103].expand(6, 96)]
    for x in views:
        r = torch.randn(x.shape, device="cuda").to(dtype)
        want = m.add_rms_norm_int8(x.contiguous().clone(), w, r)
        got = m.add_rms_norm_int8(x, w, r)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        got = m.add_rms_norm_int8(r, w, x)
        want = m.add_rms_norm_int8(r, w, x.contiguous().clone())
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    x3 = torch.randn(4, 5, 96, device="cuda").to(dtype)
    q, s, t = m.add_rms_norm_int8(x3, w, x3)
    assert q.shape == (4, 5, 96) and s.shape == (4, 5) and t.shape == x3.shape
    x1 = x3[0, 0]
    q1, s1, t1 = m.add_rms_norm_int8(x1, w, x1)
    assert torch.equal(q1, q[0, 0]) and torch.equal(s1, s[0, 0]) and torch.equal(t1, t[0, 0])


@pytest.mark.parametrize("cols", [24, 1153, 1920, 9000])
def test_special_rows(m, cols):
    x = torch.randn(8, cols, device="cuda")
    x[0] = 0
    x[1, cols // 2] = float("nan")
    x[2, 3] = float("inf")
    x[3] = 1e-30
    x[4] *= 1e15
    w = torch.ones(cols, device="cuda")
    q, scale, summed = m.add_rms_norm_int8(x, w, torch.zeros_like(x), eps=1e-6)
    assert (q[0] == 0).all() and abs(scale[0].item() * 127 / 1e-8 - 1) < 1e-6
    assert (q[1:3] == 0).all() and torch.isnan(scale[1:3]).all()
    assert torch.isnan(m.dequantize_rows_int8(q, scale)[1:3]).all()
    s = x[3:].double()
    _check(q[3:], scale[3:], s, 1 / torch.sqrt((s * s).mean(-1) + 1e-6), cols)
    # The quantisation alone: the largest value maps to 127, NaN to a NaN scale.
    q, scale = m.quantize_rows_int8(x)
    assert torch.isnan(scale[1]) and (q[1] == 0).all() and (q[0] == 0).all()
    assert (q[4:].abs().amax(-1) == 127).all()


def test_in_place_and_streams(m):
    x, r, w = _inputs(300, 1920, torch.bfloat16, 9)
    want = m.add_rms_norm_int8(x, w, r)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = m.add_rms_norm_int8(x, w, r)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # The C entry may write the sum over the residual.
    from pollux_b200 import _native as N
    q, s = torch.empty_like(want[0]), torch.empty_like(want[1])
    r2 = r.clone()
    N.call("h24_add_rms_norm_int8", x.data_ptr(), r2.data_ptr(), w.data_ptr(), N.DTYPE_BF16, 300, 1920, 1920, 1920,
           N.DTYPE_BF16, 1e-6, q.data_ptr(), s.data_ptr(), r2.data_ptr(), torch.cuda.current_stream().cuda_stream)
    assert torch.equal(q, want[0]) and torch.equal(s, want[1]) and torch.equal(r2, want[2])


def test_host_tensors_and_empty(m):
    x, r, w = _inputs(3, 48, torch.float32, 11)
    want = m.add_rms_norm_int8(x, w, r)
    got = m.add_rms_norm_int8(x.cpu(), w.cpu(), r.cpu())
    assert all(g.device.type == "cpu" and torch.equal(g, t.cpu()) for g, t in zip(got, want))
    q, s, t = m.add_rms_norm_int8(x[:0], w, r[:0])
    assert q.shape == (0, 48) and s.shape == (0,) and t.shape == (0, 48)
    assert m.quantize_rows_int8(x[:0])[0].shape == (0, 48)
    assert m.dequantize_rows_int8(q, s).shape == (0, 48)


def test_more_rows_than_a_grid(m):
    x = torch.randn(70001, 24, device="cuda", dtype=torch.float16)
    w = torch.ones(24, device="cuda", dtype=torch.float16)
    q, scale, _ = m.add_rms_norm_int8(x, w)
    s = x.double()
    _check(q, scale, s, 1 / torch.sqrt((s * s).mean(-1) + 1e-6), 24)


def test_offsets_beyond_32_bits(m):
    """Rows 1.2e9 elements apart: element offsets pass 2^31, byte offsets 2^32."""
    base = torch.empty(2_400_000_200, device="cuda", dtype=torch.bfloat16)
    for cols in (96, 93):
        x = base.as_strided((3, cols), (1_200_000_000, 1))
        x.copy_(torch.randn(3, cols, device="cuda"))
        w = torch.randn(cols, device="cuda").to(torch.bfloat16)
        r = torch.randn(3, cols, device="cuda").to(torch.bfloat16)
        for args in ((x, w, r), (r, w, x)):
            got = m.add_rms_norm_int8(*args)
            want = m.add_rms_norm_int8(*(a.contiguous() for a in args))
            assert all(torch.equal(a, b) for a, b in zip(got, want))
