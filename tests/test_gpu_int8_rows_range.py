"""Rows whose squares leave fp32's range, and rows without elements.

Bounds as in test_gpu_int8_rows.py: q within 1/2 + 127 * 8u of the exact
quotient; the scale within the roundings of s, v, the root, the division and of
a sum of cols squares."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def m(lib):
    from pollux_b200 import int8
    return int8


def _check(q, scale, v, inv, cols):
    mu = torch.clamp_min(v.abs().amax(-1) * inv, 1e-8)
    tol = (16 + (cols / 32 + 32) / 2) * U
    assert torch.isfinite(scale).all()
    assert ((scale.double() - mu / 127).abs() <= tol * mu / 127).all()
    err = (q.double() - v * (inv / mu * 127)[..., None]).abs()
    assert err.max() <= 0.5 + 127 * 8 * U, err.max()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("cols", [1, 24, 93, 1153, 1920, 9000, 20001, 70003])
@pytest.mark.parametrize("residual", [True, False])
def test_squares_beyond_fp32(m, dtype, cols, residual):
    """Finite rows whose sum of squares exceeds the largest fp32 number, beside ordinary ones in the same blocks."""
    g = torch.Generator(device="cuda").manual_seed(cols)
    rows = 700
    x = torch.randn(rows, cols, generator=g, device="cuda")
    power = torch.tensor([0.0, 1e17, 3e18, 1e19, 2e19, 1e25, 1e31, 1e37], device="cuda")[torch.arange(rows, device="cuda") % 8]
    x = torch.where(power[:, None] > 0, x.clamp(-5, 5) * power[:, None], x)
    x[5::8, cols // 2] = 3e25  # (an element far above its row)
    x[1::8, cols - 1] = 1e30
    x = x.to(dtype)
    r = x.roll(1, 1).clone() if residual else None
    w = (1 + 0.3 * torch.randn(cols, generator=g, device="cuda").clamp(-2, 2)).to(dtype)
    q, scale, summed = m.add_rms_norm_int8(x, w, r, eps=1e-5)
    s = x.double() + (r.double() if residual else 0)
    _check(q, scale, s * w.double(), 1 / torch.sqrt((s * s).mean(-1) + 1e-5), cols)
    if residual:
        assert torch.equal(summed, (x.float() + r.float()).to(dtype))
    # The row alone gives the same bits.
    for i in (0, 4, 5, 6, 7):
        q1, s1, _ = m.add_rms_norm_int8(x[i:i + 1], w, None if r is None else r[i:i + 1], eps=1e-5)
        assert torch.equal(q1[0], q[i]) and torch.equal(s1[0], scale[i])


@pytest.mark.parametrize("cols", [93, 1920, 70003])
def test_squares_beyond_fp32_special(m, cols):
    """In such rows too: a NaN or an infinite element gives a NaN scale, gains of 0 the least scale, and eps counts."""
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(6, cols, generator=g, device="cuda").clamp(-3, 3) * 1e25
    x[1, 3], x[2, 3], x[3, cols - 1] = float("nan"), float("inf"), float("-inf")
    w = torch.ones(cols, device="cuda")
    q, scale, _ = m.add_rms_norm_int8(x, w)
    assert torch.isnan(scale[1:4]).all() and (q[1:4] == 0).all()
    assert torch.isfinite(scale[[0, 4, 5]]).all()
    q, scale, _ = m.add_rms_norm_int8(x[4:], torch.zeros_like(w))
    assert (q == 0).all() and ((scale * 127 / 1e-8 - 1).abs() < 1e-6).all()
    small = torch.full_like(w, 1e-12)
    s = x[4:].double()
    q, scale, _ = m.add_rms_norm_int8(x[4:], small)
    _check(q, scale, s * small.double(), 1 / torch.sqrt((s * s).mean(-1) + 1e-6), cols)
    big = torch.tensor(1e38).item()
    inv = 1 / torch.sqrt((s * s).mean(-1) * 1e-12 + big)  # rows of 1e19 with an eps of their squares' size
    q, scale, _ = m.add_rms_norm_int8((s * 1e-6).float(), w, eps=big)
    _check(q, scale, (s * 1e-6).float().double(), inv, cols)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("cols", [93, 1920, 70008])
def test_squares_beyond_fp32_in_place(m, dtype, cols):
    """The sum may lie over x or the residual.  Such rows of 16 bits may be of the rounded sum, each element within
    2^-9: v / max|v| within 2^-8, so that q moves by 127 * 2^-8 < 1/2 before its rounding, and the scale within 2^-8."""
    from pollux_b200 import _native as N
    code = {torch.float32: N.DTYPE_F32, torch.bfloat16: N.DTYPE_BF16}[dtype]
    x = (torch.randn(40, cols, device="cuda").clamp(-3, 3) * 1e22).to(dtype)
    r = (torch.randn(40, cols, device="cuda").clamp(-3, 3) * 1e22).to(dtype)
    w = torch.ones(cols, device="cuda", dtype=dtype)
    want = m.add_rms_norm_int8(x, w, r)
    assert torch.isfinite(want[1]).all() and (want[0].abs().amax(-1) == 127).all()
    for over_x in (False, True):
        xc, rc = x.clone(), r.clone()
        q, s = torch.empty_like(want[0]), torch.empty_like(want[1])
        out = xc if over_x else rc
        N.call("h24_add_rms_norm_int8", xc.data_ptr(), rc.data_ptr(), w.data_ptr(), code, 40, cols, cols, cols,
               code, 1e-6, q.data_ptr(), s.data_ptr(), out.data_ptr(), torch.cuda.current_stream().cuda_stream)
        assert torch.equal(out, want[2])
        if dtype == torch.float32 or cols > 65536:
            assert torch.equal(q, want[0]) and torch.equal(s, want[1])
        else:
            assert (q.int() - want[0].int()).abs().max() <= 1
            assert ((s.double() / want[1].double() - 1).abs() <= 2.0 ** -8 * 1.01).all()
