"""norm.add_rms_norm and add_layer_norm against their formulas in 64 bits, with gradients.

Bounds.  u = 2^-24, h half a step of the type relative to the value (eps / 2).  A row's sums run over chains of at most
16 + 5 + 32 additions, a factor of 64 u of the sum of magnitudes with the division.
  mean     em = 64 u mean|s|
  s - m    ed = em + u (|s| + |m|)
  i        relative ei = 34 u + rms(ed) / sigma
  n        en = ed i + |n| (ei + 3 u)
  y        |w| en + 4 u (|n w| + |b|) + h |y|, half a smallest step
  c1, c2   the means of v n and v: mean(|v| en) + 68 u mean|v n|, and 66 u mean|v|
  dx       i (3 u |v| + |n| ec1 + |c1| en + ec2 + 4 u (|n c1| + |c2|)) + ei |ds| + 2 u (|ds| + |dsummed|) + h |dx|
  dw, db   sum|dy| en, and for the chain (a block's rows, blocks in 32 groups, the groups) rows / 64 + 100 additions"""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}


@pytest.fixture(scope="module")
def m(lib):
    from pollux_b200 import norm
    return norm


def _inputs(rows, cols, dtype, residual=True, layer=True, seed=0):
    g = torch.Generator(device="cuda").manual_seed(rows * 100003 + cols + seed)

    def rand(*shape):
        return torch.randn(*shape, generator=g, device="cuda")
    out = {"x": rand(rows, cols).to(dtype), "residual": (3 * rand(rows, cols)).to(dtype) if residual else None,
           "weight": (1 + 0.3 * rand(cols)).to(dtype), "bias": (0.5 * rand(cols)).to(dtype) if layer else None,
           "dy": rand(rows, cols).to(dtype), "dsummed": rand(rows, cols).to(dtype) if residual else None}
    return out


def _call(m, i, layer, eps):
    if layer:
        return m.add_layer_norm(i["x"], i["weight"], i["bias"], residual=i["residual"], eps=eps)
    return m.add_rms_norm(i["x"], i["weight"], residual=i["residual"], eps=eps)


def _run(m, i, layer, eps=1e-5):
    i = dict(i)
    for k in ("x", "residual", "weight", "bias"):
        if i[k] is not None:
            i[k] = i[k].detach().requires_grad_(True)
    y, summed = _call(m, i, layer, eps)
    outs, grads = ([y], [i["dy"]]) if summed is None else ([y, summed], [i["dy"], i["dsummed"]])
    leaves = {k: i[k] for k in ("x", "residual", "weight", "bias") if i[k] is not None}
    got = dict(zip(leaves, torch.autograd.grad(outs, list(leaves.values()), grads)))
    return y.detach(), None if summed is None else summed.detach(), got


def _half(t):
    return torch.finfo(t).eps / 2


def _close(got, want, bound, what):
    bad = ~((got.double() - want).abs() <= bound)
    assert not bool(bad.any()), (what, int(bad.sum()), float(((got.double() - want).abs() / bound).max()))


def _check(m, i, layer, eps=1e-5, param=None):
    dtype = i["x"].dtype
    y, summed, got = _run(m, i, layer, eps)
    if i["residual"] is None:
        assert summed is None
        s = i["x"].double()
    else:
        assert torch.equal(summed, (i["x"].float() + i["residual"].float()).to(dtype))
        s = summed.double()
    rows, cols = s.shape
    w = i["weight"].double()
    b = i["bias"].double() if i["bias"] is not None else torch.zeros_like(w)
    mu = s.mean(1, keepdim=True) if layer else torch.zeros_like(s[:, :1])
    sigma = torch.sqrt(((s - mu) ** 2).mean(1, keepdim=True) + eps)
    inv, n = 1 / sigma, (s - mu) / sigma
    ed = (64 * U * s.abs().mean(1, keepdim=True) if layer else 0) + U * (s.abs() + mu.abs())
    ei = 34 * U + torch.sqrt((ed ** 2).mean(1, keepdim=True)) / sigma
    en = ed * inv + n.abs() * (ei + 3 * U)
    want = n * w + b
    _close(y, want, w.abs() * en + 4 * U * ((n * w).abs() + b.abs()) + _half(dtype) * want.abs() * 1.01 + TINY[dtype], "y")
    dy = i["dy"].double()
    v = dy * w
    c1 = (v * n).mean(1, keepdim=True)
    c2 = v.mean(1, keepdim=True) if layer else torch.zeros_like(c1)
    ec1 = (v.abs() * en).mean(1, keepdim=True) + 68 * U * (v * n).abs().mean(1, keepdim=True)
    ec2 = 66 * U * v.abs().mean(1, keepdim=True) if layer else 0
    ds = inv * (v - c2 - n * c1)
    tail = i["dsummed"].double() if i["dsummed"] is not None else torch.zeros_like(ds)
    want = ds + tail
    bound = inv * (3 * U * v.abs() + n.abs() * ec1 + c1.abs() * en + ec2 + 4 * U * ((n * c1).abs() + c2.abs()))
    bound = bound + ei * ds.abs() + 2 * U * (ds.abs() + tail.abs())
    bound = bound * 1.01 + _half(dtype) * (want.abs() + bound) + TINY[dtype]
    _close(got["x"], want, bound, "dx")
    if i["residual"] is not None:
        assert torch.equal(got["residual"], got["x"])
    chain = (rows / 64 + 100) * U
    for name, parts, e in (("weight", dy * n, (dy.abs() * en).sum(0)), ("bias", dy, 0)):
        if i[name] is None:
            continue
        assert got[name].dtype == i[name].dtype
        want = parts.sum(0)
        bound = e + chain * parts.abs().sum(0)
        kind = i[name].dtype
        _close(got[name], want, bound + _half(kind) * (want.abs() + bound) + TINY[kind], "d" + name)


SIZES = [(1, 1), (1, 24), (3, 7), (1, 1920), (5, 1152), (130, 1920), (33, 1153), (7, 512), (9, 513), (2, 4099), (4, 8192),
         (3, 8200), (2, 16384), (2, 16392), (2, 20001), (1000, 48), (3001, 100), (2500, 640), (0, 48)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", SIZES)
@pytest.mark.parametrize("layer", [False, True])
@pytest.mark.parametrize("residual", [True, False])
def test_norm_and_gradients(m, dtype, rows, cols, layer, residual):
    _check(m, _inputs(rows, cols, dtype, residual, layer), layer)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1000, 1), (5001, 2), (700, 5), (70003, 8), (333, 9), (2050, 16), (30, 17), (50001, 64),
                                       (777, 65), (1001, 127), (20000, 128), (900, 129), (901, 256), (500, 257), (601, 500)])
@pytest.mark.parametrize("layer", [False, True])
def test_narrow_rows(m, dtype, rows, cols, layer):
    """Several rows a warp, as the norms of a model's heads have them."""
    _check(m, _inputs(rows, cols, dtype, cols % 2 == 0, layer), layer)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1024, 513), (1025, 1153), (1500, 1930), (1111, 4100), (1060, 6947), (1030, 8198),
                                       (1026, 16383)])
@pytest.mark.parametrize("layer", [False, True])
def test_many_rows_off_16_bytes(m, dtype, rows, cols, layer):
    """Rows at every offset come through the ring, the first and the last by themselves; what lies around the outputs stays."""
    i = _inputs(rows, cols, dtype, cols % 2 == 1, layer)
    _check(m, i, layer)
    for off in (1, 3):
        for pitch in (cols, cols + 5):
            j = dict(i)
            for k in ("x", "residual", "dy", "dsummed"):
                if i[k] is None:
                    continue
                flat = torch.full((rows * pitch + 8,), float("nan"), device="cuda", dtype=dtype)
                j[k] = flat[off:off + rows * pitch].view(rows, pitch)[:, :cols]
                j[k].copy_(i[k])
            a, b = _run(m, i, layer), _run(m, j, layer)
            assert torch.equal(a[0], b[0]) and all(torch.equal(a[2][k], b[2][k]) for k in ("x",))
            for k in a[2]:
                assert bool(torch.isfinite(b[2][k]).all())


def test_outputs_off_16_bytes_leave_their_surroundings(m, lib):
    """Through the C entry, where outputs may lie anywhere."""
    from pollux_b200 import _native as N
    rows, cols = 1300, 1153
    i = _inputs(rows, cols, torch.bfloat16, True, True)
    want = _run(m, i, True)
    stream = torch.cuda.current_stream().cuda_stream
    for off in range(1, 9):
        y, s, dx = (torch.full((rows * cols + 16,), 7.0, device="cuda", dtype=torch.bfloat16) for _ in range(3))
        stats = torch.empty(2 * rows, device="cuda")
        at = 2 * off
        N.check(lib.h24_add_norm(i["x"].data_ptr(), i["residual"].data_ptr(), i["weight"].data_ptr(), i["bias"].data_ptr(),
                                 N.DTYPE_BF16, 1, rows, cols, cols, cols, N.DTYPE_BF16, 1e-5, y.data_ptr() + at,
                                 s.data_ptr() + at, stats.data_ptr(), stream), "norm")
        N.check(lib.h24_add_norm_backward(s.data_ptr() + at, i["weight"].data_ptr(), N.DTYPE_BF16, 1, rows, cols, cols,
                                          N.DTYPE_BF16, stats.data_ptr(), i["dy"].data_ptr(), cols, i["dsummed"].data_ptr(),
                                          cols, dx.data_ptr() + at, None, None, stream), "back")
        for t, w in ((y, want[0]), (s, want[1]), (dx, want[2]["x"])):
            assert torch.equal(t[off:off + rows * cols].view(rows, cols), w)
            assert bool((t[:off] == 7).all()) and bool((t[off + rows * cols:] == 7).all())
    N.check(lib.h24_check(stream), "check")


@pytest.mark.parametrize("layer", [False, True])
def test_parameter_types(m, layer):
    for dtype in (torch.bfloat16, torch.float16):
        i = _inputs(40, 1920, dtype, True, layer)
        other = torch.float16 if dtype == torch.bfloat16 else torch.bfloat16
        for wt, bt in ((torch.float32, torch.float32), (dtype, torch.float32), (other, dtype)):
            j = dict(i, weight=i["weight"].to(wt), bias=i["bias"].to(bt) if layer else None)
            _check(m, j, layer)


@pytest.mark.parametrize("dtype", DTYPES)
def test_layer_norm_far_from_zero(m, dtype):
    """A mean a hundred times the spread."""
    i = _inputs(50, 1152, dtype, False, True)
    i["x"] = (i["x"].float() + 100).to(dtype)
    _check(m, i, True)


@pytest.mark.parametrize("layer", [False, True])
def test_without_bias(m, layer):
    i = _inputs(20, 96, torch.bfloat16, True, False)
    _check(m, i, layer)


@pytest.mark.parametrize("cols", [40, 1153, 1920])
@pytest.mark.parametrize("layer", [False, True])
def test_strides_and_shapes(m, cols, layer):
    """Rows with a stride, an offset of one element, a gradient that is expanded, three dimensions."""
    i = _inputs(12, cols, torch.bfloat16, True, layer)
    y, summed, got = _run(m, i, layer)
    wide = {k: torch.zeros(12, cols + 9, dtype=torch.bfloat16, device="cuda")[:, 1:cols + 1] for k in
            ("x", "residual", "dy", "dsummed")}
    for k, t in wide.items():
        t.copy_(i[k])
    y2, summed2, got2 = _run(m, dict(i, **wide), layer)
    assert torch.equal(y, y2) and torch.equal(summed, summed2)
    for k in got:
        assert torch.equal(got[k], got2[k]), k
    flat = dict(i, **{k: i[k].view(3, 4, cols) for k in ("x", "residual", "dy", "dsummed")})
    y3, _, got3 = _run(m, flat, layer)
    assert y3.shape == (3, 4, cols) and torch.equal(y3.view(12, cols), y) and torch.equal(got3["weight"], got["weight"])
    cross = dict(i, x=i["x"].t().contiguous().t(), dy=torch.ones((), device="cuda").bfloat16().expand(12, cols))
    plain = dict(i, dy=torch.ones(12, cols, device="cuda").bfloat16())
    a, b = _run(m, cross, layer), _run(m, plain, layer)
    assert torch.equal(a[0], b[0]) and torch.equal(a[2]["x"], b[2]["x"]) and torch.equal(a[2]["weight"], b[2]["weight"])


@pytest.mark.parametrize("cols", [5, 48, 64, 200, 300, 1920, 20001])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("layer", [False, True])
def test_rows_beyond_the_range_of_squares(m, cols, dtype, layer):
    """Finite rows whose squares pass fp32's range are normed as others; their neighbours' bits do not change, and rows
    with NaN or infinity stay by themselves."""
    i = _inputs(9, cols, dtype, False, layer)
    base = _run(m, i, layer)
    j = dict(i, x=i["x"].clone())
    j["x"][2] = (i["x"][2].double() * 2.0 ** 100).to(dtype)
    j["x"][5] = (i["x"][5].double() * 2.0 ** 124).clamp(-3e38, 3e38).to(dtype)
    j["x"][6, 3] = float("nan")
    j["x"][7, 1] = float("inf")
    y, _, got = _run(m, j, layer)
    for r in (0, 1, 3, 4, 8):
        assert torch.equal(y[r], base[0][r]) and torch.equal(got["x"][r], base[2]["x"][r])
    s = j["x"][[2, 5]].double()
    mu = s.mean(1, keepdim=True) if layer else 0
    n = (s - mu) / torch.sqrt(((s - mu) ** 2).mean(1, keepdim=True) + 1e-5)
    want = n * i["weight"].double() + (i["bias"].double() if layer else 0)
    # y's own rounding is half a step of |y| <= |n w| + |b|, and a bias passes 1.
    size = n.abs() * i["weight"].double().abs() + (i["bias"].double().abs() if layer else 0)
    tol = (_half(dtype) + 300 * U) * (size + 1)
    assert bool(((y[[2, 5]].double() - want).abs() <= tol).all())
    assert bool(y[6].isnan().any()) and bool(y[7].isnan().any())
    # The weight's gradient without the two rows that are not finite.
    keep = [0, 1, 2, 3, 4, 5, 8]
    k = dict(j, x=j["x"][keep], dy=j["dy"][keep])
    _, _, got = _run(m, k, layer)
    s = k["x"].double()
    mu = s.mean(1, keepdim=True) if layer else 0
    n = (s - mu) / torch.sqrt(((s - mu) ** 2).mean(1, keepdim=True) + 1e-5)
    dy = k["dy"].double()
    tol = _half(dtype) * (dy * n).sum(0).abs() + 400 * U * (dy.abs() * (n.abs() + 1)).sum(0)
    assert bool(((got["weight"].double() - (dy * n).sum(0)).abs() <= tol).all())


@pytest.mark.parametrize("layer", [False, True])
def test_rows_of_zeros_and_constants(m, layer):
    i = _inputs(4, 96, torch.float32, True, layer)
    i["x"].zero_()
    i["residual"].zero_()
    i["residual"][1] = 3.0
    _check(m, i, layer, eps=1e-3)


@pytest.mark.parametrize("layer", [False, True])
def test_which_gradients_are_asked(m, layer):
    i = _inputs(33, 200, torch.bfloat16, True, layer)
    _, _, full = _run(m, i, layer)
    names = [k for k in ("x", "residual", "weight", "bias") if i[k] is not None]
    for asked in names:
        j = dict(i)
        j[asked] = i[asked].detach().requires_grad_(True)
        y, summed = _call(m, j, layer, 1e-5)
        (g,) = torch.autograd.grad([y, summed], [j[asked]], [i["dy"], i["dsummed"]])
        assert torch.equal(g, full[asked]), asked
    # Only one of the outputs is used.
    j = dict(i, **{k: i[k].detach().requires_grad_(True) for k in names})
    y, summed = _call(m, j, layer, 1e-5)
    g = torch.autograd.grad(summed, [j[k] for k in names], i["dsummed"], retain_graph=True, allow_unused=True)
    assert torch.equal(g[0], i["dsummed"]) and torch.equal(g[1], i["dsummed"]) and not bool(g[2].any())
    g = torch.autograd.grad(y, [j[k] for k in names], i["dy"])
    want = _run(m, dict(i, dsummed=torch.zeros_like(i["dsummed"])), layer)[2]
    assert all(torch.equal(a, want[k]) for a, k in zip(g, names))
    with torch.no_grad():
        assert not _call(m, j, layer, 1e-5)[0].requires_grad
    with torch.inference_mode():
        assert torch.equal(_call(m, i, layer, 1e-5)[0], y.detach())


@pytest.mark.parametrize("layer", [False, True])
def test_against_differences(m, layer):
    """The gradient of sum(dy y) + sum(dsummed summed) along random directions, in fp32: a central difference with step
    2^-7 has an error of step^2 / 6 times the third derivative (below 2^-13 of a few units here) and of 2^-24 / step of
    the sum."""
    i = _inputs(3, 40, torch.float32, True, layer)
    _, _, got = _run(m, i, layer)
    step = 2.0 ** -7
    for k in got:
        d = torch.randn_like(i[k])

        def f(sign):
            y, s = _call(m, dict(i, **{k: i[k] + sign * step * d}), layer, 1e-5)
            return float((y.double() * i["dy"].double()).sum() + (s.double() * i["dsummed"].double()).sum())
        along = float((got[k].double() * d.double()).sum())
        assert abs((f(1) - f(-1)) / (2 * step) - along) <= 2e-2 * (1 + abs(along)), k


def test_same_bits_every_time(m):
    i = _inputs(2111, 1920, torch.bfloat16, True, True)
    a, b = _run(m, i, True), _run(m, i, True)
    assert torch.equal(a[0], b[0]) and all(torch.equal(a[2][k], b[2][k]) for k in a[2])


def test_in_place_change_is_seen(m):
    x = torch.randn(4, 48, device="cuda", requires_grad=True)
    h = x * 1
    y, _ = m.add_rms_norm(h, torch.ones(48, device="cuda"))
    h.mul_(2)
    with pytest.raises(RuntimeError, match="inplace"):
        y.sum().backward()


@pytest.mark.parametrize("layer", [False, True])
def test_another_stream_and_the_host(m, layer):
    i = _inputs(100, 640, torch.float16, True, layer)
    want = _run(m, i, layer)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = _run(m, i, layer)
    torch.cuda.current_stream().wait_stream(s)
    host = _run(m, {k: None if t is None else t.cpu() for k, t in i.items()}, layer)
    for other in (got, host):
        assert torch.equal(other[0].cuda(), want[0]) and all(torch.equal(other[2][k].cuda(), want[2][k]) for k in want[2])
    assert host[0].device.type == "cpu" and host[2]["weight"].device.type == "cpu"
