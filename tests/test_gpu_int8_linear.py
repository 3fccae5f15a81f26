"""int8.int8_linear against the product in 64 bits.

The int32 sum is exact, so y = fl(fl(fl(acc) * scale * ws) + b): four fp32
roundings (u = 2^-24) of the product and the sum, then one to the output type."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
OUT = {torch.float32: (2.0 ** -24, 2.0 ** -150), torch.float16: (2.0 ** -11, 2.0 ** -25),
       torch.bfloat16: (2.0 ** -8, 2.0 ** -134)}  # rounding, half the smallest step


@pytest.fixture(scope="module")
def m(lib):
    from pollux_b200 import int8
    return int8


def _inputs(tokens, out_f, in_f, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = torch.randint(-128, 128, (tokens, in_f), generator=g, device="cuda", dtype=torch.int8)
    w = torch.randint(-128, 128, (out_f, in_f), generator=g, device="cuda", dtype=torch.int8)
    scale = torch.rand(tokens, generator=g, device="cuda") * 0.05
    mu = (torch.rand(out_f, generator=g, device="cuda") * 0.2 + 0.01).half()
    b = torch.randn(out_f, generator=g, device="cuda")
    return q, scale, w, mu, b


def _check(y, q, scale, w, mu, b):
    acc = torch.matmul(q.double(), w.double().t()) if q.shape[1] else torch.zeros(y.shape, device="cuda", dtype=torch.float64)
    prod = acc * scale.double()[:, None] * (mu.float() / 127).half().double()[None]
    want = prod + (b.double()[None] if b is not None else 0)
    rel, step = OUT[y.dtype]
    tol = U * (4 * prod.abs() + want.abs()) * 1.01 + rel * want.abs() * 1.01 + step
    bad = (y.double() - want).abs() > tol
    assert not bad.any(), (int(bad.sum()), torch.nonzero(bad)[:4].tolist())


SHAPES = [(1, 1, 1), (1, 1152, 1152), (1, 50688, 1920), (2, 130, 48), (3, 257, 1921), (7, 1920, 7680), (16, 384, 128),
          (17, 129, 127), (31, 1000, 24), (32, 7680, 1920), (33, 1152, 4608), (64, 1920, 1920), (65, 128, 256),
          (100, 333, 777), (128, 1152, 1152), (129, 640, 1000), (200, 96, 20016), (255, 7680, 1920), (256, 256, 128),
          (257, 257, 272), (300, 1920, 7680), (511, 2000, 1152), (1024, 1920, 1920), (1500, 5000, 240), (2048, 7680, 1920),
          (5000, 24, 24)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("tokens,out_f,in_f", SHAPES)
def test_matches_exact(m, tokens, out_f, in_f, dtype):
    q, scale, w, mu, b = _inputs(tokens, out_f, in_f, tokens * 7 + out_f + in_f)
    if dtype == torch.float16:
        scale = scale / max(1, in_f) ** 0.5 / 50  # within fp16's range
    _check(m.int8_linear(q, scale, w, mu, None, dtype), q, scale, w, mu, None)
    _check(m.int8_linear(q, scale, w, mu, b, dtype), q, scale, w, mu, b)


def test_largest_sums_do_not_overflow(m):
    q = torch.full((3, 131000), -128, device="cuda", dtype=torch.int8)
    w = torch.full((130, 131000), -128, device="cuda", dtype=torch.int8)
    w[5:9] = 127
    scale, mu = torch.ones(3, device="cuda"), torch.full((130,), 127.0, device="cuda").half()
    _check(m.int8_linear(q, scale, w, mu), q, scale, w, mu, None)


def test_strides_and_shapes(m):
    q, scale, w, mu, b = _inputs(40, 300, 480, 3)
    want = m.int8_linear(q, scale, w, mu, b)
    wide = torch.zeros(40, 1024, device="cuda", dtype=torch.int8)
    for off, pitch in ((0, 1024), (16, 1024), (3, 1024), (1, 997)):
        v = wide.view(-1)[: 40 * pitch].view(40, pitch)[:, off:off + 480]
        v.copy_(q)
        assert torch.equal(m.int8_linear(v, scale, w, mu, b), want)
    assert torch.equal(m.int8_linear(q.t().contiguous().t(), scale, w, mu, b), want)
    assert torch.equal(m.int8_linear(q.view(4, 10, 480), scale.view(4, 10), w, mu, b), want.view(4, 10, 300))
    assert torch.equal(m.int8_linear(q[3], scale[3], w, mu, b), want[3])
    rows = q[:1].expand(40, 480)
    assert torch.equal(m.int8_linear(rows, scale, w, mu, b), m.int8_linear(rows.contiguous(), scale, w, mu, b))
    # A weight that starts off a 16-byte boundary, and one given by columns.
    raw = torch.empty(300 * 480 + 1, device="cuda", dtype=torch.int8)
    raw[1:].copy_(w.view(-1))
    assert torch.equal(m.int8_linear(q, scale, raw[1:].view(300, 480), mu, b), want)
    assert torch.equal(m.int8_linear(q, scale, w.t().contiguous().t(), mu, b), want)


def test_empty_sizes_and_host_tensors(m):
    q, scale, w, mu, b = _inputs(4, 50, 96, 8)
    assert m.int8_linear(q[:0], scale[:0], w, mu, b).shape == (0, 50)
    assert m.int8_linear(q, scale, w[:0], mu[:0]).shape == (4, 0)
    y = m.int8_linear(q[:, :0], scale, w[:, :0], mu, b)
    assert torch.equal(y, b.expand(4, 50))
    assert (m.int8_linear(q[:, :0], scale, w[:, :0], mu) == 0).all()
    y = m.int8_linear(q.cpu(), scale.cpu(), w.cpu(), mu.cpu(), b.cpu())
    assert y.device.type == "cpu" and torch.equal(y, m.int8_linear(q, scale, w, mu, b).cpu())


def test_rows_do_not_depend_on_the_batch(m):
    """The exact sum makes a token's outputs the same whatever the split."""
    q, scale, w, mu, b = _inputs(700, 1920, 1920, 12)
    want = m.int8_linear(q, scale, w, mu, b)
    for n in (1, 5, 16, 64, 200, 333):
        assert torch.equal(m.int8_linear(q[:n], scale[:n], w, mu, b), want[:n])


def test_special_scales(m):
    q, scale, w, mu, b = _inputs(5, 70, 96, 4)
    scale[1], scale[2], mu[3] = float("nan"), 0.0, float("inf")
    y = m.int8_linear(q, scale, w, mu, b)
    assert torch.isnan(y[1]).all()
    keep = torch.arange(70, device="cuda") != 3
    assert torch.equal(y[2][keep], b[keep])
    assert not torch.isfinite(y[:, 3]).any()


def test_streams_and_many_calls(m):
    """Calls of different sizes on two streams at once."""
    sets = [_inputs(t, o, k, t) for t, o, k in ((1, 5000, 1920), (300, 1920, 1920), (20, 640, 7680), (900, 2000, 480))]
    want = [m.int8_linear(*s) for s in sets]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
    got = []
    for i in range(24):
        with torch.cuda.stream(streams[i % 2]):
            got.append((i % 4, m.int8_linear(*sets[i % 4])))
    torch.cuda.synchronize()
    from pollux_b200 import castor
    castor.device_check(torch.device("cuda", 0))
    assert all(torch.equal(y, want[i]) for i, y in got)


def test_head_without_materialize(m):
    """enable_int8_forward against the materialised layer: the input's row
    quantisation is the only difference, at most half a step of each element."""
    from pollux_b200 import packed_linear as pl, pack
    lin = pl.PackedInt8Linear(480, 1000).cuda()
    wq, mu = pack.quantize_int8_device(torch.randn(1000, 480, device="cuda") * 0.02)
    lin.weight_int8.copy_(wq)
    lin.mu_rows.copy_(mu)
    x = torch.randn(2, 9, 480, device="cuda", dtype=torch.bfloat16)
    assert m.enable_int8_forward(torch.nn.Sequential(lin)) == 1
    y = lin(x)
    assert y.shape == (2, 9, 1000) and y.dtype == torch.bfloat16
    w = wq.double() * (mu.float() / 127).half().double()[:, None]
    q, s = m.quantize_rows_int8(x)
    bound = 0.5 * s.double()[..., None] * w.abs().sum(1) * 1.001
    want = torch.matmul(x.double(), w.t())
    assert ((y.double() - want).abs() <= bound + want.abs() * 2.0 ** -8 + 1e-6).all()
    lin.materialize()
    assert torch.equal(lin(x), torch.nn.functional.linear(x, lin.weight.to(x.dtype)))


def test_offsets_beyond_32_bits(m):
    """An output of 2.5e9 elements, and input rows 1.5e9 bytes apart."""
    q, scale, w, mu, b = _inputs(50000, 50688, 32, 6)
    scale = scale / 100
    y = m.int8_linear(q, scale, w, mu, b, torch.bfloat16)
    for rows in (slice(0, 3), slice(24990, 24994), slice(49997, 50000)):
        _check(y[rows], q[rows], scale[rows], w, mu, b)
    del y
    base = torch.empty(4_500_000_100, device="cuda", dtype=torch.int8)
    for tokens in (3, 4):
        for k in (96, 93):
            v = base.as_strided((tokens, k), (1_500_000_000, 1))[:3]
            v.copy_(q[:3].repeat(1, 3)[:, :k])
            w2, s2 = w[:300].repeat(1, 3)[:, :k].contiguous(), scale[:3]
            assert torch.equal(m.int8_linear(v, s2, w2, mu[:300]), m.int8_linear(v.contiguous(), s2, w2, mu[:300]))
    del base
    base = torch.empty(4_500_000_100, device="cuda", dtype=torch.int8)
    v = base.as_strided((6, 96), (800_000_000, 1))
    v.copy_(q[:6].repeat(1, 3))
    w2 = w[:300].repeat(1, 3)
    assert torch.equal(m.int8_linear(v, scale[:6], w2, mu[:300]), m.int8_linear(v.contiguous(), scale[:6], w2, mu[:300]))


@pytest.mark.parametrize("tokens,in_f", [(1, 1920), (3, 333), (40, 480), (40, 333), (700, 1001)])
def test_in_a_graph(m, tokens, in_f):
    """Every path, the copy of unaligned rows among them, captured and replayed on new inputs in place."""
    q, scale, w, mu, b = _inputs(tokens, 1000, in_f, 21)
    m.int8_linear(q, scale, w, mu, b)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = m.int8_linear(q, scale, w, mu, b)
    for seed in (1, 2):
        for dst, src in zip((q, scale, w, mu, b), _inputs(tokens, 1000, in_f, seed)):
            dst.copy_(src)
        graph.replay()
        _check(y, q, scale, w, mu, b)


@pytest.mark.parametrize("tokens", [1, 5, 300, 3000])
def test_empty_sum(m, tokens):
    """in_features 0 in every size that would take another path: the bias, or zeros, after a call that left sums in TMEM."""
    full = _inputs(tokens, 50688, 128, 3)
    m.int8_linear(*full, torch.bfloat16)
    q, scale, w, mu, b = full
    y = m.int8_linear(q[:, :0], scale, w[:, :0], mu, b, torch.bfloat16)
    assert torch.equal(y, b.to(torch.bfloat16).expand(tokens, 50688))
    assert (m.int8_linear(q[:, :0], scale, w[:, :0], mu, None, torch.float16) == 0).all()
