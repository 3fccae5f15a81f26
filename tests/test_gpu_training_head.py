"""The norms and the loss of the training head path as they are used: together, on other streams, in CUDA graphs, under
autocast, with masks and values that go wrong elsewhere."""
from __future__ import annotations

import os
import subprocess
import sys

import pytest
import torch

from conftest import REPO

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.fixture(scope="module")
def m(lib):
    from pollux_b200 import loss, norm
    return norm, loss.linear_cross_entropy


def _grads(ce, x, w, t, reduction="mean", dloss=None, **kw):
    x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    value = ce(x, w, t, reduction=reduction, **kw)
    return (value.detach(), *torch.autograd.grad(value, (x, w), dloss))


def _data(tokens=70, vocab=515, k=120, dtype=BF, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(tokens, k, generator=g, device="cuda").to(dtype)
    w = (torch.randn(vocab, k, generator=g, device="cuda") * 0.2).to(dtype)
    return x, w, torch.randint(0, vocab, (tokens,), generator=g, device="cuda")


@pytest.mark.parametrize("tokens", [70, 300])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_masked_rows_hold_anything(m, tokens, reduction):
    """Rows without a loss have no say, whatever stands in them: not in the loss, not in the gradients."""
    x, w, t = _data(tokens)
    t[torch.arange(0, tokens, 3, device="cuda")] = -100
    d = torch.rand(tokens, device="cuda") if reduction == "none" else None
    want = _grads(m[1], x, w, t, reduction, d)
    y = x.clone()
    y[0], y[3], y[6] = float("nan"), float("inf"), torch.finfo(BF).max
    dn = d
    if d is not None:
        dn = d.clone()
        dn[9], dn[12] = float("nan"), float("inf")
    got = _grads(m[1], y, w, t, reduction, dn)
    for a, b in zip(want, got):
        assert torch.equal(a, b) and bool(torch.isfinite(a).all())
    kept = t != -100
    assert not bool(got[1][~kept].any())


@pytest.mark.parametrize("tokens", [1, 5, 130, 600])
def test_no_token_has_a_loss(m, tokens):
    x, w, t = _data(tokens)
    t.fill_(-100)
    for reduction in ("mean", "sum", "none"):
        d = torch.ones(tokens, device="cuda") if reduction == "none" else None
        value, dx, dw = _grads(m[1], x * float("nan"), w, t, reduction, d)
        if reduction == "mean":
            assert bool(value.isnan())
        else:
            assert not bool(value.any())
        assert not bool(dx.any()) and not bool(dw.any())


def test_no_tokens_at_all(m):
    x, w, t = _data()
    x, t = x[:0], t[:0]
    for reduction, want in (("mean", float("nan")), ("sum", 0.0)):
        value, dx, dw = _grads(m[1], x, w, t, reduction)
        assert torch.equal(value.cpu(), torch.tensor(want)) or (want != want and bool(value.isnan()))
        assert dx.shape == x.shape and not bool(dw.any())
    value, dx, dw = _grads(m[1], x, w, t, "none", torch.ones(0, device="cuda"))
    assert value.shape == (0,) and not bool(dw.any())


@pytest.mark.parametrize("tokens", [7, 200])
@pytest.mark.parametrize("bad", [515, -1, 2 ** 40, -2 ** 40])
def test_a_target_outside_the_vocabulary_is_loud(m, tokens, bad):
    x, w, t = _data(tokens)
    want = m[1](x, w, t, reduction="none")
    t[3] = bad
    value, dx, dw = _grads(m[1], x, w, t, "none", torch.ones(tokens, device="cuda"))
    assert bool(value[3].isnan()) and bool(dx[3].isnan().all()) and bool(dw.isnan().all())
    keep = torch.arange(tokens, device="cuda") != 3
    assert torch.equal(value[keep], want[keep]) and bool(torch.isfinite(dx[keep]).all())
    assert bool(m[1](x, w, t).isnan())
    # As an ignored number it is left out.
    assert bool(torch.isfinite(m[1](x, w, t, ignore_index=bad)))


@pytest.mark.parametrize("dtype", [BF, torch.float16])
@pytest.mark.parametrize("tokens", [9, 300])
def test_values_without_a_finite_loss(m, tokens, dtype):
    """A NaN or an infinity in a state or a head's row goes where it goes in torch."""
    x, w, t = _data(tokens, dtype=dtype)
    base = m[1](x, w, t, reduction="none")
    y = x.clone()
    y[2, 5], y[4] = float("nan"), float("inf")
    got = m[1](y, w, t, reduction="none")
    keep = torch.ones(tokens, dtype=torch.bool, device="cuda")
    keep[[2, 4]] = False
    assert torch.equal(got[keep], base[keep]) and bool(got[2].isnan())
    ref = torch.nn.functional.cross_entropy(y.double() @ w.double().t(), t, reduction="none")
    assert bool(got[4].isnan()) == bool(ref[4].isnan())
    v = w.clone()
    v[7, 0] = float("nan")
    assert bool(m[1](x, v, t, reduction="none").isnan().all())


def test_large_logits(m):
    """Logits of +-3000: the probabilities are 0 and 1, the losses differences of logits."""
    x, w, t = _data(40, 300, 64)
    x = x * 120
    value, dx, dw = _grads(m[1], x, w, t, "none", torch.ones(40, device="cuda"))
    z = x.double() @ w.double().t()
    want = torch.logsumexp(z, 1) - z.gather(1, t[:, None])[:, 0]
    assert bool(((value.double() - want).abs() <= 1e-5 * z.abs().amax(1)).all())
    assert bool(torch.isfinite(dx).all()) and bool(torch.isfinite(dw).all())


@pytest.mark.parametrize("tokens", [33, 400])
def test_strides_shapes_and_types_of_targets(m, tokens):
    x, w, t = _data(tokens, 515, 120)
    want = _grads(m[1], x, w, t, "none", torch.ones(tokens, device="cuda"))
    wide = torch.full((tokens, 133), float("nan"), device="cuda", dtype=BF)[:, 3:123]
    wide.copy_(x)
    tall = torch.full((515, 131), float("nan"), device="cuda", dtype=BF)[:, 1:121]
    tall.copy_(w)
    got = _grads(m[1], wide, tall, t.to(torch.int32), "none", torch.ones((), device="cuda").expand(tokens))
    for a, b in zip(want, got):
        assert torch.equal(a, b)
    across = _grads(m[1], x.t().contiguous().t(), w.t().contiguous().t(), t[:, None].expand(tokens, 2)[:, 0], "none",
                    torch.ones(2 * tokens, device="cuda")[::2])
    for a, b in zip(want, across):
        assert torch.equal(a, b)
    if tokens % 4 == 0:
        value, dx, dw = _grads(m[1], x.view(4, tokens // 4, 120), w, t.view(4, -1), "none",
                               torch.ones(4, tokens // 4, device="cuda"))
        assert value.shape == (4, tokens // 4) and dx.shape == (4, tokens // 4, 120)
        assert torch.equal(value.view(-1), want[0]) and torch.equal(dx.view(tokens, 120), want[1])
        assert torch.equal(dw, want[2])


def test_a_head_off_its_alignment(m):
    """Rows on 2, 4 and 8 bytes, dW at any address: the same values as on 16 bytes with zeros behind."""
    for k in (113, 114, 116, 120, 127):
        for tokens in (20, 150):
            x, w, t = _data(tokens, 260, k)
            value, dx, dw = _grads(m[1], x, w, t)
            xp = torch.zeros(tokens, 128, device="cuda", dtype=BF)
            wp = torch.zeros(260, 128, device="cuda", dtype=BF)
            xp[:, :k], wp[:, :k] = x, w
            v2, dx2, dw2 = _grads(m[1], xp, wp, t)
            assert torch.equal(value, v2) and torch.equal(dx, dx2[:, :k]) and torch.equal(dw, dw2[:, :k])


@pytest.mark.parametrize("tokens", [60, 500])
def test_which_gradients_are_asked(m, tokens):
    x, w, t = _data(tokens)
    _, dx, dw = _grads(m[1], x, w, t)
    xs = x.detach().requires_grad_(True)
    (g,) = torch.autograd.grad(m[1](xs, w, t), xs)
    # (The sum over the vocabulary may be cut into other slices when dW is not wanted.)
    assert bool(((g.double() - dx.double()).abs() <= 2.0 ** -7 * dx.double().abs() + 1e-6).all())
    ws = w.detach().requires_grad_(True)
    (g,) = torch.autograd.grad(m[1](x, ws, t), ws)
    assert torch.equal(g, dw)
    assert not m[1](x, w, t).requires_grad
    with torch.no_grad():
        assert not m[1](xs, ws, t).requires_grad
    with torch.inference_mode():
        assert torch.equal(m[1](x, w, t), m[1](xs, ws, t))


def test_same_bits_every_time(m):
    for tokens, vocab, k in ((100, 5000, 200), (700, 5000, 200), (2000, 40000, 64)):
        x, w, t = _data(tokens, vocab, k)
        a = _grads(m[1], x, w, t)
        for _ in range(3):
            assert all(torch.equal(p, q) for p, q in zip(a, _grads(m[1], x, w, t)))


def test_second_derivatives_are_refused(m):
    x, w, t = _data(30)
    x.requires_grad_(True)
    (g,) = torch.autograd.grad(m[1](x, w, t), x, create_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        g.float().square().sum().backward()
    y, _ = m[0].add_rms_norm(x, torch.ones(120, device="cuda", dtype=BF))
    (g,) = torch.autograd.grad(y.float().square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        g.float().square().sum().backward()


def test_an_input_that_changed_is_noticed(m):
    x, w, t = _data(30)
    h = x.detach().requires_grad_(True) * 1
    value = m[1](h, w.requires_grad_(True), t)
    with torch.no_grad():
        h.mul_(2)
    with pytest.raises(RuntimeError, match="inplace"):
        value.backward()


def test_against_differences(m):
    """Along random directions, in fp16 with a large step: the loss's gradients against central differences.  The
    directions' steps of 2^-6 are exact multiples of what fp16 holds only to 2^-11 of each element, which changes the
    difference by that much of sum|g d|; third derivatives along them are below 1."""
    x, w, t = _data(40, 90, 64, torch.float16)
    _, dx, dw = _grads(m[1], x, w, t, "sum")
    for leaf, g in ((0, dx), (1, dw)):
        d = torch.randn_like((x, w)[leaf]) * 0.25
        step = 2.0 ** -4

        def f(sign):
            a = [x, w]
            moved = (a[leaf].float() + sign * step * d.float()).half()
            a[leaf] = moved
            return float(m[1](a[0], a[1], t, reduction="sum")), moved.double()
        (up, pu), (down, pd) = f(1), f(-1)
        along = float((g.double() * (pu - pd)).sum())  # what was really moved
        assert abs((up - down) - along) <= 2e-2 * float((g.double() * (pu - pd)).abs().sum()) + 1e-3


@pytest.mark.parametrize("dtype", [BF, torch.float16])
def test_autocast(m, dtype):
    x, w, t = _data(50)
    xf, wf = x.float().requires_grad_(True), w.float().requires_grad_(True)
    with torch.autocast("cuda", dtype=dtype):
        value = m[1](xf, wf, t)
    dx, dw = torch.autograd.grad(value, (xf, wf))
    assert value.dtype == torch.float32 and dx.dtype == torch.float32 and dw.dtype == torch.float32
    v2, dx2, dw2 = _grads(m[1], x.to(dtype), w.to(dtype), t)
    assert torch.equal(value.detach(), v2) and torch.equal(dx, dx2.float()) and torch.equal(dw, dw2.float())
    with pytest.raises(TypeError, match="float16"):
        m[1](xf, wf, t)


def test_tensors_on_the_host(m):
    x, w, t = _data(50)
    want = _grads(m[1], x, w, t)
    got = _grads(m[1], x.cpu(), w.cpu(), t.cpu())
    assert all(g.device.type == "cpu" and torch.equal(g.cuda(), v) for g, v in zip(got, want))


def _step(m, x, r, gain, w, t):
    y, summed = m[0].add_rms_norm(x, gain, residual=r)
    return m[1](y, w, t) + summed.float().square().mean()


@pytest.mark.parametrize("tokens,vocab,k", [(64, 600, 240), (600, 5000, 240)])
def test_norm_and_loss_together(m, tokens, vocab, k):
    """The end of a training step against the same in 64 bits with the roundings in its places: the norm's output and its
    gradient are rounded to bf16 once each (2^-8 of themselves), the products' operands once."""
    g = torch.Generator(device="cuda").manual_seed(1)
    x, r = (torch.randn(tokens, k, generator=g, device="cuda").to(BF) for _ in range(2))
    gain = (1 + 0.2 * torch.randn(k, generator=g, device="cuda")).to(BF)
    w = (torch.randn(vocab, k, generator=g, device="cuda") * 0.1).to(BF)
    t = torch.randint(0, vocab, (tokens,), generator=g, device="cuda")
    t[::5] = -100
    leaves = [a.detach().requires_grad_(True) for a in (x, r, gain, w)]
    value = _step(m, *leaves, t)
    got = torch.autograd.grad(value, leaves)
    ref = [a.detach().double().requires_grad_(True) for a in (x, r, gain, w)]
    s = (x.float() + r.float()).to(BF).double() + (ref[0] + ref[1] - (ref[0] + ref[1]).detach())
    y = s / torch.sqrt((s * s).mean(1, keepdim=True) + 1e-6) * ref[2]
    want = torch.nn.functional.cross_entropy(y @ ref[3].t(), t) + s.square().mean()
    assert abs(float(value.detach()) - float(want.detach())) <= 2.0 ** -8 * (1 + abs(float(want.detach())))
    for a, b in zip(got, torch.autograd.grad(want, ref)):
        assert float((a.double() - b).norm()) <= 4 * 2.0 ** -8 * float(b.norm())


@pytest.mark.parametrize("tokens,vocab,k", [(40, 700, 120), (300, 3000, 113), (1500, 40000, 64)])
def test_captured_and_replayed(m, tokens, vocab, k):
    """Two captured steps, backward and all, with new values replayed in turn: they share no scratch."""
    x, w, t = _data(tokens, vocab, k)
    r, gain = torch.randn_like(x), torch.ones(k, device="cuda", dtype=BF)
    leaves = [a.detach().requires_grad_(True) for a in (x, r, gain, w)]

    def step():
        value = _step(m, *leaves, t)
        return (value, *torch.autograd.grad(value, leaves))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    with torch.cuda.graph(other):
        out2 = step()
    for seed in range(3):
        with torch.no_grad():
            for a in leaves:
                a.copy_(torch.randn(a.shape, device="cuda") * 0.3)
            t.random_(0, vocab)
            t[seed::4] = -100
        for g in (graph, other, graph):
            g.replay()
        want = step()
        for a, b, c in zip(out, out2, want):
            assert torch.equal(a, c) and torch.equal(b, c)
    torch.cuda.synchronize()


def test_two_streams_at_once(m):
    """Calls that overlap on two streams do not share scratch."""
    data = [_data(500, 4000, 200, seed=s) for s in range(2)]
    want = [_grads(m[1], *d) for d in data]
    streams = [torch.cuda.Stream() for _ in data]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, (s, d) in enumerate(zip(streams, data)):
            with torch.cuda.stream(s):
                got[i].append(_grads(m[1], *d))
    torch.cuda.synchronize()
    for i in range(2):
        for g in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(g, want[i]))


def test_without_the_torch_module(m):
    """The general path makes the same calls."""
    from pollux_b200 import _native as N
    x, w, t = _data(150, 900, 96)
    r, gain, bias = torch.randn_like(x), torch.ones(96, device="cuda", dtype=BF), torch.zeros(96, device="cuda", dtype=BF)

    def everything():
        out = list(_grads(m[1], x, w, t)) + list(_grads(m[1], x, w, t, "none", torch.ones(150, device="cuda")))
        a = [p.detach().requires_grad_(True) for p in (x, r, gain, bias)]
        for (y, s), asked in ((m[0].add_rms_norm(a[0], a[2], residual=a[1]), a[:3]),
                              (m[0].add_layer_norm(a[0], a[2], a[3], residual=a[1]), a)):
            out += [y.detach(), s.detach(), *torch.autograd.grad((y, s), asked, (x, r))]
        return out
    want = everything()
    fast, N._torch_calls = N._torch_calls, N._GeneralPath()
    try:
        got = everything()
    finally:
        N._torch_calls = fast
    assert len(got) == len(want) and all(torch.equal(a, b) for a, b in zip(got, want))


def test_states_beyond_32_bits(m):
    """A head of more than 2^31 elements, and dW's rows behind that."""
    free, _ = torch.cuda.mem_get_info()
    if free < 40 << 30:
        pytest.skip("needs 40 GB")
    vocab, k, tokens = 1_100_000, 2048, 6
    w = torch.zeros(vocab, k, device="cuda", dtype=BF)
    g = torch.Generator(device="cuda").manual_seed(3)
    rows = torch.tensor([5, 1_048_700, 1_099_999, 1_048_575, 77, 1_050_000], device="cuda")
    w[rows] = torch.randn(6, k, generator=g, device="cuda").to(BF)
    x = (torch.randn(tokens, k, generator=g, device="cuda") * 0.3).to(BF)
    value, dx, dw = _grads(m[1], x, w, rows, "none", torch.ones(tokens, device="cuda"))
    z = x.double() @ w[rows].double().t()
    lse = torch.log(torch.exp(z).sum(1) + (vocab - 6))
    assert bool(((value.double() - (lse - z.diag())).abs() <= 1e-4).all())
    p = torch.exp(z - lse[:, None]) - torch.eye(6, device="cuda")
    want = p.t() @ x.double()
    assert bool(((dw[rows].double() - want).abs() <= 2.0 ** -7 * (p.abs().t() @ x.double().abs()) + 1e-6).all())
    del w, dw


CODE = """
import sys, torch
sys.path.insert(0, {repo!r})
from pollux_b200 import norm, loss
tokens = {tokens}
x = torch.randn(tokens, 96, device="cuda", dtype=torch.bfloat16)
w = torch.randn(700, 96, device="cuda", dtype=torch.bfloat16) * 0.2
g = torch.ones(96, device="cuda", dtype=torch.bfloat16)
t = torch.randint(0, 700, (tokens,), device="cuda")
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    y, _ = norm.add_rms_norm(x, g)
    z = loss.linear_cross_entropy(y, w, t, reduction="none")
for _ in range(2):
    x.normal_()
    graph.replay()
    assert torch.equal(z, loss.linear_cross_entropy(norm.add_rms_norm(x, g)[0], w, t, reduction="none"))
torch.cuda.synchronize()
print("captured")
"""


@pytest.mark.parametrize("tokens", [3, 500])
def test_first_call_inside_a_capture(lib, tokens):
    r = subprocess.run([sys.executable, "-c", CODE.format(repo=REPO, tokens=tokens)],
                       capture_output=True, text=True, timeout=300, cwd=os.path.dirname(REPO))
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


ALIVE = """
import sys, torch
sys.path.insert(0, {repo!r})
from pollux_b200 import norm, loss
def leaf(*shape):
    return (torch.randn(*shape, device="cuda") * 0.3).bfloat16().requires_grad_(True)
x, g, w = leaf(300, 96), leaf(96), leaf(700, 96)
t = torch.randint(0, 700, (300,), device="cuda")
def step():
    y, s = norm.add_rms_norm(x, g, residual=x)
    value = loss.linear_cross_entropy(y, w, t) + s.float().mean()
    return torch.autograd.grad(value, (x, g, w))
want = step()
y, _ = norm.add_rms_norm(x, g)
alive = loss.linear_cross_entropy(y, w, t)
side = torch.cuda.Stream()
side.wait_stream(torch.cuda.current_stream())
try:
    with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
        step()
    print("captured")
except RuntimeError as e:
    print("refused", type(e).__name__)
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(step(), want))
alive.backward()
assert bool(torch.isfinite(w.grad).all())
print("goes on")
"""


def test_a_capture_beside_a_live_eager_graph_does_not_end_the_process(lib):
    """torch ties a leaf's accumulator to the stream of the graph that lives, and a captured backward pass that meets it is
    refused; the process goes on."""
    r = subprocess.run([sys.executable, "-c", ALIVE.format(repo=REPO)], capture_output=True, text=True, timeout=300,
                       cwd=os.path.dirname(REPO))
    assert r.returncode == 0 and "goes on" in r.stdout, r.stdout + r.stderr[-2000:]
