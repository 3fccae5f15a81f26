"""sampling.sample_tokens against its definition in 64 bits.

The scaled logits z are two fp32 roundings that numpy repeats; CUDA's expf is
within 2 ulp, so a weight, a mass and a limit are within 2^-21 of the exact
ones.  A token is right if it is the definition's token for limits moved by at
most that: the check tries the limits of the two cuts at both ends and accepts
a running mass that meets the target within it."""
from __future__ import annotations

import itertools

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DELTA = 2.0 ** -21
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def m(lib):
    from pollux_b200 import sampling
    return sampling


def _valid(logits, u, token, t, k, p, min_p):
    """Whether `token` is right for one row (logits: fp32 numpy), and its log-probability."""
    v = logits.size
    l = np.where(np.isnan(logits), -np.inf, logits).astype(np.float32)
    if not t > 0:
        t, k = 1.0, 1
    mx = l.max()
    if mx == -np.inf:
        return token == -1, -np.inf
    with np.errstate(invalid="ignore", over="ignore"):
        z = np.where(l == mx, np.float32(0), (l - mx) * (np.float32(1) / np.float32(t))).astype(np.float32)
    w = np.rint(np.exp(z.astype(np.float64)) * 2.0 ** 40)
    order = np.lexsort((np.arange(v), -z.astype(np.float64)))
    if not 0 < k < v:
        k = v
    if not 0 <= token < v:
        return False, 0.0
    logprob = float(z[token]) - float(np.log(w.sum() / 2.0 ** 40))
    top = order[:k]
    wt = w[top]
    before = np.cumsum(wt) - wt
    p, min_p = float(np.float32(p)), float(np.float32(min_p))
    for a, b in itertools.product((1 - DELTA, 1.0, 1 + DELTA), repeat=2):
        keep = np.ones(k, bool) if p >= 1 else before < max(1.0, p * wt.sum() * a)
        keep &= wt >= max(1.0, min(max(min_p, 0), 1) * 2.0 ** 40 * b if min_p < 1 else 2.0 ** 40)
        kept = np.zeros(v)
        kept[top[keep]] = wt[keep]
        mass = kept.sum()
        uu = float(np.float32(u)) if u > 0 else 0.0
        target = min(np.floor(uu * mass), mass - 1)
        c = np.cumsum(kept)
        slack = DELTA * mass
        if kept[token] > 0 and c[token] > target - slack and c[token] - kept[token] <= target + slack:
            return True, logprob
    return False, logprob


def _check(m, logits, u, **kw):
    tok, lp = m.sample_tokens(logits, u, return_logprob=True, **kw)
    assert tok.dtype == torch.int64 and lp.dtype == torch.float32
    assert torch.equal(m.sample_tokens(logits, u, **kw), tok)
    rows = logits.shape[0]
    col = {n: (v.cpu().numpy() if isinstance(v, torch.Tensor) else [v] * rows)
           for n, v in dict(dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0), **kw).items()}
    ln, un = logits.float().cpu().numpy(), u.cpu().numpy()
    for r in range(rows):
        ok, want = _valid(ln[r], un[r], int(tok[r]), float(col["temperature"][r]), int(col["top_k"][r]),
                          float(col["top_p"][r]), float(col["min_p"][r]))
        assert ok, (r, int(tok[r]), {n: col[n][r] for n in col})
        got = float(lp[r])
        assert got == want or abs(got - want) <= 2.0 ** -20 * (1 + abs(want)), (r, got, want)
    return tok


def _logits(rows, vocab, seed, dtype=torch.float32, spread=3.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(rows, vocab, generator=g, device="cuda") * spread).to(dtype), \
        torch.rand(rows, generator=g, device="cuda")


SETTINGS = [dict(), dict(top_k=1), dict(top_k=50), dict(top_p=0.9), dict(top_k=40, top_p=0.8),
            dict(min_p=0.05), dict(temperature=0.7, top_k=20, top_p=0.95, min_p=0.02), dict(temperature=0.0),
            dict(temperature=2.5, top_p=0.999), dict(top_p=0.0), dict(min_p=1.0), dict(top_k=10 ** 6),
            dict(temperature=1e-30), dict(temperature=1e30, top_k=3)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kw", SETTINGS, ids=lambda k: "-".join(f"{a}{b}" for a, b in k.items()) or "plain")
def test_settings(m, kw, dtype):
    logits, u = _logits(9, 5003, 17, dtype)
    _check(m, logits, u, **kw)


@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (5, 31), (2, 32), (4, 33), (2, 255), (7, 1000), (3, 1024),
                                        (1, 4097), (2, 50304), (1, 50688), (70, 50688), (2, 131072), (1, 262151),
                                        (150, 3001), (300, 640), (1, 600001)])
def test_sizes(m, rows, vocab):
    for dtype, kw in ((torch.float32, dict(top_k=50, top_p=0.9, temperature=0.8)), (torch.bfloat16, dict(top_p=0.95)),
                      (torch.float16, dict(min_p=0.01, top_k=100))):
        logits, u = _logits(rows, vocab, rows + vocab, dtype)
        if rows > 16:  # the 64-bit check is a row at a time
            tok = m.sample_tokens(logits, u, **kw)
            pick = torch.arange(0, rows, rows // 8)
            assert torch.equal(_check(m, logits[pick], u[pick], **kw), tok[pick])
        else:
            _check(m, logits, u, **kw)


@pytest.mark.parametrize("vocab", [50, 4000, 50688])
@pytest.mark.parametrize("kw", [dict(), dict(top_k=7), dict(top_p=0.3), dict(top_k=33, top_p=0.5), dict(min_p=0.5)],
                         ids=str)
def test_ties_go_to_the_lowest_index(m, vocab, kw):
    rows = torch.stack([torch.zeros(vocab, device="cuda"), torch.arange(vocab, device="cuda") % 3 * 1.0,
                        (torch.arange(vocab, device="cuda") == vocab - 2) * 5.0])
    for u in (0.0, 0.25, 0.999):
        _check(m, rows, torch.full((3,), u, device="cuda"), **kw)
    # All equal: exactly the first k are kept, so u picks among them.
    tok = m.sample_tokens(rows[:1].expand(64, vocab), torch.arange(64, device="cuda") / 64.0, top_k=8)
    assert torch.equal(tok, torch.arange(64, device="cuda") // 8)


@pytest.mark.parametrize("vocab", [3, 100, 5003, 50688])
def test_masked_and_special_logits(m, vocab):
    inf, nan = float("inf"), float("nan")
    logits, _ = _logits(8, vocab, vocab)
    logits[0] = -inf
    logits[1] = nan
    logits[2, 1:] = -inf
    logits[3, ::2] = nan
    logits[4, vocab - 1] = inf
    logits[5] = torch.finfo(torch.float32).min
    logits[6] = torch.finfo(torch.float32).min
    logits[6, vocab // 2] = 0
    logits[7, : vocab // 2] = -inf
    for kw in (dict(), dict(top_k=2), dict(top_p=0.5), dict(temperature=0.0), dict(min_p=0.2, top_k=5)):
        for u in (0.0, 0.6, 1.0 - 2.0 ** -24):
            tok = _check(m, logits, torch.full((8,), u, device="cuda"), **kw)
            assert tok[0] == -1 and tok[1] == -1 and tok[2] == 0 and tok[4] == vocab - 1 and tok[6] == vocab // 2


def test_numbers_at_and_beyond_the_ends(m):
    logits, _ = _logits(6, 3000, 2)
    u = torch.tensor([0.0, 1.0 - 2.0 ** -24, 1.0, 7.0, -1.0, float("nan")], device="cuda")
    tok = m.sample_tokens(logits, u)
    last = torch.clamp_max(u.nan_to_num(0).clamp_min(0), 1.0 - 2.0 ** -24)
    first = m.sample_tokens(logits, torch.where(u >= 1, last, u.nan_to_num(0).clamp_min(0)))
    assert torch.equal(tok[[0, 1, 4, 5]], first[[0, 1, 4, 5]])
    assert (tok >= 0).all() and (tok < 3000).all()


def test_settings_of_each_row(m):
    logits, u = _logits(40, 5003, 23)
    g = torch.Generator(device="cuda").manual_seed(1)
    t = torch.rand(40, generator=g, device="cuda") * 1.5
    t[::5] = 0
    k = torch.randint(0, 60, (40,), generator=g, device="cuda")
    p = torch.rand(40, generator=g, device="cuda") * 1.2
    p = p.clamp_max(1.0)
    mp = torch.rand(40, generator=g, device="cuda") * 0.1
    tok = _check(m, logits, u, temperature=t, top_k=k, top_p=p, min_p=mp)
    for r in range(0, 40, 3):  # a row alone, its settings as numbers
        one = m.sample_tokens(logits[r:r + 1], u[r:r + 1], float(t[r]), int(k[r]), float(p[r]), float(mp[r]))
        assert one[0] == tok[r]


def test_rows_do_not_depend_on_the_batch(m):
    logits, u = _logits(600, 20001, 31, torch.bfloat16)
    kw = dict(temperature=0.9, top_k=200, top_p=0.97, min_p=0.001)
    want = m.sample_tokens(logits, u, **kw)
    for n in (1, 2, 7, 40, 100, 300):
        assert torch.equal(m.sample_tokens(logits[:n], u[:n], **kw), want[:n])


def test_frequencies(m):
    """65,536 draws of a small distribution: each count within 6 standard deviations."""
    logits = torch.tensor([[2.0, 0.0, 1.0, -1.0, 1.5, -30.0]], device="cuda").expand(65536, 6)
    u = (torch.arange(65536, device="cuda") + 0.5) / 65536
    tok = m.sample_tokens(logits, u)
    p = torch.softmax(logits[0].double(), 0).cpu().numpy()
    n = np.bincount(tok.cpu().numpy(), minlength=6)
    assert (np.abs(n - 65536 * p) <= 6 * np.sqrt(65536 * p * (1 - p)) + 1).all()


def test_strides_shapes_and_host(m):
    wide, u = _logits(12, 2100, 41, torch.float16)
    for off in (0, 1, 3, 8):
        v = wide[:, off:off + 2000]
        assert torch.equal(m.sample_tokens(v, u, top_p=0.9), m.sample_tokens(v.contiguous().clone(), u, top_p=0.9))
    v = wide[::3, 5:2005]
    assert torch.equal(m.sample_tokens(v, u[::3]), m.sample_tokens(v.contiguous(), u[::3].contiguous()))
    assert torch.equal(m.sample_tokens(wide.t().contiguous().t(), u), m.sample_tokens(wide, u))
    three = m.sample_tokens(wide.view(3, 4, 2100), u.view(3, 4), top_k=9)
    assert three.shape == (3, 4) and torch.equal(three.view(-1), m.sample_tokens(wide, u, top_k=9))
    one = m.sample_tokens(wide[2], u[2], top_k=9)
    assert one.dim() == 0 and one == three.view(-1)[2]
    host, lp = m.sample_tokens(wide.cpu(), u.cpu(), top_k=9, return_logprob=True)
    assert host.device.type == "cpu" and lp.device.type == "cpu" and torch.equal(host, three.view(-1).cpu())
    assert m.sample_tokens(wide[:0], u[:0]).shape == (0,)


def test_another_stream(m):
    logits, u = _logits(20, 50688, 51)
    want = m.sample_tokens(logits, u, top_p=0.9)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [m.sample_tokens(logits, u, top_p=0.9) for _ in range(5)]
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


def test_offsets_beyond_32_bits(m):
    base = torch.empty(2_400_060_000, device="cuda", dtype=torch.bfloat16)
    logits = base.as_strided((3, 50688), (1_200_000_000, 1))
    src, u = _logits(3, 50688, 61, torch.bfloat16)
    logits.copy_(src)
    for kw in (dict(), dict(top_k=40, top_p=0.9), dict(top_p=0.9)):
        assert torch.equal(m.sample_tokens(logits, u, **kw), m.sample_tokens(src, u, **kw))


def test_kinds_of_settings(m):
    """64-bit counts, numpy numbers, ints for floats, and settings on the host."""
    logits, u = _logits(4, 700, 62)
    want = m.sample_tokens(logits, u, temperature=1.0, top_k=30, top_p=1.0, min_p=0.0)
    assert torch.equal(m.sample_tokens(logits, u, temperature=1, top_k=30.0, top_p=1, min_p=0), want)
    assert torch.equal(m.sample_tokens(logits, u, temperature=np.float32(1), top_k=np.int64(30), top_p=np.float64(1)), want)
    assert torch.equal(m.sample_tokens(logits, u.cpu().double(), top_k=torch.full((4,), 30)), want)
    assert torch.equal(m.sample_tokens(logits, u, top_k=torch.full((4,), 2 ** 40 + 30, device="cuda")), m.sample_tokens(logits, u))
    assert torch.equal(m.sample_tokens(logits, u, top_k=10 ** 12), m.sample_tokens(logits, u))
    with pytest.raises(ValueError, match="top_p"):
        m.sample_tokens(logits, u, top_p=torch.ones(3, device="cuda"))
    with pytest.raises(ValueError, match="u must"):
        m.sample_tokens(logits, u[:3])


@pytest.mark.parametrize("rows", [3, 400])
def test_many_equal_tokens_at_a_cut(m, rows):
    """More tokens of one value than the sorted list holds, at the cut of k and of p."""
    vocab = 30000
    logits = torch.zeros(rows, vocab, device="cuda")
    logits[:, ::7] = 1.0
    logits[:, 5] = 4.0
    u = torch.linspace(0, 0.999, rows, device="cuda")
    for kw in (dict(top_k=3000), dict(top_k=9000), dict(top_p=0.3), dict(top_p=0.7), dict(top_k=9000, top_p=0.5)):
        tok = m.sample_tokens(logits, u, **kw)
        pick = torch.arange(0, rows, max(1, rows // 3))
        assert torch.equal(_check(m, logits[pick], u[pick], **kw), tok[pick])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("spread", [0.5, 2.0, 6.0])
def test_cut_at_p_does_not_depend_on_the_batch(m, spread, dtype):
    """From flat rows, whose nucleus is most of the vocabulary, to peaked ones, alone and in batches of every kind."""
    logits, u = _logits(600, 9001, 71, dtype, spread)
    for kw in (dict(top_p=0.5), dict(top_p=0.9), dict(top_p=0.95), dict(top_p=0.97, temperature=0.7), dict(top_p=0.9, min_p=0.001)):
        want = m.sample_tokens(logits, u, **kw)
        for n in (1, 7, 40, 100, 160):
            assert torch.equal(m.sample_tokens(logits[:n], u[:n], **kw), want[:n])
        pick = torch.tensor([0, 299, 599], device="cuda")
        assert torch.equal(_check(m, logits[pick], u[pick], **kw), want[pick])


@pytest.mark.parametrize("rows", [4, 300])
def test_settings_out_of_range_in_tensors(m, rows):
    """What a number would be refused for has a meaning in a tensor, which is
    not looked at on the host: below 0 as 0, above 1 and NaN as no cut."""
    logits, u = _logits(rows, 4001, 81)
    def one(v):
        return torch.full((rows,), v, device="cuda")
    plain = m.sample_tokens(logits, u)
    best = logits.argmax(-1)
    assert torch.equal(m.sample_tokens(logits, u, top_p=one(-5.0)), best)
    assert torch.equal(m.sample_tokens(logits, u, top_p=one(float("-inf"))), best)
    assert torch.equal(m.sample_tokens(logits, u, top_p=one(7.0)), plain)
    assert torch.equal(m.sample_tokens(logits, u, top_p=one(float("nan"))), plain)
    assert torch.equal(m.sample_tokens(logits, u, min_p=one(-1.0)), plain)
    assert torch.equal(m.sample_tokens(logits, u, min_p=one(9.0)), best)
    assert torch.equal(m.sample_tokens(logits, u, min_p=one(float("nan"))), plain)
    assert torch.equal(m.sample_tokens(logits, u, top_k=one(-3)), plain)
    assert torch.equal(m.sample_tokens(logits, u, temperature=one(-2.0)), best)
    assert torch.equal(m.sample_tokens(logits, u, temperature=one(float("nan"))), best)
    spread = m.sample_tokens(logits, u, temperature=one(float("inf")))
    flat = m.sample_tokens(torch.zeros_like(logits), u)
    assert torch.equal(spread, flat)
