"""Values for each row (scales, numbers, settings) are taken in the rows' order:
another order of the same count is refused, a flat list is not."""
from __future__ import annotations

import pytest
import torch


@pytest.fixture(scope="module", params=["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def dev(request, lib):
    return request.param


def test_refused_orders(dev):
    from pollux_b200 import int8, sampling
    q = torch.zeros(4, 10, 48, device=dev, dtype=torch.int8)
    w, mu = torch.zeros(5, 48, device=dev, dtype=torch.int8), torch.ones(5, device=dev).half()
    for shape in ((10, 4), (10, 4, 1), (2, 20), (2, 2, 10)):
        s = torch.ones(shape, device=dev)
        with pytest.raises(ValueError, match="scale"):
            int8.int8_linear(q, s, w, mu)
        with pytest.raises(ValueError, match="scale"):
            int8.dequantize_rows_int8(q, s)
    l, good = torch.zeros(4, 10, 8, device=dev), torch.zeros(4, 10, device=dev)
    with pytest.raises(ValueError, match="u must hold"):
        sampling.sample_tokens(l, torch.zeros(10, 4, device=dev))
    for name in ("temperature", "top_k", "top_p", "min_p"):
        v = torch.ones(10, 4, device=dev, dtype=torch.int32 if name == "top_k" else torch.float32)
        with pytest.raises(ValueError, match=name):
            sampling.sample_tokens(l, good, **{name: v})


def test_which_shapes_hold_the_rows():
    from pollux_b200.int8 import _holds_rows
    z = torch.zeros
    for shape, lead in (((40,), (4, 10)), ((4, 10), (4, 10)), ((4, 10, 1), (4, 10)), ((1, 4, 10), (4, 10)),
                        ((4, 10), (40,)), ((4, 10), (4, 1, 10)), ((1,), ()), ((), ()), ((), (1,)), ((0,), (0, 3)),
                        ((0, 3), (0,))):
        assert _holds_rows(z(shape), lead), (shape, lead)
    for shape, lead in (((10, 4), (4, 10)), ((39,), (4, 10)), ((2, 20), (4, 10)), ((2,), ()), ((), (2,))):
        assert not _holds_rows(z(shape), lead), (shape, lead)


@pytest.mark.gpu
def test_accepted_shapes(lib):
    from pollux_b200 import int8, sampling
    g = torch.Generator(device="cuda").manual_seed(0)
    q = torch.randint(-127, 128, (4, 10, 48), generator=g, device="cuda", dtype=torch.int8)
    w = torch.randint(-127, 128, (5, 48), generator=g, device="cuda", dtype=torch.int8)
    mu, s = torch.ones(5, device="cuda").half(), torch.rand(4, 10, generator=g, device="cuda")
    want, back = int8.int8_linear(q, s, w, mu), int8.dequantize_rows_int8(q, s)
    for v in (s.view(40), s.view(4, 10, 1), s.view(1, 4, 10), s.t().contiguous().t()):
        assert torch.equal(int8.int8_linear(q, v, w, mu), want)
        assert torch.equal(int8.dequantize_rows_int8(q, v), back)
    assert torch.equal(int8.int8_linear(q.view(40, 48), s, w, mu), want.view(40, 5))
    l = torch.randn(4, 10, 500, generator=g, device="cuda")
    t = 0.5 + s
    tok = sampling.sample_tokens(l, s, temperature=t)
    for v in (s.view(40), s.view(4, 10, 1), s.t().contiguous().t()):
        assert torch.equal(sampling.sample_tokens(l, v, temperature=0.5 + v), tok)
