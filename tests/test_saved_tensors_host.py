"""What hooks on saved tensors give back is looked at before a kernel gets its address: other strides are put right, another
type or shape is refused.  The general path on the CPU, with the kernels' calls recorded and left out."""
from __future__ import annotations

import ctypes

import pytest
import torch
from torch.autograd.graph import saved_tensors_hooks


@pytest.fixture
def general(lib, monkeypatch):
    from pollux_b200 import _native as N
    from pollux_b200 import loss, norm
    calls = []
    monkeypatch.setattr(N, "_torch_calls", N._GeneralPath())
    for m in (loss, norm):
        monkeypatch.setattr(m, "_call", lambda dev, name, *a: calls.append((name, a, {i: _read(p) for i, p in enumerate(a)})))
        monkeypatch.setattr(m, "_stream", lambda dev: 0)
        monkeypatch.setattr(m, "_work_device", lambda t: t.device)
    return loss, norm, calls


def _read(p):
    """What lies at an address: the first 48 bytes (every matrix here has more)."""
    return ctypes.string_at(p, 48) if isinstance(p, int) and p > 1 << 20 else None


def _bytes(t):
    return t.detach().contiguous().view(torch.uint8).flatten()[:48].numpy().tobytes()


def _other_strides(t):
    if t.dim() == 2:
        return t.t().contiguous().t()
    wide = t.new_zeros(2 * t.numel())
    wide[::2] = t.flatten()
    return wide[::2].view(t.shape) if t.dim() == 1 else t


def _steps(loss, norm):
    g = torch.Generator().manual_seed(0)
    x, r = (torch.randn(5, 24, generator=g).requires_grad_(True) for _ in range(2))
    w, b = torch.randn(24, generator=g).requires_grad_(True), torch.randn(24, generator=g).requires_grad_(True)
    xh, wh = (torch.randn(n, 24, generator=g).half().requires_grad_(True) for n in (5, 7))
    t = torch.zeros(5, dtype=torch.int64)
    return {"norm": (lambda: norm.add_layer_norm(x, w, b)[0], 5, {0: x, 1: w}),
            "residual": (lambda: norm.add_rms_norm(x, w, residual=r)[0], 5, {1: w}),
            "loss": (lambda: loss.linear_cross_entropy(xh, wh, t), (2, 5), {0: xh, 3: wh})}


@pytest.mark.parametrize("name", ["norm", "residual", "loss"])
def test_other_strides(general, name):
    loss, norm, calls = general
    fn, strides, pointers = _steps(loss, norm)[name]
    with saved_tensors_hooks(lambda t: t, _other_strides):
        out = fn()
        (out.float().sum() if out.dim() else out.float()).backward()
    entry, args, read = calls[-1]
    assert entry.endswith("backward")
    for i in strides if isinstance(strides, tuple) else (strides,):
        assert args[i] == 24, (i, args)
    for i, t in pointers.items():
        assert read[i] == _bytes(t)


@pytest.mark.parametrize("name", ["norm", "residual", "loss"])
@pytest.mark.parametrize("change", [lambda t: t.double(), lambda t: t[..., :-1], lambda t: t.bfloat16(), lambda t: t[None]])
def test_other_types_and_shapes(general, name, change):
    loss, norm, calls = general
    fn, _, _ = _steps(loss, norm)[name]
    for which in range(3):
        seen = []

        def unpack(t):
            seen.append(1)
            return change(t) if len(seen) == which + 1 else t
        with saved_tensors_hooks(lambda t: t, unpack):
            out = fn()
            n = len(calls)
            with pytest.raises(RuntimeError, match="hook on saved tensors"):
                (out.sum() if out.dim() else out).backward()
            assert len(calls) == n
