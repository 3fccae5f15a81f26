"""Refusals of the training head path that need no GPU: wrong types, sizes and settings raise before anything is
launched, in Python and at the C entries."""
from __future__ import annotations

import pytest
import torch


def test_norm_refusals(lib):
    from pollux_b200 import norm
    x, w = torch.zeros(2, 8), torch.ones(8)
    for fn in (norm.add_rms_norm, norm.add_layer_norm):
        with pytest.raises(TypeError):
            fn(x.double(), w)
        with pytest.raises(TypeError):
            fn(x.to(torch.int32), w)
        with pytest.raises(ValueError, match="residual"):
            fn(x, w, residual=torch.zeros(2, 7))
        with pytest.raises(ValueError, match="residual"):
            fn(x, w, residual=x.half())
        for eps in (-1.0, float("nan")):
            with pytest.raises(ValueError, match="eps"):
                fn(x, w, eps=eps)
        with pytest.raises(ValueError, match="dimension"):
            fn(torch.tensor(1.0), w)
        with pytest.raises(ValueError, match="empty"):
            fn(x[:, :0], w[:0])


def test_norm_parameter_refusals(lib):
    if not torch.cuda.is_available():
        pytest.skip("parameters are looked at after the device")
    from pollux_b200 import norm
    x, w = torch.zeros(2, 8), torch.ones(8)
    with pytest.raises(TypeError, match="weight"):
        norm.add_rms_norm(x, w.to(torch.int32))
    with pytest.raises(ValueError, match="weight"):
        norm.add_rms_norm(x, w[:7])
    with pytest.raises(ValueError, match="bias"):
        norm.add_layer_norm(x, w, w[:7])


def test_loss_refusals(lib):
    from pollux_b200.loss import linear_cross_entropy as ce
    x, w, t = torch.zeros(2, 8).half(), torch.zeros(5, 8).half(), torch.zeros(2, dtype=torch.int64)
    for bad in ("avg", None, 1):
        with pytest.raises(ValueError, match="reduction"):
            ce(x, w, t, reduction=bad)
    with pytest.raises(ValueError, match="ignore_index"):
        ce(x, w, t, ignore_index=2 ** 63)
    with pytest.raises(TypeError, match="float16"):
        ce(x.float(), w.float(), t)
    with pytest.raises(TypeError, match="float16"):
        ce(x, w.to(torch.bfloat16), t)
    with pytest.raises(TypeError, match="int64"):
        ce(x, w, t.to(torch.uint8))
    with pytest.raises(TypeError, match="int64"):
        ce(x, w, t.float())
    with pytest.raises(RuntimeError, match="shapes"):
        ce(x[:, :7], w, t)
    with pytest.raises(ValueError, match="empty"):
        ce(x, w[:0], t)
    with pytest.raises(ValueError, match="empty"):
        ce(x[:, :0], w[:, :0], t)
    with pytest.raises(ValueError, match="weight two"):
        ce(x, w[0], t)
    with pytest.raises(ValueError, match="target"):
        ce(x, w, t[:1])
    with pytest.raises(ValueError, match="target"):
        ce(torch.zeros(2, 3, 8).half(), w, torch.zeros(3, 2, dtype=torch.int64))


def test_c_entries_refuse(lib):
    from pollux_b200 import _native as N
    bad, ok = N.H24_ERR_INVALID, N.H24_OK
    p = 4096  # never dereferenced: every call is refused before a launch
    fwd = dict(x=p, tokens=4, xs=8, w=p, vocab=9, ws=8, k=8, dtype=1, target=p, ignore=-100, red=1, loss=p, state=p)

    def forward(**kw):
        a = dict(fwd, **kw)
        return lib.h24_linear_ce_forward(*a.values(), None)
    for kw in (dict(tokens=-1), dict(vocab=0), dict(k=0), dict(k=(1 << 24) + 1), dict(dtype=0), dict(dtype=3), dict(red=3),
               dict(x=None), dict(w=None), dict(target=None), dict(loss=None), dict(state=None), dict(xs=-8), dict(ws=-1),
               dict(x=p + 1), dict(tokens=1 << 31), dict(vocab=1 << 31), dict(tokens=1 << 30, vocab=1 << 30)):
        assert forward(**kw) == bad, kw
    assert forward(tokens=0, red=0, loss=None, target=None, state=None) == ok
    bwd = dict(x=p, tokens=4, xs=8, w=p, vocab=9, ws=8, k=8, dtype=1, red=1, dloss=p, ds=0, state=p, dx=p, dw=p)

    def backward(**kw):
        a = dict(bwd, **kw)
        return lib.h24_linear_ce_backward(*a.values(), None)
    for kw in (dict(tokens=-1), dict(dtype=0), dict(ds=-1), dict(dloss=None), dict(state=None), dict(red=-1), dict(x=None)):
        assert backward(**kw) == bad, kw
    assert backward(dx=None, dw=None) == ok
    assert backward(tokens=0, dw=None) == ok
    nrm = dict(x=p, res=None, gain=p, bias=None, ptype=0, layer=0, rows=2, cols=8, xs=8, rs=0, dtype=0, eps=1e-6, y=p,
               summed=None, stats=p)

    def norm(**kw):
        a = dict(nrm, **kw)
        return lib.h24_add_norm(*a.values(), None)
    for kw in (dict(rows=-1), dict(cols=0), dict(dtype=5), dict(ptype=2), dict(eps=-1.0), dict(gain=None), dict(x=None),
               dict(y=None), dict(stats=None), dict(xs=-1), dict(bias=p), dict(res=p), dict(summed=p), dict(rows=1 << 31),
               dict(res=p, summed=p, rs=-1)):
        assert norm(**kw) == bad, kw
    assert norm(rows=0, x=None, y=None, stats=None) == ok
    back = dict(s=p, gain=p, ptype=0, layer=0, rows=2, cols=8, ss=8, dtype=0, stats=p, dy=p, dys=8, ds=None, dss=0, dx=p,
                dg=p, db=None)

    def norm_back(**kw):
        a = dict(back, **kw)
        return lib.h24_add_norm_backward(*a.values(), None)
    for kw in (dict(rows=-1), dict(cols=0), dict(dtype=5), dict(ptype=1), dict(gain=None), dict(s=None), dict(dy=None),
               dict(stats=None), dict(dys=-1), dict(ss=-1), dict(db=p)):
        assert norm_back(**kw) == bad, kw
    assert norm_back(dx=None, dg=None) == ok


def test_no_gpu_no_answer(lib):
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    from pollux_b200 import loss, norm
    with pytest.raises(RuntimeError, match="CUDA"):
        norm.add_rms_norm(torch.zeros(2, 8), torch.ones(8))
    with pytest.raises(RuntimeError, match="CUDA"):
        loss.linear_cross_entropy(torch.zeros(2, 8).half(), torch.zeros(5, 8).half(), torch.zeros(2, dtype=torch.int64))
