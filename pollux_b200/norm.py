"""RMS and layer norm of a residual stream on libh24, with gradients: the norm of
a training step, or of a model that is not quantised (int8.add_rms_norm_int8 is
the one whose rows go on in 8 bits).

``add_rms_norm`` adds the residual, hands the sum on and norms it (the
reference's pre-norm, pollux.py:566-702) in one pass; ``add_layer_norm`` is the
same with the mean taken off and a bias.  Backward is one pass too, with the sums
of the weight's gradient in registers.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _native as N
from .castor import _call, _stream, _work_device
from .int8 import _DTYPES, _code, _rows, _save, _saved, _tracked


def _forward(x, residual, weight, bias, eps: float, layer: bool):
    """(y, summed or None, stats) of rows x [rows, cols]."""
    rows, cols = x.shape
    dev = x.device
    y = torch.empty(rows, cols, dtype=x.dtype, device=dev)
    summed = None if residual is None else torch.empty(rows, cols, dtype=x.dtype, device=dev)
    stats = torch.empty(2 * rows, dtype=torch.float32, device=dev)
    _call(dev, "h24_add_norm", x.data_ptr(), None if residual is None else residual.data_ptr(), weight.data_ptr(),
          None if bias is None else bias.data_ptr(), _DTYPES[weight.dtype], layer, rows, cols, x.stride(0),
          0 if residual is None else residual.stride(0), _DTYPES[x.dtype], eps, y.data_ptr(),
          None if summed is None else summed.data_ptr(), stats.data_ptr(), _stream(dev))
    return y, summed, stats


class _AddNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, bias, eps, layer):
        y, summed, stats = _forward(x, residual, weight, bias, eps, layer)
        _save(ctx, x if summed is None else summed, weight, stats)
        ctx.layer = layer
        ctx.set_materialize_grads(False)
        return y, summed

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dsummed):
        s, weight, stats = _saved(ctx)
        need_x, need_r, need_w, need_b = ctx.needs_input_grad[:4]
        rows, cols = s.shape
        dev = s.device
        if dy is None:  # nothing reached y
            zero = torch.zeros(cols, dtype=weight.dtype, device=dev) if need_w or need_b else None
            return (dsummed if need_x else None, dsummed if need_r else None, zero if need_w else None,
                    zero if need_b else None, None, None)
        dy = _rows(dy, dev)
        dsummed = None if dsummed is None else _rows(dsummed, dev)
        dx = torch.empty(rows, cols, dtype=s.dtype, device=dev) if need_x or need_r else None
        dw = torch.empty(cols, dtype=weight.dtype, device=dev) if need_w else None
        db = torch.empty(cols, dtype=weight.dtype, device=dev) if need_b else None
        _call(dev, "h24_add_norm_backward", s.data_ptr(), weight.data_ptr(), _DTYPES[weight.dtype], ctx.layer, rows, cols,
              s.stride(0), _DTYPES[s.dtype], stats.data_ptr(), dy.data_ptr(), dy.stride(0),
              None if dsummed is None else dsummed.data_ptr(), 0 if dsummed is None else dsummed.stride(0),
              None if dx is None else dx.data_ptr(), None if dw is None else dw.data_ptr(),
              None if db is None else db.data_ptr(), _stream(dev))
        return dx if need_x else None, dx if need_r else None, dw, db, None, None


def _param(t: torch.Tensor, cols: int, dtype: torch.dtype, dev: torch.device, what: str) -> torch.Tensor:
    _code(t.dtype, what)
    if t.numel() != cols:
        raise ValueError(f"{what} must hold {cols} values, got {tuple(t.shape)}")
    return t.reshape(cols).to(device=dev, dtype=dtype).contiguous()


def _add_norm(x, weight, bias, residual, eps, layer: bool):
    if x.dim() < 1:
        raise ValueError("x must have at least one dimension")
    _code(x.dtype, "x")
    if not eps >= 0:
        raise ValueError(f"eps must not be negative, got {eps}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError(f"residual must be {x.dtype} of shape {tuple(x.shape)}, got {residual.dtype} "
                         f"of {tuple(residual.shape)}")
    cols = x.shape[-1]
    if cols < 1:
        raise ValueError(f"the rows of x are empty: {tuple(x.shape)}")
    dev = _work_device(x)
    # The kernels read parameters of x's type or fp32, both alike; another type widens exactly.
    kinds = {weight.dtype} if bias is None else {weight.dtype, bias.dtype}
    param = x.dtype if kinds == {x.dtype} else torch.float32
    w = _param(weight, cols, param, dev, "weight")
    b = None if bias is None else _param(bias, cols, param, dev, "bias")
    xr = _rows(x, dev)
    rr = None if residual is None else _rows(residual, dev)
    if _tracked(xr, rr, w, b):
        y, summed = _AddNorm.apply(xr, rr, w, b, eps, layer)
    else:
        y, summed, _ = _forward(xr, rr, w, b, eps, layer)
    if x.dim() != 2:
        y = y.reshape(x.shape)
        summed = None if summed is None else summed.reshape(x.shape)
    if x.device != dev:
        y = y.to(x.device)
        summed = None if summed is None else summed.to(x.device)
    return y, summed


def add_rms_norm(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None,
                 eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor | None]:
    """RMS norm of ``x + residual`` over the last dimension, times ``weight``.

    Returns ``(y, summed)`` in x's dtype (float32, float16 or bfloat16):
    ``summed = x + residual``, the next layer's residual (None without
    ``residual``), and its norm; sums and statistics are fp32.  Both outputs have
    gradients, which go to x, residual and weight."""
    got = (N._torch_calls or N.torch_calls()).add_norm(x, weight, None, residual, eps, False)
    return _add_norm(x, weight, None, residual, eps, False) if got is None else got


def add_layer_norm(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None,
                   residual: torch.Tensor | None = None,
                   eps: float = 1e-5) -> tuple[torch.Tensor, torch.Tensor | None]:
    """Layer norm of ``x + residual`` over the last dimension, times ``weight``
    plus ``bias``; otherwise as ``add_rms_norm``."""
    got = (N._torch_calls or N.torch_calls()).add_norm(x, weight, bias, residual, eps, True)
    return _add_norm(x, weight, bias, residual, eps, True) if got is None else got
