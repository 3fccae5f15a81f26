"""The INT8 head path on libh24: activations in 8 bits and their product with an
INT8 layer, without materialising it.

``add_rms_norm_int8`` adds the residual, takes the RMS norm (the reference's
pre-norm, pollux.py:566-702) and quantises each row to int8 with one fp32
scale, in one pass.  ``int8_linear`` multiplies such rows with the INT8 weights
and fp16 row scales that the ``.plx`` container holds for ``tok_emb`` and
``head`` (pack.py:124-136), exactly in int32.  ``quantize_rows_int8`` and
``dequantize_rows_int8`` are the quantisation without a norm and its inverse.

``enable_int8_forward`` makes the not-yet-materialised ``PackedInt8Linear``
layers of a model (the reference's included) run this way: the head is read as
1 byte a weight where ``materialize`` + ``F.linear`` (pollux.py:545-558) read 2.
All of it is for inference: the weights are buffers and nothing has a gradient.
Where an input requires one, the outputs do too, and a backward pass that reaches
them raises NotImplementedError.
"""
from __future__ import annotations

import math

import torch
import torch.nn as nn
import torch.nn.functional as F

from . import _native as N
from .castor import _aligned, _call, _stream, _work_device

_DTYPES = {torch.float32: N.DTYPE_F32, torch.float16: N.DTYPE_F16, torch.bfloat16: N.DTYPE_BF16}
MAX_IN_FEATURES = 131_000  # above this an int32 sum of int8 products could overflow


def _code(t: torch.dtype, what: str) -> int:
    code = _DTYPES.get(t)
    if code is None:
        raise TypeError(f"{what} must be float32, float16 or bfloat16, got {t}")
    return code


def _rows(t: torch.Tensor, dev: torch.device) -> torch.Tensor:
    """``t`` as [rows, cols] on ``dev`` with contiguous rows (a row stride is
    kept as it is; anything else is copied)."""
    if t.device != dev:
        t = t.to(dev)
    if t.dim() != 2:
        t = t.reshape(math.prod(t.shape[:-1]), t.shape[-1])  # (-1 has no answer where the last is 0)
    if t.stride(1) != 1 and t.shape[1] > 1:
        t = t.contiguous()
    return t


class _NoGradient(torch.autograd.Function):
    """A call whose outputs stand in the graph, so that a gradient that is asked of it raises and is not lost."""

    @staticmethod
    def forward(ctx, fn, *args):
        ctx.name = fn.__name__
        return fn(*args)

    @staticmethod
    def backward(ctx, *grads):
        raise NotImplementedError(f"{ctx.name} is for inference and has no gradient; call it under torch.no_grad() "
                                  "or on detached tensors")


def _tracked(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _vector(t: torch.Tensor, n: int, dtype: torch.dtype | None, dev: torch.device, what: str) -> torch.Tensor:
    if t.numel() != n:
        raise ValueError(f"{what} must hold {n} values, got {tuple(t.shape)}")
    if t.device != dev or (dtype is not None and t.dtype != dtype):
        t = t.to(device=dev, dtype=dtype)
    return t if t.is_contiguous() else t.contiguous()


def _holds_rows(t: torch.Tensor, lead) -> bool:
    """Whether ``t`` has a value for each row of leading dimensions ``lead``, in their order: the same dimensions
    up to ones, or one of the two a flat list."""
    if t.numel() != math.prod(lead):
        return False
    own, want = [n for n in t.shape if n != 1], [n for n in lead if n != 1]
    return own == want or len(own) <= 1 or len(want) <= 1 or t.numel() == 0


def _check_scale(scale: torch.Tensor, q: torch.Tensor) -> None:
    if not _holds_rows(scale, q.shape[:-1]):
        raise ValueError(f"scale must hold one value for each row of q, {tuple(q.shape[:-1])}, got {tuple(scale.shape)}")


def _check_rows(t: torch.Tensor, what: str) -> None:
    if t.dim() < 1:
        raise ValueError(f"{what} must have at least one dimension")


def add_rms_norm_int8(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None,
                      eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor | None]:
    """RMS norm of ``x + residual`` over the last dimension, as int8 rows.

    Returns ``(q, scale, summed)``: ``q`` int8 of x's shape and ``scale`` fp32 of
    its leading shape, with ``q * scale`` the normed rows times ``weight``, and
    ``summed = x + residual`` in x's dtype, the next layer's residual (None
    without ``residual``).  Sums, statistics and the norm are fp32, taken of the
    unrounded sum.  A row with a NaN gets a NaN scale and zeros."""
    got = (N._torch_calls or N.torch_calls()).add_rms_norm_int8(x, weight, residual, eps)
    if got is not None:
        return got
    if _tracked(x, weight, residual):
        return _NoGradient.apply(add_rms_norm_int8, x, weight, residual, eps)
    _check_rows(x, "x")
    code = _code(x.dtype, "x")
    if eps < 0:
        raise ValueError(f"eps must not be negative, got {eps}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError(f"residual must be {x.dtype} of shape {tuple(x.shape)}, got {residual.dtype} "
                         f"of {tuple(residual.shape)}")
    _code(weight.dtype, "weight")
    dev = _work_device(x)
    cols = x.shape[-1]
    xr = _rows(x, dev)
    rr = None if residual is None else _rows(residual, dev)
    # The kernel reads gains of x's dtype or fp32; another 16-bit type widens exactly.
    w = _vector(weight, cols, None if weight.dtype in (x.dtype, torch.float32) else torch.float32, dev, "weight")
    rows = xr.shape[0]
    q = xr.new_empty(x.shape, dtype=torch.int8)
    scale = xr.new_empty(x.shape[:-1], dtype=torch.float32)
    summed = None if rr is None else xr.new_empty(x.shape)
    if rows:
        _call(dev, "h24_add_rms_norm_int8", xr.data_ptr(), None if rr is None else rr.data_ptr(), w.data_ptr(),
              code if w.dtype == x.dtype else N.DTYPE_F32, rows, cols, xr.stride(0),
              0 if rr is None else rr.stride(0), code, eps, q.data_ptr(), scale.data_ptr(),
              None if summed is None else summed.data_ptr(), _stream(dev))
    if x.device != dev:
        q, scale = q.to(x.device), scale.to(x.device)
        summed = None if summed is None else summed.to(x.device)
    return q, scale, summed


def quantize_rows_int8(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Per-row int8 of ``x`` over its last dimension: ``(q, scale)`` with
    ``q * scale`` within half a scale of x."""
    got = (N._torch_calls or N.torch_calls()).quantize_rows_int8(x)
    if got is not None:
        return got
    if _tracked(x):
        return _NoGradient.apply(quantize_rows_int8, x)
    _check_rows(x, "x")
    code = _code(x.dtype, "x")
    dev = _work_device(x)
    xr = _rows(x, dev)
    rows, cols = xr.shape
    q = xr.new_empty(x.shape, dtype=torch.int8)
    scale = xr.new_empty(x.shape[:-1], dtype=torch.float32)
    if rows:
        _call(dev, "h24_rows_int8_quantize", xr.data_ptr(), rows, cols, xr.stride(0), code, q.data_ptr(),
              scale.data_ptr(), _stream(dev))
    return (q, scale) if x.device == dev else (q.to(x.device), scale.to(x.device))


def dequantize_rows_int8(q: torch.Tensor, scale: torch.Tensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``q * scale`` per row, rounded once to ``dtype``."""
    got = (N._torch_calls or N.torch_calls()).dequantize_rows_int8(q, scale, dtype)
    if got is not None:
        return got
    if _tracked(scale):
        return _NoGradient.apply(dequantize_rows_int8, q, scale, dtype)
    _check_rows(q, "q")
    if q.dtype != torch.int8:
        raise TypeError(f"q must be int8, got {q.dtype}")
    code = _code(dtype, "dtype")
    _check_scale(scale, q)
    dev = _work_device(q)
    cols = q.shape[-1]
    rows = q.numel() // cols if cols else 0
    qr = _aligned(q if q.device == dev else q.to(dev))
    out = qr.new_empty(q.shape, dtype=dtype)
    if rows and cols:
        s = _vector(scale, rows, torch.float32, dev, "scale")
        _call(dev, "h24_rows_int8_dequant", qr.data_ptr(), s.data_ptr(), rows, cols, code, out.data_ptr(),
              _stream(dev))
    return out if q.device == dev else out.to(q.device)


def int8_linear(q: torch.Tensor, scale: torch.Tensor, weight_int8: torch.Tensor, mu_rows: torch.Tensor,
                bias: torch.Tensor | None = None, out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """``(q * scale) @ W.T + bias`` for int8 rows ``q`` [..., in] with fp32
    ``scale`` [...] (or as a flat list), and the INT8 layer ``weight_int8`` [out, in] with fp16
    ``mu_rows`` [out] (``W = weight_int8 * fp16(mu / 127)``, as
    ``PackedInt8Linear``).  The sum is exact in int32; the scaling and the bias
    are fp32; the result is rounded once to ``out_dtype``."""
    got = (N._torch_calls or N.torch_calls()).int8_linear(q, scale, weight_int8, mu_rows, bias, out_dtype)
    if got is not None:
        return got
    if _tracked(scale, mu_rows, bias):
        return _NoGradient.apply(int8_linear, q, scale, weight_int8, mu_rows, bias, out_dtype)
    _check_rows(q, "q")
    if q.dtype != torch.int8 or weight_int8.dtype != torch.int8:
        raise TypeError(f"q and weight_int8 must be int8, got {q.dtype} and {weight_int8.dtype}")
    if mu_rows.dtype != torch.float16:
        raise TypeError(f"mu_rows must be float16, got {mu_rows.dtype}")
    if weight_int8.dim() != 2:
        raise ValueError(f"weight_int8 must be 2-D, got {tuple(weight_int8.shape)}")
    out_f, in_f = weight_int8.shape
    if q.shape[-1] != in_f:
        raise RuntimeError(f"mat1 and mat2 shapes cannot be multiplied "
                           f"({q.numel() // max(1, q.shape[-1])}x{q.shape[-1]} and {in_f}x{out_f})")
    if in_f > MAX_IN_FEATURES:
        raise ValueError(f"in_features must be at most {MAX_IN_FEATURES}, got {in_f}")
    code = _code(out_dtype, "out_dtype")
    _check_scale(scale, q)
    dev = _work_device(q)
    qr = _rows(q, dev)
    w = weight_int8 if weight_int8.device == dev else weight_int8.to(dev)
    if not w.is_contiguous():
        w = w.contiguous()
    tokens = qr.shape[0]
    s = _vector(scale, tokens, torch.float32, dev, "scale")
    mu = _vector(mu_rows, out_f, None, dev, "mu_rows")
    b = None if bias is None else _vector(bias, out_f, torch.float32, dev, "bias")
    y = qr.new_empty(q.shape[:-1] + (out_f,), dtype=out_dtype)
    if tokens and out_f:
        _call(dev, "h24_int8_linear", qr.data_ptr(), s.data_ptr(), tokens, qr.stride(0), w.data_ptr(), mu.data_ptr(),
              out_f, in_f, None if b is None else b.data_ptr(), code, y.data_ptr(), _stream(dev))
    return y if q.device == dev else y.to(q.device)


def _int8_forward(self, x: torch.Tensor) -> torch.Tensor:
    if getattr(self, "_materialized", False):
        return F.linear(x, self.weight.to(dtype=x.dtype), self.bias)
    q, scale = quantize_rows_int8(x)
    return int8_linear(q, scale, self.weight_int8, self.mu_rows, self.bias, out_dtype=x.dtype)


def enable_int8_forward(model: nn.Module) -> int:
    """Make every not-yet-materialised INT8 linear layer of ``model`` run
    forward on its 8-bit weights, with its input quantised row by row (instance
    attribute, so the reference's PackedInt8Linear is covered too); returns the
    number of layers.  Embeddings keep their forward."""
    n = 0
    for m in model.modules():
        if hasattr(m, "weight_int8") and hasattr(m, "mu_rows") and hasattr(m, "out_features") \
                and not getattr(m, "_materialized", False):
            m.forward = _int8_forward.__get__(m, type(m))
            n += 1
    return n
