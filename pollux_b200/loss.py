"""Softmax cross entropy of a model's head on libh24, with its gradients and
without its logits.

``linear_cross_entropy(x, weight, target)`` is
``F.cross_entropy(F.linear(x, weight), target)`` for fp16 or bf16 states and
head: the [tokens, vocab] logits are reduced tile by tile as the tensor cores
finish them, and computed again, a piece of the vocabulary at a time, where a
gradient is asked for.  With ``reduction="none"`` and no gradient it scores
text: each token's negative log-likelihood.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _native as N
from .castor import _call, _stream, _work_device
from .int8 import _holds_rows, _rows, _save, _saved, _tracked

_DTYPES = {torch.float16: N.DTYPE_F16, torch.bfloat16: N.DTYPE_BF16}
_REDUCTIONS = {"none": N.REDUCE_NONE, "mean": N.REDUCE_MEAN, "sum": N.REDUCE_SUM}


def _args(x: torch.Tensor, weight: torch.Tensor) -> tuple:
    return (x.data_ptr(), x.shape[0], x.stride(0), weight.data_ptr(), weight.shape[0], weight.stride(0), x.shape[1],
            _DTYPES[x.dtype])


def _forward(x, weight, target, ignore_index: int, reduction: int):
    """(loss, state) of rows x [tokens, in] and target [tokens]."""
    tokens, dev = x.shape[0], x.device
    loss = torch.empty(tokens if reduction == N.REDUCE_NONE else (), dtype=torch.float32, device=dev)
    state = torch.empty(3 * tokens + 1, dtype=torch.int32, device=dev)
    _call(dev, "h24_linear_ce_forward", *_args(x, weight), target.data_ptr(), ignore_index, reduction, loss.data_ptr(),
          state.data_ptr(), _stream(dev))
    return loss, state


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, target, ignore_index, reduction):
        loss, state = _forward(x, weight, target, ignore_index, reduction)
        _save(ctx, x, weight, state)
        ctx.reduction = reduction
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss):
        x, weight, state = _saved(ctx)
        dev = x.device
        dx = torch.empty(x.shape, dtype=x.dtype, device=dev) if ctx.needs_input_grad[0] else None
        dw = torch.empty(weight.shape, dtype=weight.dtype, device=dev) if ctx.needs_input_grad[1] else None
        _call(dev, "h24_linear_ce_backward", *_args(x, weight), ctx.reduction, dloss.data_ptr(),
              dloss.stride(0) if dloss.dim() else 0, state.data_ptr(), None if dx is None else dx.data_ptr(),
              None if dw is None else dw.data_ptr(), _stream(dev))
        return dx, dw, None, None, None


def linear_cross_entropy(x: torch.Tensor, weight: torch.Tensor, target: torch.Tensor, ignore_index: int = -100,
                         reduction: str = "mean") -> torch.Tensor:
    """Cross entropy of the softmax of ``x @ weight.T`` against ``target``.

    ``x`` [..., in] and ``weight`` [vocab, in] are both float16 or both bfloat16
    (under autocast they are cast as ``F.linear`` casts them); ``target`` [...]
    (or as a flat list) holds int64 or int32 token numbers.  Tokens whose target
    is ``ignore_index`` have no loss, give nothing to a gradient and take no time
    in the products; what their rows of x hold does not matter.  A target
    outside the vocabulary makes its loss NaN, and the gradients.

    ``reduction`` "mean" (over the tokens that are not ignored; NaN where there
    is none), "sum" or "none" (x's leading shape, 0 where ignored).  The result
    is fp32.  Gradients go to x and weight in their type, each rounded once from
    fp32 sums; on their way the probabilities are rounded to that type."""
    red = _REDUCTIONS.get(reduction)
    if red is None:
        raise ValueError(f"reduction must be 'none', 'mean' or 'sum', got {reduction!r}")
    if not -2 ** 63 <= ignore_index < 2 ** 63:
        raise ValueError(f"ignore_index must be a token number of 64 bits, got {ignore_index}")
    got = (N._torch_calls or N.torch_calls()).linear_ce(x, weight, target, ignore_index, red)
    if got is not None:
        return got
    if x.dim() < 1 or weight.dim() != 2:
        raise ValueError(f"x must have at least one dimension and weight two, got {tuple(x.shape)} and "
                         f"{tuple(weight.shape)}")
    if torch.is_autocast_enabled("cuda"):
        low = torch.get_autocast_dtype("cuda")
        # (float64 is not cast by autocast: it is refused below, as without.)
        x, weight = (a.to(low) if a.is_floating_point() and a.dtype != torch.float64 else a for a in (x, weight))
    if x.dtype not in _DTYPES or weight.dtype != x.dtype:
        raise TypeError(f"x and weight must both be float16 or both bfloat16, got {x.dtype} and {weight.dtype}")
    vocab, in_f = weight.shape
    if vocab < 1 or in_f < 1:
        raise ValueError(f"weight must not be empty, got {tuple(weight.shape)}")
    if x.shape[-1] != in_f:
        raise RuntimeError(f"mat1 and mat2 shapes cannot be multiplied "
                           f"({x.numel() // max(1, x.shape[-1])}x{x.shape[-1]} and {in_f}x{vocab})")
    if target.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"target must be int64 or int32, got {target.dtype}")
    lead = x.shape[:-1]
    if not _holds_rows(target, lead):
        raise ValueError(f"target must hold one token number for each row of x, {tuple(lead)}, "
                         f"got {tuple(target.shape)}")
    dev = _work_device(x)
    rows = _rows(x, dev)
    w = _rows(weight, dev)
    t = target.reshape(-1)
    if t.device != dev or t.dtype != torch.int64:
        t = t.to(device=dev, dtype=torch.int64)
    if not t.is_contiguous():
        t = t.contiguous()
    if _tracked(rows, w):
        loss = _LinearCrossEntropy.apply(rows, w, t, ignore_index, red)
    else:
        loss = _forward(rows, w, t, ignore_index, red)[0]
    if red == N.REDUCE_NONE and loss.shape != lead:
        loss = loss.reshape(lead)
    return loss if x.device == dev else loss.to(x.device)
