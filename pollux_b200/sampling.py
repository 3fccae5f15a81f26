"""Token sampling on libh24: temperature, top-k, top-p and min-p (the settings
of generate.py:143-329, with min-p) from given uniform numbers.

Probabilities are 64-bit fixed-point weights, so every sum is exact and a row's
token depends only on its logits, its settings and its number -- not on the
batch it is in or on how the GPU splits the row.
"""
from __future__ import annotations

import torch

from . import _native as N
from .castor import _call, _stream, _work_device
from .int8 import _NoGradient, _code, _holds_rows, _rows, _tracked

MAX_VOCAB = 1 << 22
_INF = float("inf")


def _setting(v, dtype: torch.dtype, dev: torch.device):
    """(tensor kept alive, pointer or None, scalar) of one sampling setting."""
    if not isinstance(v, torch.Tensor):
        return None, None, float(v)
    if dtype == torch.int32 and v.dtype == torch.int64:
        v = v.clamp(0, MAX_VOCAB)  # what the vocabulary holds, and no more than 32 bits
    if v.device != dev or v.dtype != dtype:
        v = v.to(device=dev, dtype=dtype)
    if not v.is_contiguous():
        v = v.contiguous()
    return v, v.data_ptr(), 0


def sample_tokens(logits: torch.Tensor, u: torch.Tensor, temperature: float | torch.Tensor = 1.0,
                  top_k: int | torch.Tensor = 0, top_p: float | torch.Tensor = 1.0,
                  min_p: float | torch.Tensor = 0.0, return_logprob: bool = False):
    """One token for each row of ``logits`` [..., vocab] from uniform numbers
    ``u`` [...] in [0, 1).

    Tokens are ordered by scaled logit, ties by index.  Kept are the first
    ``top_k`` (0: all); of these the shortest run from the top that reaches
    ``top_p`` of their mass (1: all); of these the ones with at least ``min_p``
    of the most probable token's probability.  The token is where the running
    mass of what is kept, in the order of the vocabulary, passes ``u`` of it.
    ``temperature`` 0 takes the largest logit.  Each setting is a number or a
    tensor with one value a row, of the leading shape or a flat list.

    NaN logits are never chosen, +inf counts as the largest fp32 number; a row
    with no logit above -inf gives -1.
    Returns int64 tokens of the leading shape, with ``return_logprob`` also the
    fp32 log-probabilities of the tokens at that temperature before the cuts
    (-inf for a row that gives -1); no gradient goes through them."""
    got = (N._torch_calls or N.torch_calls()).sample_tokens(logits, u, temperature, top_k, top_p, min_p, return_logprob)
    if got is not None:
        return got
    if return_logprob and _tracked(logits):
        return _NoGradient.apply(sample_tokens, logits, u, temperature, top_k, top_p, min_p, return_logprob)
    if logits.dim() < 1:
        raise ValueError("logits must have at least one dimension")
    code = _code(logits.dtype, "logits")
    lead, vocab = logits.shape[:-1], logits.shape[-1]
    if not 0 < vocab <= MAX_VOCAB:
        raise ValueError(f"the vocabulary must hold 1 to {MAX_VOCAB} tokens, got {vocab}")
    rows = logits.numel() // vocab
    for name, v, most in (("temperature", temperature, _INF), ("top_k", top_k, _INF), ("top_p", top_p, 1.0),
                          ("min_p", min_p, 1.0)):
        if isinstance(v, torch.Tensor):
            if not _holds_rows(v, lead):
                raise ValueError(f"{name} must be a number or hold one value for each row, {tuple(lead)}, "
                                 f"got {tuple(v.shape)}")
        elif not 0 <= v <= most:
            raise ValueError(f"{name} out of range: {v}")
    if not _holds_rows(u, lead):
        raise ValueError(f"u must hold one number for each row, {tuple(lead)}, got {tuple(u.shape)}")
    dev = _work_device(logits)
    ts, tp, t1 = _setting(temperature, torch.float32, dev)
    ks, kp, k1 = _setting(top_k, torch.int32, dev)
    ps, pp, p1 = _setting(top_p, torch.float32, dev)
    ms, mp, m1 = _setting(min_p, torch.float32, dev)
    us, up, _ = _setting(u, torch.float32, dev)
    lr = _rows(logits, dev)
    tokens = lr.new_empty(lead, dtype=torch.int64)
    logprob = lr.new_empty(lead, dtype=torch.float32) if return_logprob else None
    if rows:
        _call(dev, "h24_sample_tokens", lr.data_ptr(), code, rows, vocab, lr.stride(0), up, tp, t1, kp,
              vocab if k1 > vocab else int(k1), pp, p1, mp, m1, tokens.data_ptr(),
              None if logprob is None else logprob.data_ptr(), _stream(dev))
    if logits.device != dev:
        tokens = tokens.to(logits.device)
        logprob = None if logprob is None else logprob.to(logits.device)
    return (tokens, logprob) if return_logprob else tokens
