"""Under autocast the loss casts what F.linear casts, and refuses the rest as it does without.  (Autocast's state is put in
its place: without a GPU torch does not enable it.)"""
from __future__ import annotations

import pytest
import torch


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_float64_is_not_cast(lib, monkeypatch, dtype):
    from pollux_b200.loss import linear_cross_entropy as ce
    monkeypatch.setattr(torch, "is_autocast_enabled", lambda *a: True)
    monkeypatch.setattr(torch, "get_autocast_dtype", lambda *a: dtype)
    x, w, t = torch.zeros(2, 8), torch.zeros(5, 8), torch.zeros(2, dtype=torch.int64)
    for a, b in ((x.double(), w.double()), (x, w.double()), (x.double(), w), (x, w.to(torch.int8))):
        with pytest.raises(TypeError, match="float16"):
            ce(a, b, t)
