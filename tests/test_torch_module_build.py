"""The module _h24_torch: found by the torch and interpreter it was built for alone, and never needed for libh24."""
from __future__ import annotations

import os
import sysconfig

import pytest
import torch


def test_its_name_holds_the_versions(lib):
    from pollux_b200 import _native, build
    name = os.path.basename(_native.torch_module_path())
    assert torch.__version__ in name and sysconfig.get_config_var("SOABI") in name and name.endswith(".so")
    assert build.build_torch_module() == _native.torch_module_path() and os.path.exists(_native.torch_module_path())


def test_another_torch_does_not_load_it(lib, monkeypatch):
    from pollux_b200 import _native, int8
    monkeypatch.setattr(_native, "_torch_calls", None)
    monkeypatch.setattr(torch, "__version__", torch.__version__ + ".other")
    with pytest.warns(RuntimeWarning, match="has not been built"):
        calls = _native.torch_calls()
    assert calls.int8_linear(1, 2, 3) is None and _native.torch_calls() is calls
    with pytest.raises(TypeError):  # the general path answers
        int8.quantize_rows_int8(torch.zeros(2, 8, dtype=torch.int8))


def test_libh24_is_linked_without_it(lib, monkeypatch, tmp_path):
    from pollux_b200 import build
    monkeypatch.setattr(build, "OUT_DIR", str(tmp_path))
    monkeypatch.setattr(build, "LIB", str(tmp_path / "libh24.so"))
    monkeypatch.setattr(build, "torch_module_path", lambda: str(tmp_path / "module.so"))
    monkeypatch.setattr(build, "torch_command", lambda src, out: ["false"])
    with pytest.warns(RuntimeWarning, match="was not built"):
        assert build.build() == str(tmp_path / "libh24.so")
    assert os.listdir(tmp_path) == ["libh24.so"]
    with pytest.raises(RuntimeError, match="compilation failed"):
        build.build_torch_module()


@pytest.mark.gpu
def test_the_same_answers_without_it(lib, monkeypatch):
    from pollux_b200 import _native, int8, sampling
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(5, 48, generator=g, device="cuda")
    w = torch.randint(-127, 128, (70, 48), generator=g, device="cuda", dtype=torch.int8)
    mu, u = torch.rand(70, generator=g, device="cuda").half(), torch.rand(5, generator=g, device="cuda")

    def path():
        q, s, r = int8.add_rms_norm_int8(x, torch.ones(48, device="cuda"), x)
        y = int8.int8_linear(q, s, w, mu)
        return (q, s, r, y, int8.dequantize_rows_int8(q, s), *int8.quantize_rows_int8(x),
                *sampling.sample_tokens(y, u, 0.8, 10, 0.9, 0.01, return_logprob=True))
    want = path()
    monkeypatch.setattr(_native, "_torch_calls", _native._GeneralPath())
    assert all(torch.equal(a, b) for a, b in zip(path(), want))
