"""The three operators of the INT8 head path together, as examples/next_token.py
runs them, against the same path in 64 bits."""
from __future__ import annotations

import importlib.util
import os

import pytest
import torch

from conftest import REPO

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example(lib):
    spec = importlib.util.spec_from_file_location("next_token", os.path.join(REPO, "examples", "next_token.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


@pytest.mark.parametrize("batch", [1, 3, 17])
def test_greedy_token_of_the_path(example, batch):
    """The greedy token's logit in 64 bits is within the quantisation's error of
    the largest: half a step of each input element times the head's row sums."""
    vocab, d = 1000, 480
    head = example.make_head(vocab, d, seed=batch)
    x = torch.randn(batch, d, device="cuda", dtype=torch.bfloat16)
    r = torch.randn(batch, d, device="cuda", dtype=torch.bfloat16)
    gain = 1 + 0.1 * torch.randn(d, device="cuda")
    tok, lp = example.next_tokens(x, r, gain, head, torch.zeros(batch, device="cuda"), temperature=0.0)
    s = x.double() + r.double()
    y = s / torch.sqrt((s * s).mean(-1, keepdim=True) + 1e-6) * gain.double()
    w = head.weight_int8.double() * (head.mu_rows.float() / 127).half().double()[:, None]
    logits = y @ w.t()
    err = 0.5 * (y.abs().amax(-1) / 127) * w.abs().sum(1).max() * 1.01
    best = logits.max(-1).values
    assert (logits.gather(1, tok[:, None]).squeeze(1) >= best - 2 * err).all()
    assert (lp <= 0).all()


def test_path_in_a_graph(example):
    """Captured once and replayed on new inputs in place: the same tokens as called one by one."""
    head = example.make_head(5000, 240)
    gain = torch.ones(240, device="cuda", dtype=torch.bfloat16)
    x = torch.zeros(6, 240, device="cuda", dtype=torch.bfloat16)
    r, u = torch.zeros_like(x), torch.zeros(6, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        example.next_tokens(x, r, gain, head, u, top_k=20, top_p=0.9)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tok, lp = example.next_tokens(x, r, gain, head, u, top_k=20, top_p=0.9)
    for seed in range(3):
        g = torch.Generator(device="cuda").manual_seed(seed)
        x.copy_(torch.randn(6, 240, generator=g, device="cuda"))
        r.copy_(torch.randn(6, 240, generator=g, device="cuda"))
        u.copy_(torch.rand(6, generator=g, device="cuda"))
        graph.replay()
        want, want_lp = example.next_tokens(x, r, gain, head, u, top_k=20, top_p=0.9)
        assert torch.equal(tok, want) and torch.equal(lp, want_lp)


def test_example_runs(example, monkeypatch, capsys):
    monkeypatch.setattr("sys.argv", ["next_token.py", "2", "3"])
    example.main()
    out = capsys.readouterr().out
    assert "tokens of the first sequence" in out and "us a step" in out
