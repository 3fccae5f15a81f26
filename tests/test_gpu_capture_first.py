"""The first call of a process may lie inside a graph capture: nothing that the
library sets up then ends the capture."""
from __future__ import annotations

import os
import subprocess
import sys

import pytest

from conftest import REPO

pytestmark = pytest.mark.gpu

CODE = """
import sys, torch
sys.path.insert(0, {repo!r})
from pollux_b200 import int8, sampling
tokens = {tokens}
q = torch.randint(-127, 128, (tokens, 93), device="cuda", dtype=torch.int8)
w = torch.randint(-127, 128, (300, 93), device="cuda", dtype=torch.int8)
s, mu = torch.rand(tokens, device="cuda"), torch.ones(300, device="cuda").half()
x, g, u = torch.randn(tokens, 93, device="cuda"), torch.ones(93, device="cuda"), torch.rand(tokens, device="cuda")
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    y = int8.int8_linear(q, s, w, mu)
    n = int8.add_rms_norm_int8(x, g)
    t = sampling.sample_tokens(y, u, top_k=5)
for _ in range(2):
    q.random_(-127, 128)
    graph.replay()
    want = int8.int8_linear(q, s, w, mu)
    assert torch.equal(y, want)
    assert torch.equal(t, sampling.sample_tokens(want, u, top_k=5))
    assert torch.equal(n[0], int8.add_rms_norm_int8(x, g)[0])
torch.cuda.synchronize()
print("captured")
"""


@pytest.mark.parametrize("tokens", [1, 40, 700])
def test_first_call_inside_a_capture(lib, tokens):
    r = subprocess.run([sys.executable, "-c", CODE.format(repo=REPO, tokens=tokens)],
                       capture_output=True, text=True, timeout=300, cwd=os.path.dirname(REPO))
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]
