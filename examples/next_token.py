"""From the last hidden states to the next tokens on an INT8 output head that
is never materialised: residual addition + RMS norm + int8 rows, int8 product
with the head, sampling.

    python examples/next_token.py [batch] [steps]

The head has the d=1920 model's shape ([50688, 1920], random weights).  Each
step stands in for the model's blocks with a random state for the last token;
what runs on the GPU besides that lookup are three kernels a step.
"""
from __future__ import annotations

import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from pollux_b200 import int8, pack, packed_linear, sampling  # noqa: E402


def next_tokens(hidden: torch.Tensor, residual: torch.Tensor, gain: torch.Tensor,
                head: packed_linear.PackedInt8Linear, u: torch.Tensor, **settings):
    """(tokens, log-probabilities) for the last hidden states [batch, d]."""
    q, scale, _ = int8.add_rms_norm_int8(hidden, gain, residual=residual)
    logits = int8.int8_linear(q, scale, head.weight_int8, head.mu_rows, head.bias)
    return sampling.sample_tokens(logits, u, return_logprob=True, **settings)


def make_head(vocab: int, d: int, seed: int = 0) -> packed_linear.PackedInt8Linear:
    """A packed head of random weights."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    w = torch.randn(vocab, d, generator=g, device="cuda") * 0.05
    head = packed_linear.PackedInt8Linear(d, vocab).cuda()
    q, mu = pack.quantize_int8_device(w)
    head.weight_int8.copy_(q)
    head.mu_rows.copy_(mu)
    return head


def main() -> None:
    batch = int(sys.argv[1]) if len(sys.argv) > 1 else 4
    steps = int(sys.argv[2]) if len(sys.argv) > 2 else 32
    vocab, d = 50688, 1920
    head = make_head(vocab, d)
    gain = torch.ones(d, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    states = torch.randn(vocab, d, generator=g, device="cuda").to(torch.bfloat16)
    residual = torch.randn(batch, d, generator=g, device="cuda").to(torch.bfloat16)
    hidden = torch.zeros_like(residual)
    u = torch.rand(steps, batch, generator=g, device="cuda")
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    out = []
    for step in range(steps):
        if step == 1:
            start.record()
        tokens, logprob = next_tokens(hidden, residual, gain, head, u[step], temperature=0.8, top_k=50, top_p=0.95)
        out.append(tokens)
        hidden = states[tokens]
    end.record()
    torch.cuda.synchronize()
    print("tokens of the first sequence:", torch.stack(out)[:, 0].tolist())
    if steps > 1:
        print(f"{start.elapsed_time(end) / (steps - 1) * 1e3:.1f} us a step of {batch} sequences")


if __name__ == "__main__":
    main()
