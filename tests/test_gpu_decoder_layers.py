"""The example's decoder layers: the shared prompt, prompts and single tokens of a batch give what the same tokens give when
each sequence is one prompt of its own, and a captured step what the eager one does."""
from __future__ import annotations

import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))

pytestmark = pytest.mark.gpu
SIZES = dict(hidden=256, heads=8, kv_heads=2, dim=64, ffn=512)


def _server(layers, batch, prefix, own, kind, cache, share=None):
    from decoder_layers import Server

    torch.manual_seed(3)
    s = Server(layers, batch, prefix, own, kind=kind, cache=cache, **SIZES)
    if share is not None:
        s.layers = share.layers
    return s


@pytest.mark.parametrize("kind,cache", [("fp8", "bf16"), ("int8", "fp8"), ("w4a16", "bf16")])
def test_batch_behind_a_shared_prompt_equals_prompts_of_their_own(kind, cache):
    prefix, counts, steps = 50, [3, 17, 9], 4
    g = torch.Generator("cuda").manual_seed(1)
    shared = torch.randn(prefix, 256, generator=g, device="cuda").bfloat16()
    own = [torch.randn(n + steps, 256, generator=g, device="cuda").bfloat16() for n in counts]
    with torch.no_grad():
        s = _server(2, 3, prefix, 40, kind, cache)
        s.shared_prompt(shared)
        s.prompts(torch.cat([x[:n] for x, n in zip(own, counts)]), counts)
        got = [s.step(torch.stack([x[n + i] for x, n in zip(own, counts)])) for i in range(steps)]
        for b, (x, n) in enumerate(zip(own, counts)):
            whole = torch.cat((shared, x))
            alone = _server(2, 1, len(whole), 1, kind, cache, share=s).shared_prompt(whole)
            ref = alone[-steps:].float()
            y = torch.stack([t[b] for t in got]).float()
            # the same sums in other orders: 16-bit roundings and, at their edges, 8-bit codes differ by single steps
            assert (y - ref).norm() <= 0.05 * ref.norm(), b


def test_a_captured_step_equals_the_eager_one():
    with torch.no_grad():
        a, x = _server(2, 5, 30, 40, "fp8", "bf16"), torch.randn(5, 256, device="cuda").bfloat16()
        b = _server(2, 5, 30, 40, "fp8", "bf16", share=a)
        shared = torch.randn(30, 256, device="cuda").bfloat16()
        for s in (a, b):
            s.shared_prompt(shared)
            s.step(x)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = a.step(x)
        for _ in range(4):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, b.step(x)) and torch.equal(a.lens, b.lens)
