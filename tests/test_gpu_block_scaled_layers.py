"""The example's layers, all of the operators together: a batch of ragged prompts and single tokens gives the logits that each
sequence gives by itself, a captured step with its draw the tokens of the eager one, and the first step the formulas' logits."""
from __future__ import annotations

import os
import sys

import pytest
import torch

from forge_amd.ops_sampling import sample_tokens

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))

pytestmark = pytest.mark.gpu
SIZES = dict(vocab=1000, hidden=256, heads=8, kv_heads=2, dim=64, ffn=512, window=12, softcap=5.0)


def _generator(layers, batch, length, kind, cache, share=None):
    from block_scaled_layers import Generator

    torch.manual_seed(3)
    s = Generator(layers, batch, length, kind=kind, cache=cache, **SIZES)
    if share is not None:
        s.layers, s.embedding, s.head = share.layers, share.embedding, share.head
    return s


@pytest.mark.parametrize("kind,cache", [("fp8", "mxfp8"), ("int8", "mxfp4"), ("w4a16", "mxfp8")])
def test_a_batch_equals_its_sequences_alone(kind, cache):
    counts, steps = [3, 40, 17], 4
    g = torch.Generator("cuda").manual_seed(1)
    own = [torch.randint(0, 1000, (n + steps,), generator=g, device="cuda") for n in counts]
    with torch.no_grad():
        s = _generator(2, 3, 48, kind, cache)
        got = [s.prompts(torch.cat([x[:n] for x, n in zip(own, counts)]), counts)]
        got += [s.step(torch.stack([x[n + i] for x, n in zip(own, counts)])) for i in range(steps)]
        for b, (x, n) in enumerate(zip(own, counts)):
            alone = _generator(2, 1, 48, kind, cache, share=s)
            ref = [alone.prompts(x[:n], [n])] + [alone.step(x[n + i:n + i + 1]) for i in range(steps)]
            y, r = torch.stack([t[b] for t in got]).float(), torch.cat(ref).float()
            # the same sums in other orders: 16-bit roundings and, at their edges, codes differ by single steps
            assert (y - r).norm() <= 0.05 * r.norm(), b


def test_a_captured_step_draws_the_tokens_of_the_eager_one():
    with torch.no_grad():
        a = _generator(2, 5, 40, "fp8", "mxfp4")
        b = _generator(2, 5, 40, "fp8", "mxfp4", share=a)
        uniform = torch.rand(5, device="cuda")
        counts = [1, 9, 4, 20, 2]
        prompt = torch.randint(0, 1000, (sum(counts),), device="cuda")
        tokens = [sample_tokens(s.prompts(prompt, counts), uniform, top_k=30) for s in (a, b)]
        assert torch.equal(*tokens)

        def step(s, t):
            t.copy_(sample_tokens(s.step(t), uniform, top_k=30, top_p=0.95))

        for s, t in zip((a, b), tokens):
            step(s, t)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step(a, tokens[0])
        for _ in range(4):
            uniform.uniform_()
            graph.replay()
            torch.cuda.synchronize()
            step(b, tokens[1])
            assert torch.equal(tokens[0], tokens[1]) and torch.equal(a.lens, b.lens)


def test_one_layer_against_the_formulas():
    """A prompt through one layer on W4A16 linears, with the steps in fp32 torch over what the cache reads back."""
    from forge_amd import ops_mx

    with torch.no_grad():
        s = _generator(1, 1, 32, "w4a16", "mxfp8")
        layer, n = s.layers[0], 20
        tokens = torch.randint(0, 1000, (n,), device="cuda")
        got = s.prompts(tokens, [n]).float()

        def norm(x):
            return x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-5)

        r = s.embedding[tokens].float()
        qkv = layer.qkv(norm(r).bfloat16()).float()
        q = qkv[:, :512].view(n, 8, 64)
        cos, sin = s.table[:n].unsqueeze(1).chunk(2, -1)
        a, b = q[..., :32], q[..., 32:]
        q = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
        slots = s.pages[0, torch.arange(n, device="cuda") // 16] * 16 + torch.arange(n, device="cuda") % 16
        k, v = (t.float().repeat_interleave(4, 1) for t in ops_mx.mx_read(s.caches[0], slots.long()))
        scores = 5.0 * torch.tanh(torch.matmul(q.transpose(0, 1), k.permute(1, 2, 0).contiguous()) / 8 / 5.0)
        scores = scores.masked_fill(torch.ones(n, n, device="cuda").triu(1).bool(), -float("inf"))
        o = layer.o(torch.matmul(torch.softmax(scores, -1), v.transpose(0, 1).contiguous()).transpose(0, 1).reshape(n, -1).bfloat16()).float()
        r = r + norm(o)
        gate, up = layer.gate_up(norm(r).bfloat16()).float().chunk(2, 1)
        r = r + norm(layer.down((torch.nn.functional.silu(gate) * up).bfloat16()).float())
        ref = s.head(norm(r).bfloat16()[-1:]).float()
        # 16-bit roundings between the steps, of the residual stream among them
        assert (got - ref).norm() <= 0.03 * ref.norm()
