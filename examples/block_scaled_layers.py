"""Generating tokens with decoder layers that norm their blocks on both sides, cap their scores and keep a block-scaled cache.

Random layers of the Llama-3-8B sizes (or the ones given) take ragged prompts, then one token per sequence and step, drawn from its
logits and captured once as a HIP graph:

    embedding -> add_rmsnorm -> [qkv linear -> mx_append -> mx_attention -> o_proj linear -> postnorm_add_rmsnorm
    -> gate+up, down linears -> postnorm_add_rmsnorm] x layers -> vocabulary linear -> sample_tokens

Every other layer attends within a window.  The norms hand their codes and scales to FP8 or INT8 linears, or 16-bit rows to
W4A16 ones; keys and values lie in one paged cache per layer, in 4 or 8 bits with a scale for each 32 columns.

    python examples/block_scaled_layers.py --layers 4 --batch 64 --prompt 1000 --linears fp8 --cache mxfp4
"""
from __future__ import annotations

import argparse
import os
import sys
import time

import torch
import torch.nn as nn

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))

from decoder_layers import QUANT, DecoderLayer, rope_table  # noqa: E402

from forge_amd import ops_decoder, ops_gemm, ops_mx  # noqa: E402
from forge_amd.ops_sampling import sample_tokens  # noqa: E402


class Layer(DecoderLayer):
    """A DecoderLayer with norms behind its blocks too; its own ``norms`` are those in front of them."""

    def __init__(self, hidden: int, heads: int, kv_heads: int, dim: int, ffn: int, kind: str, dtype: torch.dtype, softcap: float,
                 window: int | None) -> None:
        super().__init__(hidden, heads, kv_heads, dim, ffn, kind, dtype)
        self.softcap, self.window = softcap, window
        self.post = nn.ParameterList(nn.Parameter(torch.ones(hidden, device="cuda", dtype=dtype), requires_grad=False)
                                     for _ in range(2))

    def _linear(self, n: ops_decoder.NormOutput, linear: nn.Module, dtype: torch.dtype) -> torch.Tensor:
        if self.kind == "fp8":
            return ops_gemm.fp8_linear(n.y, linear.weight_fp8, linear.weight_scale, x_scale=n.scale, out_dtype=dtype)
        if self.kind == "int8":
            return ops_gemm.int8_linear(n.y, linear.weight_int8, linear.weight_scale, x_scale=n.scale, out_dtype=dtype)
        return linear(n.y)

    def forward(self, n, cache, positions, slots, table, next_norm, next_quant, **attention):
        """From the norm in front of this layer to the one in front of the next (``next_norm``, its codes ``next_quant``)."""
        h, hk, d = self.heads, self.kv_heads, self.dim
        dtype = n.residual.dtype
        qkv = self._linear(n, self.qkv, dtype)
        q, k, v = (t.view(-1, t.shape[1] // d, d) for t in qkv.split((h * d, hk * d, hk * d), dim=1))
        q = ops_mx.mx_append(q, k, v, positions, table, cache, slots, q_out=q)
        o = self.o(ops_mx.mx_attention(q, cache, softcap=self.softcap, window=self.window, **attention).view(-1, h * d))
        n = ops_decoder.postnorm_add_rmsnorm(o, self.post[0], n.residual, self.norms[1], quant=QUANT[self.kind])
        gate, up = self._linear(n, self.gate_up, dtype).chunk(2, dim=1)
        x = self.down(nn.functional.silu(gate) * up)
        return ops_decoder.postnorm_add_rmsnorm(x, self.post[1], n.residual, next_norm, quant=next_quant)


class Generator:
    """Layers, their caches and the batch's page tables, for ``batch`` sequences of up to ``length`` tokens."""

    def __init__(self, layers: int, batch: int, length: int, *, vocab: int = 32000, hidden: int = 4096, heads: int = 32,
                 kv_heads: int = 8, dim: int = 128, ffn: int = 14336, kind: str = "fp8", cache: str = "mxfp4", page: int = 16,
                 softcap: float = 50.0, window: int = 1024, dtype: torch.dtype = torch.bfloat16) -> None:
        self.layers = [Layer(hidden, heads, kv_heads, dim, ffn, kind, dtype, softcap, window if i % 2 else None) for i in range(layers)]
        width = -(-length // page)
        self.caches = [ops_mx.MXKVCache.allocate(batch * width, kv_heads, page, dim, cache) for _ in range(layers)]
        self.embedding = torch.randn(vocab, hidden, device="cuda").to(dtype)
        dense = nn.Linear(hidden, vocab, bias=False, device="cuda", dtype=dtype)
        nn.init.normal_(dense.weight, std=3 * hidden ** -0.5)
        self.head = ops_gemm.make_packed_linear(kind, dense)
        self.norm = torch.ones(hidden, device="cuda", dtype=dtype)
        self.table = rope_table(length, dim)
        self.length, self.page, self.batch, self.kind = length, page, batch, kind
        self.pages = torch.arange(batch * width, dtype=torch.int32, device="cuda").view(batch, width)
        self.lens = torch.zeros(batch, dtype=torch.int32, device="cuda")

    def _run(self, tokens, seq, at, **attention):
        """The normed stream behind the last layer, of tokens that stand at ``at`` of their sequences ``seq``."""
        slots = self.pages[seq, at // self.page] * self.page + at % self.page
        n = ops_decoder.add_rmsnorm(self.embedding[tokens], self.layers[0].norms[0], quant=QUANT[self.kind])
        for i, (layer, cache) in enumerate(zip(self.layers, self.caches)):
            last = i + 1 == len(self.layers)
            n = layer(n, cache, at, slots, self.table, self.norm if last else self.layers[i + 1].norms[0],
                      None if last else QUANT[self.kind], page_table=self.pages, seq_lens=self.lens, max_seq_len=self.length, **attention)
        return n.y

    def prompts(self, tokens: torch.Tensor, counts: list[int]) -> torch.Tensor:
        """Prompts of ``counts[b]`` tokens, one after the other; the logits behind each."""
        n = torch.tensor(counts, device="cuda")
        seq = torch.repeat_interleave(n)
        start = torch.cat((n[:1] * 0, n.cumsum(0)))
        at = torch.arange(len(seq), device="cuda") - start[seq] + self.lens[seq]
        self.lens += n.int()
        y = self._run(tokens, seq, at, query_start=start.int(), max_query_len=max(counts))
        return self.head(y[start[1:] - 1])

    def step(self, tokens: torch.Tensor) -> torch.Tensor:
        """One token for each sequence; the logits behind it.  No host synchronisation, so a HIP graph holds it."""
        at = self.lens.long()
        self.lens += 1
        return self.head(self._run(tokens, torch.arange(self.batch, device="cuda"), at))


def main() -> None:
    p = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    for name, default in (("layers", 4), ("batch", 64), ("prompt", 1000), ("steps", 64)):
        p.add_argument(f"--{name}", type=int, default=default)
    p.add_argument("--linears", choices=sorted(QUANT), default="fp8")
    p.add_argument("--cache", choices=("mxfp4", "mxfp8"), default="mxfp4")
    a = p.parse_args()
    torch.manual_seed(0)
    with torch.no_grad():
        g = Generator(a.layers, a.batch, a.prompt + a.steps + 8, kind=a.linears, cache=a.cache)
        counts = [max(1, a.prompt * (b + 1) // a.batch) for b in range(a.batch)]
        logits = g.prompts(torch.randint(0, 32000, (sum(counts),), device="cuda"), counts)
        uniform = torch.rand(a.batch, device="cuda")
        tokens = sample_tokens(logits, uniform, top_k=50, top_p=0.9, temperature=0.8)

        def step():
            tokens.copy_(sample_tokens(g.step(tokens), uniform, top_k=50, top_p=0.9, temperature=0.8))

        for _ in range(2):
            step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        torch.cuda.synchronize()
        t0 = time.perf_counter()
        for _ in range(a.steps):
            uniform.uniform_()
            graph.replay()
        torch.cuda.synchronize()
        dt = time.perf_counter() - t0
        print(f"decode: {dt / a.steps * 1e3:.2f} ms a step, {a.batch * a.steps / dt:.0f} tokens/s through {a.layers} layers; last tokens "
              f"{tokens[:4].tolist()} ..", flush=True)


if __name__ == "__main__":
    main()
