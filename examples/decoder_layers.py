"""Serving decoder layers on quantised linears: a batch of sequences behind one shared prompt.

Random layers of the Llama-3-8B sizes (or the ones given) take a shared prompt, then a prompt of its own for each sequence,
then one token per sequence and step, captured once as a HIP graph:

    add_rmsnorm -> qkv linear -> rope_append -> prefix_attention -> o_proj linear -> add_rmsnorm -> gate+up, down linears

The norms hand their codes and scales to FP8 or INT8 linears, or 16-bit rows to W4A16 ones; keys and values lie in one paged
cache per layer, in 16 bits or e4m3.

    python examples/decoder_layers.py --layers 4 --batch 64 --prefix 8192 --linears fp8 --cache fp8
"""
from __future__ import annotations

import argparse
import os
import sys
import time

import torch
import torch.nn as nn

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "forge-llm_amd"))

from forge_amd import ops_decoder, ops_gemm  # noqa: E402
from forge_amd.ops_decoder import PagedKVCache  # noqa: E402

QUANT = {"fp8": "fp8", "int8": "int8", "w4a16": None}  # what the norm in front of a linear gives it


def rope_table(positions: int, dim: int, base: float = 500000.0, device: str = "cuda") -> torch.Tensor:
    angle = torch.arange(positions, device=device).view(-1, 1) * torch.pow(
        torch.tensor(base, device=device), -torch.arange(0, dim, 2, device=device) / dim)
    return torch.cat((angle.cos(), angle.sin()), 1)


class DecoderLayer(nn.Module):
    def __init__(self, hidden: int, heads: int, kv_heads: int, dim: int, ffn: int, kind: str, dtype: torch.dtype) -> None:
        super().__init__()
        self.heads, self.kv_heads, self.dim, self.kind = heads, kv_heads, dim, kind

        def linear(n: int, k: int) -> nn.Module:
            dense = nn.Linear(k, n, bias=False, device="cuda", dtype=dtype)
            nn.init.normal_(dense.weight, std=k ** -0.5)
            return ops_gemm.make_packed_linear(kind, dense)

        self.qkv, self.o = linear((heads + 2 * kv_heads) * dim, hidden), linear(hidden, heads * dim)
        self.gate_up, self.down = linear(2 * ffn, hidden), linear(hidden, ffn)
        self.norms = nn.ParameterList(nn.Parameter(torch.ones(hidden, device="cuda", dtype=dtype), requires_grad=False)
                                      for _ in range(2))

    def _normed(self, x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None, linear: nn.Module):
        """The linear of the normed residual stream, and the stream: codes and scales go from the norm to the linear."""
        n = ops_decoder.add_rmsnorm(x, weight, residual, quant=QUANT[self.kind])
        if self.kind == "fp8":
            y = ops_gemm.fp8_linear(n.y, linear.weight_fp8, linear.weight_scale, x_scale=n.scale, out_dtype=x.dtype)
        elif self.kind == "int8":
            y = ops_gemm.int8_linear(n.y, linear.weight_int8, linear.weight_scale, x_scale=n.scale, out_dtype=x.dtype)
        else:
            y = linear(n.y)
        return y, n.residual

    def forward(self, x, residual, cache: PagedKVCache, positions, slots, table, **attention):
        """``x`` and the residual stream ``[tokens, hidden]`` (None in front of the first layer) of tokens that stand at
        ``positions`` and go to ``slots`` of the cache; ``attention``: prefix_attention's lengths and page tables."""
        h, hk, d = self.heads, self.kv_heads, self.dim
        qkv, residual = self._normed(x, self.norms[0], residual, self.qkv)
        q, k, v = (t.view(-1, t.shape[1] // d, d) for t in qkv.split((h * d, hk * d, hk * d), dim=1))
        q = ops_decoder.rope_append(q, k, v, positions, table, cache, slots, q_out=q)
        o = self.o(ops_decoder.prefix_attention(q, cache, **attention).view(-1, h * d))
        gate_up, residual = self._normed(o, self.norms[1], residual, self.gate_up)
        gate, up = gate_up.chunk(2, dim=1)
        return self.down(nn.functional.silu(gate) * up), residual


class Server:
    """Layers, their caches and the batch's page tables: one shared prompt, ``batch`` sequences of up to ``own`` tokens."""

    def __init__(self, layers: int, batch: int, prefix: int, own: int, *, hidden: int = 4096, heads: int = 32,
                 kv_heads: int = 8, dim: int = 128, ffn: int = 14336, kind: str = "fp8", cache: str = "bf16", page: int = 16,
                 dtype: torch.dtype = torch.bfloat16) -> None:
        self.layers = [DecoderLayer(hidden, heads, kv_heads, dim, ffn, kind, dtype) for _ in range(layers)]
        head, width = -(-prefix // page), -(-own // page)
        kv = dtype if cache != "fp8" else torch.float8_e4m3fn
        scales = [torch.full((kv_heads,), 0.02, device="cuda") for _ in range(2)] if cache == "fp8" else [None, None]
        self.caches = [PagedKVCache.allocate(head + batch * width, kv_heads, page, dim, kv, "cuda", *scales) for _ in range(layers)]
        self.table = rope_table(prefix + own, dim)
        self.prefix, self.own, self.page, self.batch = prefix, own, page, batch
        ids = torch.arange(head + batch * width, dtype=torch.int32, device="cuda")
        self.prefix_pages, self.pages = ids[:head], ids[head:].view(batch, width)
        self.lens = torch.zeros(batch, dtype=torch.int32, device="cuda")  # own tokens in the cache

    def _run(self, x, positions, slots, **attention):
        residual = None
        for layer, cache in zip(self.layers, self.caches):
            x, residual = layer(x, residual, cache, positions, slots, self.table, **attention)
        return x + residual

    def shared_prompt(self, x: torch.Tensor) -> torch.Tensor:
        """The shared prompt's tokens ``[prefix, hidden]``: a sequence of their own in the prefix's pages."""
        at = torch.arange(self.prefix, device="cuda")
        slots = self.prefix_pages[at // self.page] * self.page + at % self.page
        one = torch.tensor([self.prefix], dtype=torch.int32, device="cuda")
        return self._run(x, at, slots.long(), page_table=self.prefix_pages.view(1, -1), seq_lens=one,
                         query_start=torch.cat((one * 0, one)), max_query_len=self.prefix)

    def _slots(self, seq: torch.Tensor, at: torch.Tensor) -> torch.Tensor:
        return self.pages[seq, at // self.page] * self.page + at % self.page

    def prompts(self, x: torch.Tensor, counts: list[int]) -> torch.Tensor:
        """A prompt of ``counts[b]`` tokens for each sequence, one after the other in ``x``."""
        n = torch.tensor(counts, device="cuda")
        seq = torch.repeat_interleave(n)
        start = torch.cat((n[:1] * 0, n.cumsum(0)))
        at = torch.arange(len(seq), device="cuda") - start[seq] + self.lens[seq]
        self.lens += n.int()
        return self._run(x, self.prefix + at, self._slots(seq, at), page_table=self.pages, seq_lens=self.lens,
                         prefix_pages=self.prefix_pages, prefix_len=self.prefix, query_start=start.int(),
                         max_query_len=max(counts), max_seq_len=self.own)

    def step(self, x: torch.Tensor) -> torch.Tensor:
        """One token for each sequence: no host synchronisation, so a HIP graph holds it."""
        at = self.lens.long()
        self.lens += 1
        seq = torch.arange(self.batch, device="cuda")
        return self._run(x, self.prefix + at, self._slots(seq, at), page_table=self.pages, seq_lens=self.lens,
                         prefix_pages=self.prefix_pages, prefix_len=self.prefix, max_seq_len=self.own)


def main() -> None:
    p = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    for name, default in (("layers", 4), ("batch", 64), ("prefix", 8192), ("prompt", 256), ("steps", 64)):
        p.add_argument(f"--{name}", type=int, default=default)
    p.add_argument("--linears", choices=sorted(QUANT), default="fp8")
    p.add_argument("--cache", choices=("bf16", "fp8"), default="bf16")
    a = p.parse_args()
    torch.manual_seed(0)
    with torch.no_grad():
        s = Server(a.layers, a.batch, a.prefix, a.prompt + a.steps + 8, kind=a.linears, cache=a.cache)

        def timed(name, fn, tokens):
            torch.cuda.synchronize()
            t0 = time.perf_counter()
            fn()
            torch.cuda.synchronize()
            dt = time.perf_counter() - t0
            print(f"{name}: {dt * 1e3:.2f} ms, {tokens / dt:.0f} tokens/s through {a.layers} layers", flush=True)

        def tokens(n):
            return torch.randn(n, 4096, device="cuda").bfloat16()

        shared, own = tokens(a.prefix), tokens(a.batch * a.prompt)
        s.shared_prompt(shared)  # the first call of each kernel
        timed("shared prompt", lambda: s.shared_prompt(shared), a.prefix)
        timed("own prompts", lambda: s.prompts(own, [a.prompt] * a.batch), a.batch * a.prompt)
        x = tokens(a.batch)
        for _ in range(2):
            s.step(x)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            s.step(x)
        timed("decode", lambda: [graph.replay() for _ in range(a.steps)], a.batch * a.steps)


if __name__ == "__main__":
    main()
