"""Rows, pages and tokens whose offsets pass 32 bits, and caches in other orders: the same bits as rows that lie side by side."""
from __future__ import annotations

import pytest
import torch

from forge_amd import ops_mx as mx
from forge_amd.ops_decoder import postnorm_add_rmsnorm
from forge_amd.ops_sampling import sample_tokens
from tests._util import gen

pytestmark = pytest.mark.gpu
DEV = "cuda"
PAGES, HK, PAGE, D = 4, 2, 16, 64
GIB = 1 << 30
ROW = {4: 32, 8: 64}  # bytes


def _orders(bits):
    row = ROW[bits]
    return {"tokens first": (HK * PAGE * row, row, HK * row), "heads first": (PAGE * row, PAGES * PAGE * row, row),
            "far pages": (12 * GIB, PAGE * row, row), "far heads": (PAGE * row, 40 * GIB, row), "far tokens": (4 * row, row, 9 * GIB // 4)}


@pytest.mark.parametrize("order", ["tokens first", "heads first", "far pages", "far heads", "far tokens"])
@pytest.mark.parametrize("bits", [4, 8])
def test_caches_of_any_order(bits, order):
    fmt, row, strides = {4: "mxfp4", 8: "mxfp8"}[bits], ROW[bits], _orders(bits)[order]
    g = gen(bits)
    near = mx.MXKVCache.allocate(PAGES, HK, PAGE, D, fmt)
    span = sum(s * (n - 1) for s, n in zip(strides, (PAGES, HK, PAGE))) + row
    apart = -(-span // 4096) * 4096 if span < GIB else 4096 * row  # the values behind the keys, or in their gaps
    codes = torch.empty(span + apart, dtype=torch.uint8, device=DEV)
    scales = torch.empty((span + apart) // (4 * bits) + 2, dtype=torch.uint8, device=DEV)
    far = mx.MXKVCache(*(codes.as_strided((PAGES, HK, PAGE, row), (*strides, 1), i * apart) for i in range(2)),
                       *(scales.as_strided((PAGES, HK, PAGE, D // 32), (*(s // (4 * bits) for s in strides), 1), i * apart // (4 * bits))
                         for i in range(2)))
    n = PAGES * PAGE
    q, k, v = (torch.randn(n, h, D, generator=g).bfloat16().to(DEV) for h in (4, HK, HK))
    table = torch.randn(100, D, generator=g).to(DEV)
    positions, slots = torch.arange(n, device=DEV), torch.randperm(n, generator=g).to(DEV)
    turned = [mx.mx_append(q, k, v, positions, table, c, slots) for c in (near, far)]
    assert torch.equal(*turned)
    for name in ("k", "v", "k_scale", "v_scale"):
        assert torch.equal(getattr(near, name), getattr(far, name)), name
    assert all(torch.equal(a, b) for a, b in zip(mx.mx_read(near, slots), mx.mx_read(far, slots)))
    pages = torch.tensor([[3, 0, 2, 1], [1, 2, -1, -1]], dtype=torch.int32, device=DEV)
    lens = torch.tensor([61, 30], dtype=torch.int32, device=DEV)
    starts = torch.tensor([0, 40, 45], dtype=torch.int32, device=DEV)
    for kw in (dict(q=turned[0][:2]), dict(q=turned[0][:45], query_start=starts, max_query_len=40, softcap=20.0, window=25)):
        query = kw.pop("q")
        got = [mx.mx_attention(query, c, pages, lens, return_lse=True, **kw) for c in (near, far)]
        assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])


def test_rows_past_32_bits():
    ld = 2 ** 31 + 16
    base = torch.empty(2 * ld + 5000, dtype=torch.bfloat16, device=DEV)
    g = gen(5)
    far, near = base.as_strided((3, 5000), (ld, 1)), (3 * torch.randn(3, 5000, generator=g)).bfloat16().to(DEV)
    far.copy_(near)
    u = torch.rand(3, generator=g).to(DEV)
    for kw in (dict(), dict(top_k=20), dict(top_p=0.9)):
        got, want = (sample_tokens(x, u, return_logprobs=True, **kw) for x in (far, near))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    r, w = torch.randn(3, 5000, generator=g).to(DEV), torch.randn(5000, generator=g).to(DEV)
    got, want = (postnorm_add_rmsnorm(x, w, r, w, gate=x, quant="int8") for x in (far, near))
    assert all(torch.equal(getattr(got, n), getattr(want, n)) for n in ("y", "scale", "residual"))
    out = base.as_strided((3, 5000), (ld, 1))
    h = near.clone()
    got, want = postnorm_add_rmsnorm(near, w, h, w, residual_out=out), postnorm_add_rmsnorm(near, w, h, w)
    assert got.residual is out and torch.equal(got.residual, want.residual) and torch.equal(got.y, want.y)
