"""prefix_attention against its definition in 64 bits: prefixes and sequences from no token to several parts, every head
layout, page size and type, query tokens one by one and many, and what stands in places that it must not read."""
from __future__ import annotations

import pytest
import torch

from forge_amd import ops_decoder as ops
from forge_amd.errors import ConfigError
from tests._decoder_ref import assert_attention, attention_ref
from tests._util import gen

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF, E4 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


class _Call:
    """Inputs of one call on the GPU; every slot that holds no token holds NaN."""

    def __init__(self, queries, lens, prefix, h, hk, d, page, dt=BF, cdt=None, seed=0, ragged=None, width=None, gain=1.0):
        g = gen(seed + 7 * sum(lens) + prefix + d)
        cdt = cdt or dt
        b = len(lens)
        width = width or max(1, -(-max([*lens, 1]) // page))
        head = -(-prefix // page)
        pages = head + b * width + 2
        perm = torch.randperm(pages, generator=g).to(torch.int32)
        self.prefix_pages, self.prefix_len = perm[:head].to(DEV), prefix
        table = perm[head:head + b * width].view(b, width).clone()
        kv = []
        for _ in range(2):
            x = torch.randn(pages, hk, page, d, generator=g) * (20 if cdt == E4 else 1)
            real = torch.zeros(pages, page, dtype=torch.bool)
            for ids, n in [(perm[:head], prefix), *((table[i], lens[i]) for i in range(b))]:
                for t in range(n):
                    real[ids[t // page], t % page] = True
            x[~real.view(pages, 1, page, 1).expand_as(x)] = float("nan")
            kv.append(x.to(cdt).to(DEV))
        scales = ((torch.rand(hk, generator=g) * 0.05 + 0.03).to(DEV) for _ in range(2)) if cdt == E4 else (None, None)
        self.cache = ops.PagedKVCache(*kv, *scales)
        for i in range(b):  # entries past the length name no page at all
            table[i, -(-lens[i] // page):] = -1 if i % 2 else 2 ** 31 - 1
        self.table, self.lens = table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV)
        starts = [0]
        for n in queries:
            starts.append(starts[-1] + n)
        self.max_q = max([*queries, 1])
        ragged = any(n != 1 for n in queries) if ragged is None else ragged
        self.starts = torch.tensor(starts, dtype=torch.int32, device=DEV) if ragged else None
        self.q = (torch.randn(starts[-1], h, d, generator=g) * gain).to(dt).to(DEV)
        self.scale = d ** -0.5

    def run(self, **kw):
        kw = {"return_lse": True, **kw}
        return ops.prefix_attention(kw.pop("q", self.q), self.cache, self.table, self.lens, prefix_pages=self.prefix_pages,
                                    prefix_len=self.prefix_len, query_start=self.starts, max_query_len=self.max_q, **kw)

    def ref(self):
        return attention_ref(self.q, self.cache, self.table.cpu(), self.lens.cpu(), self.prefix_pages.cpu(), self.prefix_len,
                             None if self.starts is None else self.starts.cpu(), self.scale)

    def check(self, **kw):
        out, lse = self.run(**kw)
        assert_attention(out, lse, self.ref(), self.q.dtype)
        return out, lse


@pytest.mark.parametrize("dt,cdt", [(BF, BF), (HF, HF), (BF, E4), (HF, E4)])
@pytest.mark.parametrize("d", [64, 128, 256, 80, 96, 16, 208])
def test_head_sizes_and_types(d, dt, cdt):
    _Call([1] * 3, [33, 1, 150], 77, 8, 2, d, 16, dt, cdt).check()


@pytest.mark.parametrize("d", [8, 72, 136])
def test_head_sizes_of_whole_units(d):
    _Call([1, 1], [33, 70], 40, 4, 2, d, 16).check()


@pytest.mark.parametrize("h,hk", [(1, 1), (3, 3), (6, 2), (5, 1), (16, 1), (17, 1), (24, 1), (40, 1), (64, 8), (130, 2)])
def test_head_layouts(h, hk):
    _Call([1] * 2, [19, 130], 65, h, hk, 64, 16).check()


@pytest.mark.parametrize("page", [1, 3, 16, 48, 256])
def test_pages_end_inside_tiles(page):
    _Call([1] * 3, [31, 97, 260], 131, 4, 2, 64, page).check()


@pytest.mark.parametrize("prefix,lens", [(0, [1]), (0, [0]), (1, [0, 0]), (1, [1, 0]), (0, [0, 5, 0]), (16, [128, 129]), (4500, [3]),
                                         (0, [4500]), (2100, [2049, 1]), (500, [31, 32, 33, 64, 127, 128, 0, 1])])
def test_lengths(prefix, lens):
    _Call([1] * len(lens), lens, prefix, 4, 2, 64, 16).check()


@pytest.mark.parametrize("b", [1, 5, 9, 33, 70])
def test_batches(b):
    """The prefix's rows are those of the whole batch: from one tile to several."""
    _Call([1] * b, [(7 * i) % 50 for i in range(b)], 200, 8, 2, 64, 16).check()


@pytest.mark.parametrize("dt,cdt", [(BF, BF), (HF, HF), (BF, E4)])
@pytest.mark.parametrize("queries,lens,prefix", [([2, 1, 3], [2, 1, 3], 0), ([4, 4], [100, 37], 64), ([1, 40, 7], [300, 40, 9], 33),
                                                 ([150, 3], [150, 200], 10), ([5, 0, 2], [5, 9, 2], 3), ([70], [70], 0)])
def test_several_query_tokens(queries, lens, prefix, dt, cdt):
    _Call(queries, lens, prefix, 6, 2, 64, 16, dt, cdt).check()
    _Call(queries, lens, prefix, 4, 4, 128, 16, dt, cdt).check()


def test_more_query_tokens_than_cached_tokens():
    """The first queries of such a sequence stand before its first token: they see the prefix, or nothing."""
    _Call([4, 3], [2, 0], 20, 4, 2, 64, 16).check()
    c = _Call([4, 3], [2, 0], 0, 4, 2, 64, 16)
    out, lse = c.check()
    assert bool((out[:2] == 0).all()) and bool((lse[4:] == float("-inf")).all())


def test_one_query_token_each_with_starts():
    c = _Call([1] * 4, [5, 0, 77, 20], 40, 8, 2, 64, 16, ragged=True)
    ragged = c.check()
    c.starts = None
    assert all(torch.equal(a, b) for a, b in zip(ragged, c.run()))


def test_large_scores_and_constant_rows():
    """Scores far apart move the running maximum in many tiles; equal ones never."""
    _Call([1] * 3, [700, 40, 300], 900, 4, 2, 128, 16, gain=30.0).check()
    c = _Call([1] * 3, [700, 40, 300], 900, 4, 2, 128, 16)
    c.q.zero_()
    c.check()


def test_strides_and_out():
    c = _Call([1] * 3, [33, 5, 150], 77, 8, 2, 64, 16)
    want, lse = c.check()
    wide = torch.zeros(3, 9, 67, dtype=BF, device=DEV)
    q = wide[:, 1:, 3:].copy_(c.q)
    out = torch.full((3, 8, 65), 7.0, dtype=BF, device=DEV)[..., 1:]
    got, got_lse = c.run(q=q, out=out)
    assert got is out and torch.equal(out, want) and torch.equal(lse, got_lse)
    turned = c.q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(c.run(q=turned)[0], want)
    # a token-major cache, a page table that is a view
    k, v = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (c.cache.k, c.cache.v))
    c.cache = ops.PagedKVCache(k, v)
    c.table = torch.cat((c.table, c.table), 1)[:, :c.table.shape[1]]
    assert torch.equal(c.run()[0], want)


def test_scale_and_no_lse():
    c = _Call([1] * 2, [33, 70], 40, 4, 2, 64, 16)
    c.scale = 0.31
    out, _ = c.check(scale=0.31)
    assert torch.equal(ops.prefix_attention(c.q, c.cache, c.table, c.lens, prefix_pages=c.prefix_pages, prefix_len=40, scale=0.31), out)


def test_max_seq_len_bounds_the_lengths():
    """A bound above the lengths changes nothing but the split; lengths above it are cut."""
    c = _Call([1] * 3, [33, 5, 150], 77, 8, 2, 64, 16, width=40)
    want = c.ref()
    for bound in (150, 151, 640):
        assert_attention(*c.run(max_seq_len=bound), want, BF)
    cut = _Call([1] * 3, [33, 5, 150], 77, 8, 2, 64, 16, width=40)
    got = cut.run(max_seq_len=100)
    cut.lens.clamp_(max=100)
    assert_attention(*got, cut.ref(), BF)


def test_tokens_of_no_sequence_and_past_the_longest():
    c = _Call([2, 3], [20, 9], 30, 4, 2, 64, 16)
    want = c.ref()
    c.q = torch.cat((c.q, torch.ones(3, 4, 64, dtype=BF, device=DEV)))
    out, lse = c.run()
    assert_attention(out[:5], lse[:5], want, BF)
    assert bool((out[5:] == 0).all()) and bool((lse[5:] == float("-inf")).all())
    c.max_q = 2
    out, lse = c.run()
    assert bool(out[4].isnan().all()) and bool(lse[4].isnan().all())
    assert torch.equal(out[:4].isnan().any(), torch.tensor(False, device=DEV))
    assert_attention(out[:4], lse[:4], tuple(x[:4] for x in want), BF)


def test_pages_outside_the_cache_hold_no_tokens():
    c = _Call([1, 1], [90, 100], 64, 4, 2, 64, 16)
    c.table[0, 1], c.table[1, 3], c.prefix_pages[2] = -5, 10 ** 6, 2 ** 31 - 1
    c.check()


def test_infinite_and_nan_keys_show():
    c = _Call([1, 1], [90, 100], 0, 4, 2, 64, 16)
    c.cache.v[c.table[0, 2], :, 3, 5] = float("inf")
    c.cache.k[c.table[1, 0], 0, 1, :] = float("nan")
    out, lse = c.run()
    assert bool((out[0, :, 5] == float("inf")).all()) and bool(out[0, :, 6].isfinite().all())
    assert bool(out[1, :2].isnan().all()) and bool(lse[1, :2].isnan().all()) and bool(out[1, 2:].isfinite().all())


def test_equal_calls_give_equal_bits():
    c = _Call([1] * 6, [33, 5, 150, 800, 2, 0], 300, 8, 2, 128, 16)
    first = c.run()
    assert all(torch.equal(a, b) for _ in range(3) for a, b in zip(first, c.run()))


def test_another_stream_and_a_graph():
    """On the caller's stream; captured once, replayed with other lengths, queries and cache contents."""
    c = _Call([1] * 4, [40, 7, 200, 90], 150, 8, 2, 64, 16, width=20)
    want = c.run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = c.run()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = c.run()
    for seed in range(3):
        n = _Call([1] * 4, [3 + 50 * seed, 100 - 40 * seed, 5, 0 if seed == 1 else 77], 150, 8, 2, 64, 16, width=20, seed=seed)
        for a in ("q", "table", "lens", "prefix_pages"):
            getattr(c, a).copy_(getattr(n, a))
        c.cache.k.copy_(n.cache.k)
        c.cache.v.copy_(n.cache.v)
        graph.replay()
        torch.cuda.synchronize()
        assert_attention(out, lse, n.ref(), BF)
        assert all(torch.equal(a, b) for a, b in zip((out, lse), c.run()))


def test_a_cache_past_32_bits():
    """Rows of pages more than 4 GiB from the first: their byte offsets pass 32 bits."""
    page, hk, d = 256, 8, 128
    pages = (9 << 30) // (2 * page * hk * d)  # 9 GiB of keys, as much of values
    cache = ops.PagedKVCache(*(torch.empty(pages, hk, page, d, dtype=BF, device=DEV) for _ in range(2)))
    ids = [pages - 1, 3, pages // 2, pages - 7]
    for x in (cache.k, cache.v):
        for p in ids:
            x[p].normal_()
    c = _Call([1] * 2, [300, 400], 0, 16, hk, d, page)
    c.table = torch.tensor([ids[:2], ids[2:]], dtype=torch.int32, device=DEV)
    small = ops.PagedKVCache(cache.k[ids].cpu(), cache.v[ids].cpu())
    c.cache = cache
    out, lse = c.run()
    want = attention_ref(c.q, small, torch.tensor([[0, 1], [2, 3]]), c.lens.cpu(), torch.zeros(0), 0, None, c.scale)
    assert_attention(out, lse, want, BF)
    slots = torch.tensor([(pages - 1) * page + 7, 5], device=DEV)
    k = torch.randn(2, hk, d, device=DEV).to(BF)
    table = torch.cat((torch.ones(1, d // 2), torch.zeros(1, d // 2)), 1).to(DEV)
    ops.rope_append(c.q, k, k, torch.zeros(2, dtype=torch.int64, device=DEV), table, cache, slots)
    assert torch.equal(cache.k[pages - 1, :, 7], k[0]) and torch.equal(cache.v[0, :, 5], k[1])


def test_no_queries_no_sequences():
    c = _Call([1], [5], 10, 4, 2, 64, 16)
    none = torch.zeros(0, dtype=torch.int32, device=DEV)
    assert ops.prefix_attention(c.q[:0], c.cache, c.table[:0], none).shape == (0, 4, 64)
    out, lse = ops.prefix_attention(c.q, c.cache, c.table[:0], none, query_start=torch.zeros(1, dtype=torch.int32, device=DEV),
                                    prefix_pages=c.prefix_pages, prefix_len=10, return_lse=True)
    assert bool((out == 0).all()) and bool((lse == float("-inf")).all())


def test_refusals():
    c = _Call([1, 1], [9, 20], 40, 4, 2, 64, 16)
    call = dict(q=c.q, cache=c.cache, page_table=c.table, seq_lens=c.lens, prefix_pages=c.prefix_pages, prefix_len=40)
    i64 = c.lens.long()
    for bad in (dict(q=c.q[:1]), dict(q=c.q.half()), dict(q=c.q[:, :3]), dict(q=c.q[..., :32]), dict(page_table=c.table.long()),
                dict(seq_lens=i64), dict(seq_lens=c.lens[:1]), dict(prefix_len=49), dict(prefix_pages=None), dict(prefix_len=-1),
                dict(max_seq_len=33), dict(max_seq_len=-1), dict(max_query_len=2), dict(max_query_len=0),
                dict(query_start=c.lens), dict(seq_lens=c.lens.cpu()), dict(out=c.q[:1]), dict(prefix_pages=c.prefix_pages.long())):
        with pytest.raises(ConfigError):
            ops.prefix_attention(**{**call, **bad})
    big = ops.PagedKVCache.allocate(1, 2, 16, 264, BF, DEV)
    with pytest.raises(Exception, match="head_dim"):
        ops.prefix_attention(torch.zeros(2, 4, 264, dtype=BF, device=DEV), big, c.table, c.lens)
    odd = ops.PagedKVCache.allocate(1, 2, 16, 72, E4, DEV)
    with pytest.raises(Exception, match="head_dim"):
        ops.prefix_attention(torch.zeros(2, 4, 72, dtype=BF, device=DEV), odd, c.table, c.lens)


def test_one_page_list_for_all_sequences():
    c = _Call([1] * 3, [33, 20, 40], 0, 8, 2, 64, 16)
    c.table = torch.tensor([[7, 1, 4]], dtype=torch.int32, device=DEV)
    for x in (c.cache.k, c.cache.v):
        x[[7, 1, 4]] = 1.0
        x[[7, 1, 4], :, 3] = -0.5
    c.table = c.table.repeat(3, 1)
    want = c.check()
    c.table = c.table[:1].expand(3, 3)
    assert all(torch.equal(a, b) for a, b in zip(want, c.run()))
