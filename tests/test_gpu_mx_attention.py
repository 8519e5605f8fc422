"""mx_attention against its definition in 64 bits: both formats, lengths from no token to several parts, every head layout and
page size, windows and caps, query tokens one by one and many, and what stands in places that it must not read."""
from __future__ import annotations

import pytest
import torch

from forge_amd import ops_gemm
from forge_amd import ops_mx as mx
from forge_amd.errors import ConfigError
from tests._decoder_ref import HALF_ULP
from tests._mx_ref import capped_attention_ref, decode_ref, encode_ref, pack_ref
from tests._util import gen

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF = torch.bfloat16, torch.float16


class _Call:
    """Inputs of one call on the GPU; every slot that holds no token holds NaN blocks."""

    def __init__(self, queries, lens, h, hk, d, page, bits=4, dt=BF, seed=0, ragged=None, width=None, gain=1.0, softcap=None, window=None):
        g = gen(seed + 7 * sum(lens) + d + bits)
        b = len(lens)
        width = width or max(1, -(-max([*lens, 1]) // page))
        pages = b * width + 2
        perm = torch.randperm(pages, generator=g).to(torch.int32)
        table = perm[:b * width].view(b, width).clone()
        real = torch.zeros(pages, page, dtype=torch.bool)
        for i in range(b):
            at = torch.arange(lens[i])
            real[table[i][at // page].long(), at % page] = True
        parts = []
        for _ in range(2):
            codes, scales = encode_ref(torch.randn(pages, hk, page, d, generator=g), bits)
            codes[~real.view(pages, 1, page, 1).expand_as(codes)] = 3
            scales[~real.view(pages, 1, page, 1).expand_as(scales)] = 255
            parts += [pack_ref(codes, bits), scales.to(torch.uint8)]
        self.cache = mx.MXKVCache(*(parts[i].to(DEV) for i in (0, 2, 1, 3)))
        for i in range(b):  # entries past the length name no page at all
            table[i, -(-lens[i] // page):] = -1 if i % 2 else 2 ** 31 - 1
        self.table, self.lens, self.n = table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV), lens
        self.first = [0]
        for n in queries:
            self.first.append(self.first[-1] + n)
        self.max_q = max([*queries, 1])
        ragged = any(n != 1 for n in queries) if ragged is None else ragged
        self.starts = torch.tensor(self.first, dtype=torch.int32, device=DEV) if ragged else None
        self.q = (torch.randn(self.first[-1], h, d, generator=g) * gain).to(dt).to(DEV)
        self.kw = {"softcap": softcap, "window": window}

    def run(self, **kw):
        kw = {"return_lse": True, **self.kw, **kw}
        return mx.mx_attention(kw.pop("q", self.q), self.cache, self.table, self.lens, query_start=self.starts, max_query_len=self.max_q,
                               **kw)

    def tokens(self):
        """Keys, values, and which are there, sequence by sequence."""
        c, page = self.cache, self.cache.page_size
        values = [decode_ref(x, s, c.bits) for x, s in ((c.k, c.k_scale), (c.v, c.v_scale))]
        got = [], [], []
        for row, n in zip(self.table.cpu(), self.n):
            at = torch.arange(n)
            ids = row[at // page].long()
            inside = (ids >= 0) & (ids < c.k.shape[0])
            for to, x in zip(got, values):
                to.append(x[ids.clamp(0, c.k.shape[0] - 1), :, at % page].transpose(0, 1))
            got[2].append(inside)
        return got

    def check(self, scale=None, **kw):
        out, lse = self.run(scale=scale, **kw)
        k, v, present = self.tokens()
        cap, window = kw.get("softcap", self.kw["softcap"]), kw.get("window", self.kw["window"])
        ref, ref_lse, mag = capped_attention_ref(self.q, k, v, present, self.n, self.first, self.q.shape[2] ** -0.5 if scale is None else scale,
                                                 cap, window)
        u, tiny = HALF_ULP[self.q.dtype]
        # each probability and the result are rounded once; scores, exponents and sums are fp32, of which the scores' rounding
        # (2^-22 of sums of up to a few hundred, twice) and the cap's (2^-20 of it, twice) are the largest
        slack = 2.0 ** -12 + (2.0 ** -19 * cap if cap else 0.0)
        err, tol = (out.cpu().double() - ref).abs(), (u + slack) * mag + u * ref.abs() + tiny
        assert bool((err <= tol).all()), f"off by {(err / tol.clamp_min(1e-300)).max().item():.3g} of the tolerance"
        lse = lse.cpu().double()
        fine = torch.isfinite(ref_lse)
        assert torch.equal(fine, torch.isfinite(lse)) and torch.equal(lse[~fine], ref_lse[~fine])
        assert bool(((lse - ref_lse)[fine].abs() <= 2.0 ** -13 * (1 + ref_lse[fine].abs()) + (2.0 ** -20 * cap if cap else 0.0)).all())
        return out, lse


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("d", [32, 64, 96, 128, 160, 192, 224, 256])
def test_head_sizes_and_types(d, dt, bits):
    _Call([1] * 3, [33, 1, 150], 8, 2, d, 16, bits, dt).check()
    _Call([1, 30, 4], [33, 40, 150], 8, 2, d, 16, bits, dt, softcap=20.0, window=37).check()


@pytest.mark.parametrize("h,hk", [(1, 1), (3, 3), (6, 2), (5, 1), (16, 1), (17, 1), (24, 1), (40, 1), (64, 8), (130, 2)])
def test_head_layouts(h, hk):
    _Call([1] * 2, [19, 130], h, hk, 64, 16).check()


@pytest.mark.parametrize("page", [1, 3, 16, 48, 256])
def test_pages_end_inside_tiles(page):
    _Call([1] * 3, [31, 97, 260], 4, 2, 64, page, 8).check()
    _Call([9, 1, 20], [31, 97, 260], 4, 2, 64, page, window=50).check()


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("lens", [[1], [0], [0, 0], [1, 0], [0, 5, 0], [128, 129], [4500], [2049, 1], [31, 32, 33, 64, 127, 128, 0, 1]])
def test_lengths(lens, bits):
    _Call([1] * len(lens), lens, 4, 2, 128, 16, bits).check()


@pytest.mark.parametrize("b", [1, 5, 9, 33, 70])
def test_batches(b):
    _Call([1] * b, [(7 * i) % 50 for i in range(b)], 8, 2, 64, 16).check()


@pytest.mark.parametrize("window", [1, 2, 31, 32, 33, 100, 128, 1000, 2 ** 31, 2 ** 40])
def test_windows(window):
    """The window's first key anywhere in a tile, in another part, before the first token."""
    for bits, d in ((4, 64), (8, 128)):
        _Call([1] * 4, [1, 64, 257, 900], 4, 2, d, 16, bits, window=window).check()
        _Call([1, 64, 3, 130], [1, 64, 257, 900], 6, 2, d, 16, bits, window=window).check()


@pytest.mark.parametrize("softcap,gain", [(5.0, 1.0), (30.0, 8.0), (50.0, 0.01), (1000.0, 4.0), (1e30, 1.0), (0.01, 1.0)])
def test_caps(softcap, gain):
    for bits, dt in ((4, BF), (8, HF)):
        _Call([1] * 3, [1, 64, 300], 4, 2, 128, 16, bits, dt, gain=gain, softcap=softcap).check()
        _Call([1, 20, 3], [1, 64, 300], 4, 2, 64, 16, bits, dt, gain=gain, softcap=softcap).check()


@pytest.mark.parametrize("scale", [0.0, -0.3, 1e-30])
def test_scales(scale):
    for cap in (None, 4.0):
        _Call([1, 1], [40, 300], 4, 2, 64, 16, softcap=cap).check(scale=scale)
        _Call([30, 1], [40, 300], 4, 2, 64, 16, softcap=cap).check(scale=scale)


@pytest.mark.parametrize("bits,dt", [(4, BF), (8, BF), (4, HF)])
@pytest.mark.parametrize("queries,lens", [([2, 1, 3], [2, 1, 3]), ([4, 4], [100, 37]), ([1, 40, 7], [300, 40, 9]), ([150, 3], [150, 200]),
                                          ([5, 0, 2], [5, 9, 2]), ([70], [70]), ([300, 20], [1500, 1100])])
def test_several_query_tokens(queries, lens, bits, dt):
    _Call(queries, lens, 6, 2, 64, 16, bits, dt).check()
    _Call(queries, lens, 4, 4, 128, 16, bits, dt).check()


def test_more_query_tokens_than_cached_tokens():
    """The first queries of such a sequence stand before its first token: they see nothing."""
    for window in (None, 1):
        c = _Call([4, 3, 30], [2, 0, 7], 4, 2, 64, 16, window=window)
        out, lse = c.check()
        assert bool((out[:2] == 0).all()) and bool((lse[4:7] == float("-inf")).all())


def test_one_query_token_each_with_starts():
    c = _Call([1] * 4, [5, 0, 77, 3000], 8, 2, 64, 16, ragged=True)
    ragged = c.run()
    c.starts = None
    assert all(torch.equal(a, b) for a, b in zip(ragged, c.run()))


def test_large_scores_and_constant_rows():
    """Scores far apart move the running maximum in many tiles; equal ones never."""
    _Call([1] * 3, [700, 40, 3000], 4, 2, 128, 16, gain=30.0).check()
    for q in (1, 40):
        c = _Call([q] * 3, [700, 40, 3000], 4, 2, 128, 16)
        c.q.zero_()
        c.check()


def test_offsets_bounds_and_tokens_of_no_sequence():
    """Offsets outside the queries, tokens in front of and behind the sequences, tokens past max_query_len, lengths past the bound."""
    for window in (None, 40):
        for lens in ([20, 30], [20, 3000]):  # one part, and several to join
            c = _Call([3, 5], lens, 4, 2, 64, 16, window=window)
            want = c.run()
            q = torch.cat((torch.ones(2, 4, 64, dtype=BF, device=DEV), c.q, torch.ones(3, 4, 64, dtype=BF, device=DEV)))
            c.starts = torch.tensor([2, 5, 10], dtype=torch.int32, device=DEV)
            out, lse = c.run(q=q)
            assert torch.equal(out[2:10], want[0]) and torch.equal(lse[2:10], want[1])
            assert bool((out[:2] == 0).all()) and bool((out[10:] == 0).all()) and bool((lse[10:] == float("-inf")).all())
            c.max_q = 4
            out, lse = c.run(q=q)
            assert torch.equal(out[2:9], want[0][:7]) and bool(out[9].isnan().all()) and bool(lse[9].isnan().all())
            c.max_q, c.starts = 5, torch.tensor([-7, 3, 1000], dtype=torch.int32, device=DEV)
            out, _ = c.run()
            assert torch.equal(out, want[0])
    c = _Call([1, 1], [20, 30], 4, 2, 64, 16, width=4)
    c.lens.copy_(torch.tensor([-5, 2 ** 30]))
    out, lse = c.run(max_seq_len=17)
    c.n = [0, 17]
    c.lens.copy_(torch.tensor([0, 17]))
    assert torch.equal(out, c.check()[0])


def test_no_sequences_and_no_tokens():
    cache = mx.MXKVCache.allocate(2, 2, 16, 64)
    table, lens = torch.zeros(0, 3, dtype=torch.int32, device=DEV), torch.zeros(0, dtype=torch.int32, device=DEV)
    starts = torch.zeros(1, dtype=torch.int32, device=DEV)
    q = torch.ones(3, 4, 64, dtype=BF, device=DEV)
    out, lse = mx.mx_attention(q, cache, table, lens, query_start=starts, max_query_len=4, return_lse=True)
    assert bool((out == 0).all()) and bool((lse == float("-inf")).all())
    assert mx.mx_attention(q[:0], cache, table, lens).shape == (0, 4, 64)


def test_pages_outside_the_cache_and_shared_pages():
    c = _Call([1] * 3, [100, 100, 40], 4, 2, 64, 16)
    c.table[0, 2], c.table[1, 0] = -3, 2 ** 30
    c.table[2, :3] = c.table[1, 1:4]
    c.check()
    c = _Call([30, 2, 2], [100, 100, 40], 4, 2, 64, 16, 8)
    c.table[0, 2], c.table[1, 0] = 10 ** 9, -1
    c.check()


def test_a_nan_block_shows_where_it_is_seen_and_only_there():
    for q in (1, 40):
        c = _Call([q, 1], [100, 100], 4, 2, 64, 16)
        want = c.run()[0]
        page, slot = int(c.table[1, 3]), 5
        c.cache.v_scale[page, 1, slot, 0] = 255
        out = c.run()[0]
        assert torch.equal(out[:q], want[:q]) and torch.equal(out[q, :2], want[q, :2])
        assert bool(out[q, 2:, :32].isnan().all()) and torch.equal(out[q, 2:, 32:], want[q, 2:, 32:])
        assert torch.equal(c.run(window=100 - 3 * 16 - 6)[0][q].isnan().any(), torch.tensor(False, device=DEV))


def test_strides_out_and_slices_of_a_cache():
    c = _Call([1] * 3, [33, 5, 150], 8, 2, 64, 16)
    want, lse = c.check()
    wide = torch.zeros(3, 9, 67, dtype=BF, device=DEV)
    q = wide[:, 1:, 3:].copy_(c.q)
    out = torch.full((3, 8, 65), 7.0, dtype=BF, device=DEV)[..., 1:]
    got, got_lse = c.run(q=q, out=out)
    assert got is out and torch.equal(out, want) and torch.equal(lse, got_lse.cpu().double())
    old = (c.cache.k, c.cache.v, c.cache.k_scale, c.cache.v_scale)
    big = [torch.full((t.shape[0], 4, 40, t.shape[3]), 255, dtype=torch.uint8, device=DEV) for t in old]
    views = [x[:, 1:3, 7:23] for x in big]
    for x, t in zip(views, old):
        x.copy_(t)
    c.cache = mx.MXKVCache(*views)
    assert torch.equal(c.run()[0], want)
    parts = c.table.clone()
    c.table = torch.cat((parts, parts), 1)[:, :parts.shape[1]]
    assert torch.equal(c.run()[0], want)


def test_same_bits_every_time_on_any_stream_and_captured():
    for queries, lens in (([1] * 3, [3000, 5, 700]), ([40, 1, 3], [3000, 5, 700])):
        c = _Call(queries, lens, 8, 2, 128, 16, softcap=30.0)
        want = c.run()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = c.run()
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, b) for a, b in zip(want, other))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = c.run()
        for i in range(3):
            c.q.copy_(torch.randn(c.q.shape, generator=gen(i)).to(BF))
            c.lens.copy_(torch.tensor([3000 - 100 * i, 5, 700 - i]))
            graph.replay()
            torch.cuda.synchronize()
            kept = [x.clone() for x in got]
            assert all(torch.equal(a, b) for a, b in zip(kept, c.run()))


def test_refusals():
    c = _Call([1] * 3, [33, 5, 150], 8, 2, 64, 16)
    good = dict(q=c.q, cache=c.cache, page_table=c.table, seq_lens=c.lens)
    for bad in (dict(q=c.q.float()), dict(q=c.q[:2]), dict(q=c.q[:, :7]), dict(q=c.q[..., :32]), dict(page_table=c.table.long()),
                dict(page_table=c.table[0]), dict(seq_lens=c.lens[:2]), dict(seq_lens=c.lens.long()), dict(max_query_len=2),
                dict(max_query_len=0), dict(max_seq_len=10 ** 6), dict(max_seq_len=-1), dict(window=0), dict(window=-4), dict(softcap=0.0),
                dict(softcap=-2.0), dict(softcap=float("nan")), dict(out=c.q.half()), dict(out=c.q[:, :1].expand(3, 8, 64)),
                dict(seq_lens=c.lens.cpu()), dict(query_start=c.lens), dict(query_start=torch.zeros(4, device=DEV))):
        with pytest.raises(ConfigError):
            mx.mx_attention(**{**good, **bad})
    with pytest.raises(ops_gemm.HardwareUnsupported):
        mx.mx_attention(**{**good, "q": c.q.cpu()})
