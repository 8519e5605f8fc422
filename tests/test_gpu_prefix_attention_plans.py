"""prefix_attention over the ways in which its work is cut: kernels for few rows, for many and for both at once, the prefix's
items first or among the others, sequences that take the prefix along, one part and many, row tables longer than their LDS
halves, and sets of keys that do and do not go round the XCDs evenly."""
from __future__ import annotations

import pytest
import torch

from forge_amd import _lib
from forge_amd import ops_decoder as ops
from tests._decoder_ref import assert_attention, attention_ref_fast

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF, E4 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


def _call(queries, lens, prefix, h, hk, d, page=16, dt=BF, cdt=None, extra=0, gain=1.0, seed=0):
    """(arguments, fp64 reference) of one call; ``extra`` query tokens of no sequence at the end."""
    g = torch.Generator(DEV).manual_seed(seed + sum(lens) + prefix + d)
    cdt = cdt or dt
    b, width, head = len(lens), -(-max([*lens, 1]) // page), -(-prefix // page)
    pages = head + b * width + 1
    kv = [torch.randn(pages, hk, page, d, generator=g, device=DEV) for _ in range(2)]
    kv = [(x * 20).to(E4) if cdt == E4 else x.to(cdt) for x in kv]
    scales = [torch.rand(hk, generator=g, device=DEV) * 0.02 + 0.04 for _ in range(2)] if cdt == E4 else []
    cache = ops.PagedKVCache(*kv, *scales)
    perm = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    starts = torch.tensor([0, *torch.tensor(queries).cumsum(0).tolist()], dtype=torch.int32, device=DEV)
    t = int(starts[-1])
    ragged = extra > 0 or any(n != 1 for n in queries)
    q = (torch.randn(t + extra, h, d, generator=g, device=DEV) * gain).to(dt)
    kw = dict(q=q, cache=cache, page_table=perm[head:head + b * width].view(b, width).contiguous(),
              seq_lens=torch.tensor(lens, dtype=torch.int32, device=DEV), prefix_pages=perm[:head].contiguous(), prefix_len=prefix,
              query_start=starts if ragged else None, max_query_len=max(queries), return_lse=True)
    ref = attention_ref_fast(q, cache, kw["page_table"], kw["seq_lens"], kw["prefix_pages"], prefix, starts, d ** -0.5)
    return kw, ref


def _check(kernel, *args, **kw):
    call, ref = _call(*args, **kw)
    out, lse = ops.prefix_attention(**call)
    assert kernel in _lib.last_kernel(), _lib.last_kernel()
    assert_attention(out, lse, ref, call["q"].dtype)
    return call, out, lse


@pytest.mark.parametrize("dt,cdt", [(BF, BF), (HF, HF), (BF, E4), (HF, E4)])
@pytest.mark.parametrize("d", [64, 128, 256, 96])
def test_both_kinds_in_one_launch(d, dt, cdt):
    """A batch's rows fill several tiles of the prefix; each sequence reads its own keys."""
    _check("attn_mixed_kernel", [1] * 40, [(37 * i) % 300 for i in range(40)], 700, 16, 2, d, 16, dt, cdt)


@pytest.mark.parametrize("hk", [1, 3, 8])
def test_the_prefix_first_and_among_the_others(hk):
    """Its products outlast short sequences' reads, or not; the sets of keys fill the XCDs evenly, or not."""
    for seq in (4, 900):
        _check("attn_mixed_kernel", [1] * 70, [1 + (13 * i) % seq for i in range(70)], 9000, 4 * hk, hk, 64)


@pytest.mark.parametrize("h,hk,prefix", [(4, 1, 3000), (6, 3, 3000), (16, 8, 5000), (9, 9, 6000)])
def test_prefix_of_few_rows_in_many_parts(h, hk, prefix):
    _check("attn_rows_kernel", [1, 1], [30, 700], prefix, h, hk, 128)


@pytest.mark.parametrize("dt,cdt", [(BF, BF), (HF, E4)])
def test_prompts_take_the_prefix_along(dt, cdt):
    """One part of more than three halves of the row table for every sequence, nothing to join."""
    call, out, lse = _check("attn_tile_kernel parts=0+1", [512, 400, 300, 512], [700, 401, 300, 512], 3100, 32, 8, 64, 16, dt, cdt, extra=5)
    assert "join" not in _lib.last_kernel()
    assert bool((out[-5:] == 0).all()) and bool((lse[-5:] == float("-inf")).all())


@pytest.mark.parametrize("h,hk", [(4, 2), (32, 2)])
def test_queries_in_front_of_their_sequence_see_the_prefix_taken_along(h, hk):
    """More query tokens than cached ones: the first stand before the sequence and see the whole prefix, no less."""
    for prefix in (20, 300):
        call, ref = _call([40, 33, 35], [2, 0, 34], prefix, h, hk, 64)
        call2, ref2 = _call([3, 2], [1, 0], prefix, 4, 4, 64)
        assert_attention(*ops.prefix_attention(**call), ref, BF)
        assert_attention(*ops.prefix_attention(**call2), ref2, BF)


def test_prompts_take_the_prefix_along_in_parts():
    _check("attn_tile_kernel parts=0+", [300], [350], 2500, 4, 1, 128, gain=4.0)
    assert "join" in _lib.last_kernel()


def test_prompts_beside_the_prefix():
    """Too few rows in each sequence to fill tiles: the prefix's rows are those of the batch."""
    call, _, _ = _check("attn_tile_kernel parts=", [9] * 12, [9 + 20 * i for i in range(12)], 800, 8, 2, 64)
    assert "parts=0+" not in _lib.last_kernel()


def test_one_part_with_tokens_of_no_sequence_and_past_the_longest():
    """What no workgroup computes is written by the sequences' own: in front, behind, and past max_query_len."""
    call, ref = _call([3, 2, 4], [60, 2, 90], 0, 8, 2, 64, extra=3)
    out, lse = ops.prefix_attention(**call)
    assert "join" not in _lib.last_kernel() and "parts=0+1" in _lib.last_kernel()
    assert_attention(out, lse, ref, BF)
    pad = {**call, "q": torch.cat((call["q"][:2], call["q"])), "query_start": call["query_start"] + 2}
    got, got_lse = ops.prefix_attention(**pad)
    assert torch.equal(got[2:], out) and bool((got[:2] == 0).all()) and bool((got_lse[:2] == float("-inf")).all())
    got, got_lse = ops.prefix_attention(**{**call, "max_query_len": 2})
    served = torch.tensor([1, 1, 0, 1, 1, 1, 1, 0, 0, 1, 1, 1], dtype=torch.bool, device=DEV)
    assert torch.equal(got[served], out[served]) and bool(got[~served].isnan().all()) and bool(got_lse[~served].isnan().all())


@pytest.mark.parametrize("prefix,lens", [(0, [20, 0, 31]), (100, [20, 0, 31]), (1000, [20, 0, 31]), (9000, [700, 0, 900])])
def test_negative_lengths_are_no_tokens(prefix, lens):
    call, ref = _call([1, 1, 1], lens, prefix, 4, 2, 64)
    call["seq_lens"][1] = -40
    assert_attention(*ops.prefix_attention(**call), ref, BF)


@pytest.mark.parametrize("scale", [-0.2, 0.0, 1e-30])
def test_scales_that_are_not_positive(scale):
    for queries, lens, prefix, h in (([1, 1], [40, 300], 70, 4), ([70, 30], [100, 300], 90, 8)):
        call, _ = _call(queries, lens, prefix, h, 2, 64)
        starts = call["query_start"] if call["query_start"] is not None else torch.arange(3)
        ref = attention_ref_fast(call["q"], call["cache"], call["page_table"], call["seq_lens"], call["prefix_pages"], prefix, starts, scale)
        assert_attention(*ops.prefix_attention(**call, scale=scale), ref, BF)


def test_nan_in_pages_that_a_tile_only_touches():
    """Keys past a sequence's end in the last page, and of pages outside the cache, in the kernel of many rows."""
    for cdt, d in ((BF, 128), (BF, 96), (E4, 128)):
        call, ref = _call([60, 70], [75, 130], 100, 8, 2, d, 16, BF, cdt)
        cache, table = call["cache"], call["page_table"]
        raw = [x.view(torch.uint8) if cdt == E4 else x for x in (cache.k, cache.v)]
        for x in raw:
            nan = 0x7f if cdt == E4 else float("nan")
            x[table[0, 4], :, 75 - 64:] = nan
            x[table[1, 8], :, 130 - 128:] = nan
            x[call["prefix_pages"][6], :, 100 - 96:] = nan
        assert_attention(*ops.prefix_attention(**call), ref, BF)


def test_a_graph_of_both_kinds_follows_its_inputs():
    call, ref = _call([1] * 40, [(37 * i) % 300 for i in range(40)], 700, 16, 2, 64)
    want = ops.prefix_attention(**call)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = ops.prefix_attention(**call)
    for k in range(3):
        call["q"].normal_(generator=torch.Generator(DEV).manual_seed(k))
        call["seq_lens"].copy_(torch.tensor([(11 * i + 50 * k) % 296 for i in range(40)], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        eager = ops.prefix_attention(**call)
        assert torch.equal(out, eager[0]) and torch.equal(lse, eager[1]) and not torch.equal(out, want[0])


@pytest.mark.parametrize("prefix,lens,h", [(0, [60, 2, 90], 8), (100, [60, 2, 90], 8), (3000, [60, 2, 90], 2), (3000, [900, 2, 1500], 64)])
def test_query_offsets_outside_the_queries(prefix, lens, h):
    """They count as the queries' begin or end: sequences in front and behind that have no queries there change nothing."""
    call, ref = _call([3, 2, 4], lens, prefix, h, 2, 64)
    want = ops.prefix_attention(**call)
    assert_attention(*want, ref, BF)
    far = 2 ** 31 - 1
    for front, back in (([-5], []), ([-far - 1, -7], [far]), ([], [far, far - 3, far])):
        # the first sequence's own tokens start in front of the queries
        starts = [*(front or [0]), *call["query_start"].tolist()[1:], *back]
        none = [torch.zeros(n, dtype=torch.int64) for n in (max(len(front) - 1, 0), len(back))]
        rows = torch.cat((none[0], torch.arange(3), none[1])).to(DEV)
        got = ops.prefix_attention(**{**call, "query_start": torch.tensor(starts, dtype=torch.int32, device=DEV),
                                      "page_table": call["page_table"][rows], "seq_lens": call["seq_lens"][rows]})
        assert_attention(*got, ref, BF)


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("queries,lens,prefix,h,kernel", [
    ([1, 1], [40, 301], 70, 4, "attn_rows_kernel"), ([70, 30], [100, 300], 90, 8, "attn_tile_kernel"),
    ([1] * 40, [(37 * i) % 300 for i in range(40)], 700, 16, "attn_mixed_kernel"), ([1], [77], 0, 4, "attn_rows_kernel")])
def test_key_scales_and_scales_that_are_not_positive(queries, lens, prefix, h, kernel, dt):
    """A cached key is code * scale of its head, whatever the scale: zero gives equal weights, a negative one turns the scores."""
    for key_scale, scale in ((0.0, 0.125), (-0.05, 0.125), (0.05, -0.125), (-0.05, -0.125), (-0.05, 0.0), (2.0 ** -120, 2.0 ** -20)):
        call, _ = _call(queries, lens, prefix, h, 2, 64, 16, dt, E4)
        call["cache"].k_scale[1] = key_scale
        starts = call["query_start"] if call["query_start"] is not None else torch.arange(len(lens) + 1)
        ref = attention_ref_fast(call["q"], call["cache"], call["page_table"], call["seq_lens"], call["prefix_pages"], prefix, starts, scale)
        got = ops.prefix_attention(**call, scale=scale)
        assert kernel in _lib.last_kernel()
        assert_attention(*got, ref, dt)


@pytest.mark.parametrize("t,h,n,kernel", [(1, 4, 2048, "attn_rows_kernel"), (1, 4, 131072, "attn_rows_kernel"), (3, 4, 250, "attn_rows_kernel"),
                                          (40, 8, 5000, "attn_tile_kernel"), (1024, 64, 131072, "attn_tile_kernel parts=0+1")])
@pytest.mark.parametrize("cdt", [HF, E4])
def test_one_key_above_many_in_fp16(t, h, n, kernel, cdt):
    """Each of the others has 2^-25 of its weight, all of them up to 0.4% of the result.  A weight is rounded by 2^-11 of itself
    and by no more than 2^-32 of the largest (half of fp16's smallest step, counted from 2^7 below that)."""
    page, score = 256, 17.25  # e^-17.25 = 2^-24.9
    pages = -(-n // page)
    k, v = torch.zeros(pages, 1, page, 64, device=DEV), torch.ones(pages, 1, page, 64, device=DEV)
    k[0, 0, 5, 0], v[0, 0, 5] = (16.0 if cdt == E4 else score), 0.0
    scales = [torch.full((1,), x, device=DEV) for x in (score / 16, 1.0)] if cdt == E4 else []
    cache = ops.PagedKVCache(k.to(cdt), v.to(cdt), *scales)
    q = torch.zeros(t, h, 64, dtype=HF, device=DEV)
    q[..., 0] = 8.0
    i32 = dict(dtype=torch.int32, device=DEV)
    out, lse = ops.prefix_attention(q, cache, torch.arange(pages, **i32).view(1, -1), torch.tensor([n], **i32), scale=0.125,
                                    query_start=torch.tensor([0, t], **i32), max_query_len=t, max_seq_len=n, return_lse=True)
    assert kernel in _lib.last_kernel(), _lib.last_kernel()
    others = (n - t + torch.arange(t, dtype=torch.float64)) * torch.exp(torch.tensor(-score, dtype=torch.float64))
    want = (others / (1 + others)).view(t, 1, 1)
    err = (out.cpu().double() - want).abs()
    assert bool((err <= (2.0 ** -10 + 2.0 ** -12) * want + n * 2.0 ** -32 + 2.0 ** -25).all()), (err.max(), want.max())
    assert bool(((lse.cpu().double() - score - torch.log1p(others).view(t, 1)).abs() <= 2.0 ** -13 * (1 + score)).all())
