"""rope_append against its definition in 64 bits, over head sizes, rotated shares, pair orders, page sizes, cache types and
strides; padding, positions outside the table, in place, views of one projection's output."""
from __future__ import annotations

import pytest
import torch

from forge_amd import ops_decoder as ops
from forge_amd.errors import ConfigError
from tests._decoder_ref import HALF_ULP, rotate_ref
from tests._util import gen

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF, E4 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


def _table(n, rot):
    angle = torch.arange(n).view(-1, 1) * torch.pow(torch.tensor(10000.0), -torch.arange(0, rot, 2) / rot)
    return torch.cat((angle.cos(), angle.sin()), 1)


def _cache(pages, hk, page, d, dt, g):
    if dt != E4:
        mk = lambda: torch.randn(pages, hk, page, d, generator=g).to(dt).to(DEV)  # noqa: E731
        return ops.PagedKVCache(mk(), mk())
    mk = lambda: (torch.randn(pages, hk, page, d, generator=g) * 20).to(E4).to(DEV)  # noqa: E731
    return ops.PagedKVCache(mk(), mk(), (torch.rand(hk, generator=g) + 0.01).to(DEV), (torch.rand(hk, generator=g) + 0.01).to(DEV))


def _bytes(t):
    return t.cpu().view(torch.uint8) if t.dtype == E4 else t.cpu().view(torch.int16)


def _check_cache(before, after, new, slots, scale, dt):
    """Slots hold the new values' roundings; every other byte is what it was."""
    page = after.shape[2]
    left = _bytes(after).clone()
    for t, slot in enumerate(slots.tolist()):
        if not 0 <= slot < after.shape[0] * page:
            continue
        got = after[slot // page, :, slot % page].cpu().float().double()
        if dt == E4:
            want = (new[t] / scale.cpu().double().view(-1, 1)).clamp(-448, 448)
            tol = want.abs() * (2.0 ** -4 + 2.0 ** -20) + 2.0 ** -10
            tol = tol + 2.0 ** -21 * (new[t].abs().amax() / scale.cpu().double().view(-1, 1))
        else:
            want = new[t]
            u, tiny = HALF_ULP[dt]
            # a difference of two products, each rounded once to fp32
            tol = (u + 2.0 ** -22) * want.abs() + 2.0 ** -22 * new[t].abs().amax() + tiny
        assert bool(((got - want).abs() <= tol).all())
        left[slot // page, :, slot % page] = _bytes(before)[slot // page, :, slot % page]
    assert torch.equal(left, _bytes(before))


def _run(t, h, hk, d, rot, page, dt, cdt, inter, idx=torch.int64, padded=0, seed=0, fused=True, in_place=False):
    g = gen(seed + t + d)
    qkv = torch.randn(t, (h + 2 * hk) * d, generator=g).to(dt)
    q, k, v = (x.view(t, -1, d) for x in qkv.split((h * d, hk * d, hk * d), 1))
    pages = -(-t // page) + 2
    cache = _cache(pages, hk, page, d, cdt, g)
    before = ops.PagedKVCache(cache.k.clone(), cache.v.clone(), cache.k_scale, cache.v_scale)
    slots = torch.randperm(pages * page, generator=g)[:t].to(idx)
    slots[:padded] = -1
    positions, table = torch.randint(0, 100, (t,), generator=g).to(idx), _table(100, rot)
    dev = qkv.to(DEV)
    qd, kd, vd = (x.view(t, -1, d) for x in dev.split((h * d, hk * d, hk * d), 1))
    if not fused:  # heads in front of tokens, values one element off
        qd, kd = qd.transpose(0, 1).contiguous().transpose(0, 1), kd.transpose(0, 1).contiguous().transpose(0, 1)
        vd = torch.zeros(t, hk, d + 1, dtype=dt, device=DEV)[..., 1:].copy_(vd)
    got = ops.rope_append(qd, kd, vd, positions.to(DEV), table.to(DEV), cache, slots.to(DEV), interleaved=inter,
                          q_out=qd if in_place else None)
    assert (got.data_ptr() == qd.data_ptr()) == in_place
    want = rotate_ref(q, positions, table, inter)
    u, tiny = HALF_ULP[dt]
    assert bool(((got.cpu().double() - want).abs() <= (u + 2.0 ** -22) * want.abs() + 2.0 ** -22 * want.abs().amax() + tiny).all())
    _check_cache(before.k, cache.k, rotate_ref(k, positions, table, inter), slots, cache.k_scale, cdt)
    _check_cache(before.v, cache.v, v.double(), slots, cache.v_scale, cdt)


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("dt,cdt", [(BF, BF), (HF, HF), (BF, E4), (HF, E4)])
@pytest.mark.parametrize("d,rot", [(128, 128), (64, 64), (256, 256), (80, 80), (96, 32), (16, 2), (128, 126), (112, 40)])
def test_heads_and_rotated_shares(d, rot, dt, cdt, inter):
    _run(5, 6, 2, d, rot, 4, dt, cdt, inter, padded=1)


@pytest.mark.parametrize("t,h,hk,page,idx", [(1, 1, 1, 1, torch.int64), (1, 32, 8, 16, torch.int32), (3, 7, 7, 5, torch.int32),
                                             (17, 24, 3, 16, torch.int64), (600, 4, 1, 48, torch.int64)])
def test_tokens_heads_and_pages(t, h, hk, page, idx):
    _run(t, h, hk, 64, 64, page, BF, BF, False, idx=idx, padded=t // 4)


@pytest.mark.parametrize("inter", [False, True])
def test_views_and_in_place(inter):
    _run(7, 8, 2, 128, 128, 16, HF, HF, inter, fused=False)
    _run(7, 8, 2, 128, 64, 16, BF, BF, inter, in_place=True)


def test_head_dim_of_eight():
    _run(5, 2, 1, 8, 4, 4, BF, BF, False)
    _run(5, 2, 1, 72, 36, 4, BF, BF, True)


def test_a_token_major_cache():
    """Any strides of whole 16-byte units: here all heads of a token next to each other."""
    g = gen(1)
    base = torch.randn(2, 6, 4, 3, 64, generator=g).to(BF).to(DEV).permute(0, 1, 3, 2, 4)  # [2, pages, heads, page, dim]
    cache = ops.PagedKVCache(base[0], base[1])
    before = base.clone()
    q, k, v = (torch.randn(9, n, 64, generator=g).to(BF) for n in (6, 3, 3))
    slots, pos, table = torch.randperm(24, generator=g)[:9], torch.arange(9), _table(9, 64)
    ops.rope_append(q.to(DEV), k.to(DEV), v.to(DEV), pos.to(DEV), table.to(DEV), cache, slots.to(DEV))
    _check_cache(before[0], cache.k, rotate_ref(k, pos, table, False), slots, None, BF)
    _check_cache(before[1], cache.v, v.double(), slots, None, BF)


def test_slots_and_positions_outside():
    g = gen(2)
    cache = _cache(2, 2, 4, 64, BF, g)
    before = ops.PagedKVCache(cache.k.clone(), cache.v.clone())
    q, k, v = (torch.randn(4, n, 64, generator=g).to(BF).to(DEV) for n in (4, 2, 2))
    slots, pos = torch.tensor([8, -7, 2 ** 40, 3]).to(DEV), torch.tensor([0, 1, 50, -1]).to(DEV)
    got = ops.rope_append(q, k, v, pos, _table(50, 32).to(DEV), cache, slots).cpu().float()
    assert bool(got[:2].isfinite().all()) and bool(got[2:, :, :32].isnan().all())
    assert torch.equal(got[2:, :, 32:], q.cpu().float()[2:, :, 32:])
    changed = (cache.k.cpu().float() != before.k.cpu().float()).any(-1).any(1)
    assert changed.nonzero().tolist() == [[0, 3]] and bool(cache.k[0, :, 3, :32].isnan().all())


def test_values_past_e4m3_are_clamped_and_nan_stays():
    cache = ops.PagedKVCache.allocate(1, 1, 4, 64, E4, DEV)
    q = torch.zeros(3, 1, 64, dtype=BF, device=DEV)
    v = torch.full((3, 1, 64), 1000.0, dtype=BF, device=DEV)
    v[1], v[2] = -1e30, float("nan")
    ops.rope_append(q, q, v, torch.zeros(3, dtype=torch.int32, device=DEV), _table(1, 64).to(DEV), cache,
                    torch.arange(3, device=DEV))
    got = cache.v.cpu().float()[0, 0]
    assert bool((got[0] == 448).all()) and bool((got[1] == -448).all()) and bool(got[2].isnan().all())


def test_no_tokens_and_refusals():
    cache = ops.PagedKVCache.allocate(2, 2, 4, 64, BF, DEV)
    q, k = torch.zeros(3, 4, 64, dtype=BF, device=DEV), torch.zeros(3, 2, 64, dtype=BF, device=DEV)
    i, table = torch.zeros(3, dtype=torch.int64, device=DEV), _table(4, 64).to(DEV)
    assert ops.rope_append(q[:0], k[:0], k[:0], i[:0], table, cache, i[:0]).shape == (0, 4, 64)
    call = dict(q=q, k=k, v=k, positions=i, cos_sin=table, cache=cache, slots=i)
    for bad in (dict(q=q.half()), dict(k=k[:2]), dict(v=q), dict(positions=i[:2]), dict(positions=i.float()), dict(slots=i.cpu()),
                dict(cos_sin=table.half()), dict(cos_sin=table[:, :5]), dict(cos_sin=torch.zeros(4, 66, device=DEV)),
                dict(q=q[..., :32]), dict(q_out=q[:2]), dict(cos_sin=table[:, :0])):
        with pytest.raises(ConfigError):
            ops.rope_append(**{**call, **bad})
    with pytest.raises(ConfigError):
        ops.PagedKVCache(cache.k, cache.v.half())
    with pytest.raises(ConfigError):
        ops.PagedKVCache(cache.k.view(torch.float8_e4m3fn), cache.v.view(torch.float8_e4m3fn))
    odd = torch.zeros(2, 2, 4, 68, dtype=BF, device=DEV)[..., :64]
    with pytest.raises(Exception, match="16-byte"):
        ops.rope_append(**{**call, "cache": ops.PagedKVCache(odd, odd)})


def test_outputs_whose_rows_overlap_are_refused():
    cache = ops.PagedKVCache.allocate(2, 2, 4, 64, BF, DEV)
    q, k = torch.zeros(3, 4, 64, dtype=BF, device=DEV), torch.zeros(3, 2, 64, dtype=BF, device=DEV)
    i, table = torch.arange(3, device=DEV), _table(4, 64).to(DEV)
    for out in (q[:1].expand(3, 4, 64), q[:, :1].expand(3, 4, 64)):
        with pytest.raises(ConfigError, match="overlap"):
            ops.rope_append(q, k, k, i, table, cache, i, q_out=out)
        with pytest.raises(ConfigError, match="overlap"):
            ops.prefix_attention(q, cache, torch.zeros(3, 1, dtype=torch.int32, device=DEV), i.int(), out=out)
