"""mx_append and mx_read against their definition: every code and scale bit for bit, every form of the rotation, places that are
not written, caches that are slices of others, slots and positions outside."""
from __future__ import annotations

import copy

import pytest
import torch

from forge_amd import ops_gemm
from forge_amd import ops_mx as mx
from forge_amd.errors import ConfigError
from tests._decoder_ref import HALF_ULP
from tests._mx_ref import decode_ref, encode_ref, pack_ref, rotate_axes_ref
from tests._util import gen

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF = torch.bfloat16, torch.float16


def _table(positions, rot):
    angle = torch.arange(positions).view(-1, 1) * torch.pow(torch.tensor(10000.0), -torch.arange(0, rot, 2) / rot)
    return torch.cat((angle.cos(), angle.sin()), 1)


def _random_cache(pages, hk, page, dim, bits, g):
    k, v = (torch.randint(0, 256, (pages, hk, page, dim * bits // 8), generator=g, dtype=torch.uint8).to(DEV) for _ in range(2))
    ks, vs = (torch.randint(100, 140, (pages, hk, page, dim // 32), generator=g, dtype=torch.uint8).to(DEV) for _ in range(2))
    return mx.MXKVCache(k, v, ks, vs)


def _tensors(cache):
    return cache.k, cache.k_scale, cache.v, cache.v_scale


def _check(q, k, v, positions, table, cache, before, slots, q_out, sections, interleaved, bits):
    pos = positions.view(len(sections), -1).cpu()
    ref_q = rotate_axes_ref(q, pos, table, sections, interleaved)
    u, tiny = HALF_ULP[q.dtype]
    rot = table.shape[1]
    # two products and a sum in fp32, each off by half a unit of at most twice the largest of the pair
    size = q.cpu().double().abs()
    turned = size[..., :rot]
    other = (turned.unflatten(-1, (-1, 2)).flip(-1).flatten(-2) if interleaved else turned.roll(rot // 2, -1)) if rot else turned
    slack = torch.zeros_like(size)
    slack[..., :rot] = 2.0 ** -22 * (turned + other)
    got = q_out.cpu().double()
    fine = torch.isfinite(ref_q)
    assert torch.equal(fine, torch.isfinite(got))
    assert bool(((got - ref_q).abs() <= (u * ref_q.abs() + slack + tiny))[fine].all())
    expect = [t.clone() for t in before]
    new = [encode_ref(rotate_axes_ref(k, pos, table, sections, interleaved).float(), bits), encode_ref(v.cpu().float(), bits)]
    page = expect[0].shape[2]
    for t, slot in enumerate(slots.tolist()):
        if 0 <= slot < expect[0].shape[0] * page:
            for i, (codes, scales) in enumerate(new):
                expect[2 * i][slot // page, :, slot % page] = pack_ref(codes[t], bits)
                expect[2 * i + 1][slot // page, :, slot % page] = scales[t].to(torch.uint8)
    for a, b in zip(_tensors(cache), expect):
        assert torch.equal(a.cpu(), b)


FORMS = [  # heads, key heads, dim, rot, sections, interleaved
    (4, 2, 128, 128, None, False), (4, 2, 64, 64, None, True), (6, 3, 96, 48, None, False), (3, 1, 32, 32, None, False),
    (2, 2, 32, 2, None, False), (5, 5, 32, 6, None, True), (8, 1, 96, 24, None, False), (2, 1, 256, 256, None, False),
    (3, 3, 160, 80, None, True), (7, 1, 224, 100, None, False), (4, 2, 128, 128, (16, 24, 24), False), (4, 4, 64, 64, (5, 0, 20, 7), True),
    (2, 1, 96, 64, (11, 21), False), (1, 1, 192, 36, (1, 16, 1), False)]


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("form", FORMS, ids=str)
def test_against_the_definition(form, dt, bits):
    h, hk, dim, rot, sections, interleaved = form
    table = _table(50, rot)
    for t, page, index in ((1, 16, torch.int64), (13, 5, torch.int32), (530, 48, torch.int64)):
        if t > 100 and dim > 128:
            continue
        g = gen(t + dim + bits)
        q = torch.randn(t, h, dim, generator=g).to(dt)
        # blocks of every size, so that scales go over their range, and values on the borders of codes
        size = torch.exp2(torch.randint(-20, 12, (t, hk, dim // 32, 1), generator=g).float())
        k, v = ((torch.randn(t, hk, dim // 32, 32, generator=g) * size).flatten(-2).to(dt) for _ in range(2))
        v[:, :, 1::3] = (v[:, :, 1::3] * 4).round() / 4
        pages = -(-t // page) + 2
        cache = _random_cache(pages, hk, page, dim, bits, g)
        before = [x.cpu().clone() for x in _tensors(cache)]
        slots = torch.randperm(pages * page, generator=g)[:t].to(index)
        if t > 3:
            slots[1], slots[3] = -1, pages * page  # padding
        axes = sections or (rot // 2,)
        positions = torch.randint(0, 50, (len(axes), t), generator=g).to(index)
        where = positions.to(DEV) if sections else positions[0].to(DEV)
        q_out = mx.mx_append(q.to(DEV), k.to(DEV), v.to(DEV), where, table.to(DEV), cache, slots.to(DEV), sections=sections,
                             interleaved=interleaved)
        _check(q, k, v, positions, table, cache, before, slots, q_out, axes, interleaved, bits)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dt", [BF, HF])
def test_every_value_of_the_type(dt, bits):
    """All 65536 bit patterns, in blocks whose other values lie around and far from them: subnormals, infinities, NaN, ties."""
    every = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dt)
    table = _table(4, 64)
    for order in range(3):
        v = every if order == 0 else every[torch.randperm(65536, generator=gen(order))]
        if order == 2:  # in the scale of the largest code: the codes' own borders
            v = v.clone().view(-1, 32)
            v[:, 0] = 6.0 if bits == 4 else 448.0
            big = v.float().abs() > v[:, :1].float()
            v[big | ~torch.isfinite(v.float())] = 0.0
            v = v.flatten()
        v = v.view(-1, 1, 64)
        t = v.shape[0]
        cache = mx.MXKVCache.allocate(1, 1, t, 64, "mxfp4" if bits == 4 else "mxfp8", DEV)
        zero = torch.zeros(t, dtype=torch.int64, device=DEV)
        mx.mx_append(v.to(DEV), torch.zeros_like(v).to(DEV), v.to(DEV), zero, table.to(DEV), cache, torch.arange(t, device=DEV))
        codes, scales = encode_ref(v.float(), bits)
        assert torch.equal(cache.v_scale[0, 0].cpu().long(), scales.view(t, 2))
        assert torch.equal(cache.v[0, 0].cpu(), pack_ref(codes, bits).view(t, -1))
        assert bool((cache.k == 0).all()) and bool((cache.k_scale == 1).all())


@pytest.mark.parametrize("bits", [4, 8])
def test_every_code_and_scale_reads_back(bits):
    """All codes under all scales; a type that cannot hold a value gives the nearest one (fp16) or is not asked to."""
    rows = 256  # a scale byte each
    codes = torch.arange(256, dtype=torch.uint8).view(1, 1, 1, 256).expand(1, 1, rows, 256).contiguous()
    blocks = 256 // (4 * bits)
    scales = torch.arange(256, dtype=torch.uint8).view(1, 1, rows, 1).expand(1, 1, rows, blocks).contiguous()
    if bits == 4:  # head_dim 512 is too wide: two caches
        parts = [(codes[..., :128].contiguous(), scales[..., :8].contiguous()), (codes[..., 128:].contiguous(), scales[..., 8:].contiguous())]
    else:
        parts = [(codes, scales)]
    for c, s in parts:
        cache = mx.MXKVCache(c.to(DEV), c.to(DEV), s.to(DEV), s.to(DEV))
        ref = decode_ref(c, s, bits)[0, 0]
        for dt in (BF, HF):
            k, v = mx.mx_read(cache, torch.arange(rows, device=DEV), dtype=dt)
            assert torch.equal(k.view(torch.int16), v.view(torch.int16))
            got = k[:, 0].cpu().double()
            least = 2.0 ** -126 if dt == BF else 2.0 ** -14
            most = torch.finfo(dt).max
            inside = ((ref.abs() >= least) & (ref.abs() <= most)) | (ref == 0)
            assert torch.equal(got[inside], ref[inside])
            assert bool(got[ref.isnan()].isnan().all())
            small = ref.abs() < least
            assert bool(((got - ref)[small].abs() <= (2.0 ** -126 if dt == BF else 2.0 ** -24)).all())


def test_read_outside_and_both_index_types():
    g = gen(3)
    cache = _random_cache(3, 2, 16, 96, 4, g)
    ref = [decode_ref(c, s, 4).transpose(1, 2).flatten(0, 1) for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale))]
    slots = torch.tensor([5, -1, 47, 48, 0, 5])
    for dt in (torch.int32, torch.int64):
        got = mx.mx_read(cache, slots.to(dt).to(DEV))
        for x, r in zip(got, ref):
            x = x.cpu().double()
            assert bool((x[1] == 0).all()) and bool((x[3] == 0).all())
            assert torch.equal(x[[0, 2, 4, 5]], r[[5, 47, 0, 5]].to(BF).double())
    k, v = mx.mx_read(cache, slots[:0].to(DEV))
    assert k.shape == v.shape == (0, 2, 96)


@pytest.mark.parametrize("bits", [4, 8])
def test_slices_views_and_places(bits):
    """A cache that is some pages, heads and tokens of another; q, k, v views of one projection; queries rotated in place."""
    g = gen(11)
    big = _random_cache(9, 4, 32, 128, bits, g)
    cache = mx.MXKVCache(*(t[1::2, 1:3, 4:20] for t in (big.k, big.v, big.k_scale, big.v_scale)))
    before_big = [t.cpu().clone() for t in _tensors(big)]
    before = [t.cpu().clone() for t in _tensors(cache)]
    t = 21
    qkv = torch.randn(t, 10, 128, generator=g).to(BF)
    x = qkv.to(DEV)
    q, k, v = x[:, :6], x[:, 6:8], x[:, 8:]
    slots = torch.randperm(4 * 16, generator=g)[:t]
    table, positions = _table(64, 128), torch.arange(t)
    got = mx.mx_append(q, k, v, positions.to(DEV), table.to(DEV), cache, slots.to(DEV), q_out=q)
    assert got is q
    _check(qkv[:, :6], qkv[:, 6:8], qkv[:, 8:], positions, table, cache, before, slots, q, (64,), False, bits)
    assert torch.equal(x[:, 6:].cpu(), qkv[:, 6:])
    untouched = [b.clone() for b in before_big]
    for now, b, small in zip(_tensors(big), untouched, _tensors(cache)):
        b[1::2, 1:3, 4:20] = small.cpu()
        assert torch.equal(now.cpu(), b)
    odd = torch.zeros(t, 6, 130, dtype=BF, device=DEV)[:, :, 1:129]  # rows at odd elements
    odd.copy_(qkv[:, :6])
    again = mx.mx_append(odd, k, v, positions.to(DEV), table.to(DEV), cache, slots.to(DEV))
    assert torch.equal(again, q)


@pytest.mark.parametrize("form", [(48, False), (100, False), (24, False), (128, True)])
def test_rotation_in_place_of_every_form(form):
    rot, interleaved = form
    g = gen(rot)
    q, kv = torch.randn(40, 3, 128, generator=g).to(HF).to(DEV), torch.randn(40, 1, 128, generator=g).to(HF).to(DEV)
    cache = mx.MXKVCache.allocate(3, 1, 16, 128)
    args = (kv, kv, torch.arange(40, device=DEV), _table(40, rot).to(DEV), cache, torch.arange(40, device=DEV))
    apart = mx.mx_append(q, *args, interleaved=interleaved)
    mx.mx_append(q, *args, interleaved=interleaved, q_out=q)
    assert torch.equal(q, apart)


def test_values_that_are_not_finite_and_positions_outside():
    g = gen(2)
    q, k, v = (torch.randn(4, n, 64, generator=g).to(BF) for n in (2, 1, 1))
    v[0, 0, 3], v[1, 0, 40] = float("inf"), float("nan")
    cache = mx.MXKVCache.allocate(1, 1, 16, 64, "mxfp8")
    positions = torch.tensor([0, 1, 7, -1])
    out = mx.mx_append(q.to(DEV), k.to(DEV), v.to(DEV), positions.to(DEV), _table(7, 64).to(DEV), cache, torch.arange(4, device=DEV))
    assert bool(out[2:].isnan().all()) and bool(out[:2].isfinite().all())
    kk, vv = (x.cpu() for x in mx.mx_read(cache, torch.arange(4, device=DEV)))
    assert bool(kk[2:].isnan().all()) and bool(kk[:2].isfinite().all())
    assert bool(vv[0, 0, :32].isnan().all()) and bool(vv[0, 0, 32:].isfinite().all())
    assert bool(vv[1, 0, 32:].isnan().all()) and bool(vv[1, 0, :32].isfinite().all()) and bool(vv[2:].isfinite().all())


def test_no_tokens_and_a_captured_call():
    g = gen(9)
    cache = _random_cache(4, 2, 16, 64, 4, g)
    table = _table(32, 64).to(DEV)
    none = torch.zeros(0, dtype=torch.int64, device=DEV)
    empty = torch.zeros(0, 2, 64, dtype=BF, device=DEV)
    assert mx.mx_append(empty, empty, empty, none, table, cache, none).shape == (0, 2, 64)
    q, k, v = (torch.randn(5, n, 64, generator=g).to(BF).to(DEV) for n in (4, 2, 2))
    positions, slots = torch.arange(5, device=DEV), torch.arange(5, device=DEV)
    mx.mx_append(q, k, v, positions, table, cache, slots)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = mx.mx_append(q, k, v, positions, table, cache, slots)
        back = mx.mx_read(cache, slots)
    for i in range(3):
        q.copy_(torch.randn(5, 4, 64, generator=g).to(BF))
        v.copy_(torch.randn(5, 2, 64, generator=g).to(BF))
        slots.copy_(torch.randperm(64, generator=g)[:5])
        graph.replay()
        torch.cuda.synchronize()
        got = [out.clone(), *(b.clone() for b in back)]
        eager = mx.mx_append(q, k, v, positions, table, cache, slots)
        assert torch.equal(got[0], eager)
        for a, b in zip(got[1:], mx.mx_read(cache, slots)):
            assert torch.equal(a, b)


def test_refusals():
    cache = mx.MXKVCache.allocate(4, 2, 16, 64)
    q, kv = torch.zeros(3, 4, 64, dtype=BF, device=DEV), torch.zeros(3, 2, 64, dtype=BF, device=DEV)
    pos, table = torch.zeros(3, dtype=torch.int64, device=DEV), _table(8, 64).to(DEV)
    good = dict(q=q, k=kv, v=kv, positions=pos, cos_sin=table, cache=cache, slots=pos)
    mx.mx_append(**good)
    for bad in (dict(q=q.float()), dict(q=q[:, :, :32]), dict(q=q[0]), dict(k=kv[:2]), dict(v=kv.half()), dict(positions=pos[:2]),
                dict(positions=pos.float()), dict(cos_sin=table.half()), dict(cos_sin=table[:, :63]), dict(cos_sin=_table(8, 66).to(DEV)),
                dict(slots=pos[:1]), dict(slots=pos.cpu()), dict(sections=(16, 16)), dict(sections=(16, 15), positions=torch.stack((pos, pos))),
                dict(sections=(33, -1), positions=torch.stack((pos, pos))), dict(sections=(8, 8, 8, 4, 4), positions=pos.expand(5, 3)),
                dict(q_out=q.half()), dict(q_out=q[:, :1].expand(3, 4, 64))):
        with pytest.raises(ConfigError):
            mx.mx_append(**{**good, **bad})
    with pytest.raises(ops_gemm.HardwareUnsupported):
        mx.mx_append(**{**good, "q": q.cpu()})
    with pytest.raises(Exception, match="strides"):
        mx.mx_append(**{**good, "q": q[:, :2], "q_out": torch.as_strided(q, (3, 2, 64), (128, 64, 1))})
    for bad in (dict(slots=pos.float()), dict(slots=pos.view(1, 3)), dict(dtype=torch.float32), dict(slots=pos.cpu())):
        with pytest.raises(ConfigError):
            mx.mx_read(**{"cache": cache, "slots": pos, **bad})
    twin = copy.deepcopy(cache)
    assert "_made" not in twin.__dict__ and torch.equal(twin.k, cache.k)
