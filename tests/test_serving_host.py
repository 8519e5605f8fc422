"""Host side of the operators around a block-scaled cache, of the two-sided norm and of the sampling, on the CPU: the C entry points
refuse bad calls before any launch (the pointers are placeholders that no kernel sees), workspace queries follow the plan."""
from __future__ import annotations

import copy
import ctypes
import pickle

import pytest
import torch

from forge_amd import _lib
from forge_amd import ops_mx as mx
from forge_amd.errors import ConfigError, HardwareUnsupported
from forge_amd.ops_decoder import postnorm_add_rmsnorm
from forge_amd.ops_sampling import sample_tokens

P = ctypes.c_void_p(256)
ODD = ctypes.c_void_p(264)


def _cache(**kw):
    c = dict(k=256, v=256, k_scale=256, v_scale=256, page_stride=2048, head_stride=512, token_stride=32, num_pages=4, bits=4, kv_heads=2,
             page_size=16, head_dim=64)
    c.update(kw)
    return ctypes.byref(_lib.MXCache(*c.values()))


def _norm(**kw):
    a = dict(x=P, ldx=64, xdt=_lib.BF16, pw=P, pwdt=_lib.BF16, g=P, ldg=64, gdt=_lib.BF16, scale=1.0, post_eps=1e-5, r=ctypes.c_void_p(512), ldr=64,
             ro=ctypes.c_void_p(512), ldro=64, rdt=_lib.BF16, w=P, wdt=_lib.BF16, eps=1e-5, y=ctypes.c_void_p(1024), ldy=64, ydt=_lib.I8, s=P,
             s_row=1, s_block=0, block=0, m=2, k=64, stream=None)
    a.update(kw)
    return _lib.lib().fg_postnorm_add_rmsnorm(*a.values())


@pytest.mark.parametrize("bad,status", [(dict(m=-1), 1), (dict(k=0), 1), (dict(k=32769), 2), (dict(x=None), 1), (dict(r=None), 1),
                                        (dict(ro=None), 1), (dict(s=None), 1), (dict(xdt=_lib.I8), 1), (dict(pwdt=_lib.I8), 1),
                                        (dict(gdt=_lib.E4M3), 1), (dict(ldg=63), 1), (dict(ldg=-64), 1), (dict(rdt=_lib.F16), 1),
                                        (dict(ydt=_lib.F16), 1), (dict(block=24), 1), (dict(ldx=63), 1), (dict(s_row=-1), 1),
                                        (dict(g=ctypes.c_void_p(512)), 1), (dict(g=ctypes.c_void_p(1024)), 1),
                                        (dict(y=ctypes.c_void_p(512), ydt=_lib.BF16, block=0, s=None), 1)])
def test_norm_refusals(bad, status):
    assert _norm(**bad) == status and "fg_postnorm_add_rmsnorm" in _lib.last_error()


def test_no_work_is_no_error():
    assert _norm(m=0, x=None, y=None) == _lib.OK
    assert _append(t=0, q=None) == _lib.OK and _read(n=0, k=None) == _lib.OK
    assert _attention(t=0, b=0, q=None, out=None) == _lib.OK and _sample(b=0, x=None) == _lib.OK


CACHES = [(dict(k=None), 1), (dict(k_scale=None), 1), (dict(v=264), 1), (dict(page_stride=2040), 1), (dict(token_stride=24), 1),
          (dict(token_stride=16), 1), (dict(head_stride=-512), 1), (dict(head_stride=0), 1), (dict(num_pages=0), 1), (dict(page_size=0), 1),
          (dict(bits=6), 1), (dict(bits=8), 1), (dict(head_dim=80), 2), (dict(head_dim=288), 2), (dict(head_dim=0), 1),
          (dict(num_pages=2 ** 30, page_stride=2 ** 11), 2), (dict(num_pages=2 ** 31), 1)]


def _append(cache=None, sections=None, **kw):
    a = dict(q=P, qt=256, qh=64, k=P, kt=128, kh=64, v=P, vt=128, vh=64, qo=P, qot=256, qoh=64, dt=_lib.BF16, pos=P, p64=1, ldp=3, axes=1,
             sections=None if sections is None else (ctypes.c_int32 * len(sections))(*sections), table=P, ld=64, max_pos=100, rot=64, inter=0,
             slots=P, s64=1, cache=_cache() if cache is None else cache, t=3, heads=4, stream=None)
    a.update(kw)
    return _lib.lib().fg_mx_append(*a.values())


def _read(cache=None, **kw):
    a = dict(cache=_cache() if cache is None else cache, slots=P, s64=1, k=P, v=P, dt=_lib.BF16, n=3, stream=None)
    a.update(kw)
    return _lib.lib().fg_mx_read(*a.values())


def _attention(cache=None, **kw):
    a = dict(q=P, qt=256, qh=64, dt=_lib.BF16, cache=_cache() if cache is None else cache, table=P, ld=100, lens=P, starts=None, t=3, b=3,
             heads=4, seq=1600, maxq=1, scale=0.1, cap=0.0, window=0, out=P, ot=256, oh=64, lse=None, ws=None, bytes=0, stream=None)
    a.update(kw)
    return _lib.lib().fg_mx_attention(*a.values())


@pytest.mark.parametrize("bad,status", CACHES)
def test_cache_refusals(bad, status):
    assert _append(_cache(**bad)) == status and _read(_cache(**bad)) == status and _attention(_cache(**bad)) == status


@pytest.mark.parametrize("bad", [dict(t=-1), dict(heads=0), dict(dt=_lib.F32), dict(q=None), dict(table=None), dict(rot=0), dict(rot=63),
                                 dict(rot=66), dict(ld=62), dict(max_pos=-1), dict(k=None), dict(slots=None), dict(qot=100), dict(qt=512),
                                 dict(axes=0), dict(axes=5), dict(axes=2), dict(axes=2, sections=(16, 15)), dict(axes=2, sections=(33, -1)),
                                 dict(axes=2, sections=(16, 16), ldp=2), dict(sections=(31,))])
def test_append_refusals(bad):
    assert _append(**bad) == _lib.EINVAL and "fg_mx_append" in _lib.last_error()


@pytest.mark.parametrize("bad", [dict(n=-1), dict(slots=None), dict(k=None), dict(v=ODD), dict(dt=_lib.F32)])
def test_read_refusals(bad):
    assert _read(**bad) == _lib.EINVAL and "fg_mx_read" in _lib.last_error()


@pytest.mark.parametrize("bad,why", [(dict(t=2), "query token"), (dict(maxq=2), "query token"), (dict(heads=3), "kv_heads"), (dict(heads=0), "sizes"),
                                     (dict(maxq=0), "sizes"), (dict(window=-1), "sizes"), (dict(seq=1601), "page table"), (dict(lens=None), "null"),
                                     (dict(out=None), "null"), (dict(table=None), "null"), (dict(), "workspace"), (dict(ws=ODD, bytes=1 << 30), "workspace"),
                                     (dict(ws=P, bytes=64), "workspace"), (dict(t=2 ** 28, b=2 ** 28), "32 bits"), (dict(cap=-1.0), "softcap"),
                                     (dict(cap=float("nan")), "softcap"), (dict(dt=_lib.F32), "fp16"), (dict(ot=100), "overlap")])
def test_attention_refusals(bad, why):
    assert _attention(**bad) == _lib.EINVAL and why in _lib.last_error()


def test_attention_workspace_follows_the_plan():
    ws = _lib.lib().fg_mx_attention_workspace_bytes
    assert ws(0, 4, 8, 2, 64, 4, 100, 1, 0, 1) == 0 and ws(4, 4, 7, 2, 64, 4, 100, 1, 0, 0) == 0
    assert ws(2 ** 28, 2 ** 28, 8, 2, 64, 4, 100, 1, 0, 0) == 0
    assert ws(64, 64, 32, 8, 128, 4, 4000, 1, 0, 0) == 0  # one part for each sequence: nothing to join
    row = 32 * (128 * 4 + 8)
    long = ws(1, 1, 32, 8, 128, 4, 8192, 1, 0, 0)
    assert long % row == 0 and long // row > 4
    assert 0 < ws(1, 1, 32, 8, 128, 4, 8192, 1, 1000, 0) < long  # a window has fewer keys to split
    assert ws(1, 1, 32, 8, 128, 4, 8192, 1, 10, 0) == 0
    assert ws(3, 0, 8, 2, 64, 8, 0, 1, 0, 1) > 0  # tokens of no sequence


def _sample(**kw):
    a = dict(x=P, ld=100, dt=_lib.F32, u=P, t=None, t_all=1.0, k=None, k_all=0, p=None, p_all=1.0, m=None, m_all=0.0, token=P, logprob=None, b=2,
             v=100, ws=P, bytes=1 << 30, stream=None)
    a.update(kw)
    return _lib.lib().fg_sample_tokens(*a.values())


@pytest.mark.parametrize("bad,why", [(dict(b=-1), "sizes"), (dict(b=1 << 16), "sizes"), (dict(v=0), "sizes"), (dict(v=2 ** 30), "sizes"), (dict(x=None), "null"),
                                     (dict(u=None), "null"), (dict(token=None), "null"), (dict(dt=_lib.I8), "dtype"), (dict(ld=-1), "stride"),
                                     (dict(ws=None), "workspace"), (dict(ws=ODD), "workspace"), (dict(bytes=100), "workspace")])
def test_sample_refusals(bad, why):
    assert _sample(**bad) == _lib.EINVAL and why in _lib.last_error()


def test_sample_workspace():
    ws = _lib.lib().fg_sample_workspace_bytes
    assert ws(0, 100) == 0 and ws(-1, 100) == 0 and ws(1, 0) == 0
    assert 0 < ws(1, 100) and ws(7, 100) == 7 * ws(1, 100)


def test_cache_descriptions():
    cache = mx.MXKVCache.allocate(4, 2, 16, 96, "mxfp8", "cpu")
    assert (cache.page_size, cache.bits, cache.head_dim) == (16, 8, 96) and cache._handle()[1:] == (2, 16, 96, 8)
    k, s = cache.k, cache.k_scale
    four = mx.MXKVCache.allocate(4, 2, 16, 96, "mxfp4", "cpu")
    assert four.k.shape[3] == 48 and four.bits == 4
    mx.MXKVCache(*(t[1:3, :, 2:9] for t in (k, cache.v, s, cache.v_scale)))
    one = [t[:1, :1] for t in (k, cache.v, s, cache.v_scale)]
    mx.MXKVCache(one[0].contiguous(), one[1].contiguous(), one[2], one[3])
    for args in ((k, k[:3], s, s), (k, k, s[:3], s[:3]), (k.int(), k.int(), s, s), (k, k, s.float(), s.float()), (k[0], k[0], s[0], s[0]),
                 (k[..., :48], k[..., :48], s[..., :2], s[..., :2]), (k, k, s[..., :2], s[..., :2]), (k, k, s[..., :0], s[..., :0]),
                 (k, k.transpose(1, 2).contiguous().transpose(1, 2), s, s),
                 (k, k, s.transpose(1, 2).contiguous().transpose(1, 2), s.transpose(1, 2).contiguous().transpose(1, 2))):
        with pytest.raises(ConfigError):
            mx.MXKVCache(*args)
    for bad in (dict(fmt="fp4"), dict(head_dim=80), dict(head_dim=0)):
        with pytest.raises(ConfigError):
            mx.MXKVCache.allocate(**{"num_pages": 1, "kv_heads": 1, "page_size": 16, "head_dim": 64, "device": "cpu", **bad})


def test_copies_and_pickles_hold_the_tensors_only():
    cache = mx.MXKVCache.allocate(2, 1, 16, 32, "mxfp4", "cpu")
    first = cache._handle()
    assert cache._handle() is first
    for twin in (copy.deepcopy(cache), pickle.loads(pickle.dumps(cache))):
        assert "_made" not in twin.__dict__ and torch.equal(twin.k, cache.k)
        assert twin._handle()[0]._obj.k == twin.k.data_ptr()


def test_nothing_runs_on_the_cpu():
    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    cache = mx.MXKVCache.allocate(2, 1, 16, 64, "mxfp4", "cpu")
    q, i = torch.zeros(2, 1, 64, dtype=torch.bfloat16), torch.zeros(2, dtype=torch.int64)
    for call in (lambda: postnorm_add_rmsnorm(x, None, x, None), lambda: mx.mx_append(q, q, q, i, torch.zeros(4, 64), cache, i),
                 lambda: mx.mx_read(cache, i), lambda: mx.mx_attention(q, cache, i.int().view(2, 1), i.int()),
                 lambda: sample_tokens(torch.zeros(2, 5), torch.zeros(2))):
        with pytest.raises(HardwareUnsupported):
            call()
