"""Host side of the operators between a decoder layer's linears, on the CPU: the C entry points refuse bad calls before any
launch (the pointers are placeholders that no kernel sees), and the workspace query follows the plan."""
from __future__ import annotations

import copy
import ctypes
import gc
import pickle
import weakref

import pytest
import torch

from forge_amd import _lib
from forge_amd import ops_decoder as ops
from forge_amd.errors import ConfigError, HardwareUnsupported

P = ctypes.c_void_p(256)
ODD = ctypes.c_void_p(264)


def _cache(**kw):
    c = dict(k=256, v=256, k_scale=None, v_scale=None, page_stride=8192, head_stride=1024, token_stride=64, num_pages=4,
             dtype=_lib.BF16, kv_heads=2, page_size=16, head_dim=64)
    c.update(kw)
    return _lib.KVCache(**c)


def _norm(**kw):
    a = dict(x=P, ldx=64, xdt=_lib.BF16, r=P, ldr=64, ro=P, ldro=64, rdt=_lib.BF16, w=P, wdt=_lib.BF16, eps=1e-5, y=P, ldy=64,
             ydt=_lib.I8, s=P, s_row=1, s_block=0, block=0, m=2, k=64, stream=None)
    a.update(kw)
    return _lib.lib().fg_add_rmsnorm(*a.values())


@pytest.mark.parametrize("bad,status", [(dict(m=-1), 1), (dict(k=0), 1), (dict(k=32769), 2), (dict(x=None), 1), (dict(ro=None), 1),
                                        (dict(s=None), 1), (dict(xdt=_lib.I8), 1), (dict(rdt=_lib.F16), 1), (dict(ydt=_lib.F16), 1),
                                        (dict(block=24), 1), (dict(block=1024), 1), (dict(ydt=_lib.BF16, block=64), 1),
                                        (dict(ldx=63), 1), (dict(ldro=5), 1), (dict(wdt=_lib.E4M3), 1), (dict(s_row=-1), 1)])
def test_norm_refusals(bad, status):
    assert _norm(**bad) == status and "fg_add_rmsnorm" in _lib.last_error()


def test_no_work_is_no_error():
    assert _norm(m=0, x=None, y=None) == _lib.OK


CACHES = [(dict(k=None), 1), (dict(k=264), 1), (dict(page_stride=8190), 1), (dict(token_stride=56), 1), (dict(head_stride=-64), 1),
          (dict(num_pages=0), 1), (dict(page_size=0), 1), (dict(dtype=_lib.F16), 1), (dict(dtype=_lib.E4M3), 1),
          (dict(dtype=_lib.F32), 1), (dict(head_dim=264, token_stride=264), 2), (dict(head_dim=60), 2),
          (dict(num_pages=2 ** 23, page_stride=2 ** 13), 2), (dict(num_pages=2 ** 31, page_stride=8), 1)]


def _append(cache=None, **kw):
    a = dict(q=P, qt=256, qh=64, k=P, kt=128, kh=64, v=P, vt=128, vh=64, qo=P, qot=256, qoh=64, dt=_lib.BF16, pos=P, p64=1,
             table=P, ld=64, max_pos=100, rot=64, inter=0, slots=P, s64=1,
             cache=ctypes.byref(_cache() if cache is None else cache), t=3, heads=4, stream=None)
    a.update(kw)
    return _lib.lib().fg_rope_append(*a.values())


@pytest.mark.parametrize("bad", [dict(t=-1), dict(heads=0), dict(dt=_lib.F32), dict(q=None), dict(table=None), dict(rot=0),
                                 dict(rot=63), dict(rot=66), dict(ld=62), dict(max_pos=-1), dict(k=None)])
def test_append_refusals(bad):
    assert _append(**bad) == _lib.EINVAL and "fg_rope_append" in _lib.last_error()


@pytest.mark.parametrize("bad,status", CACHES)
def test_cache_refusals(bad, status):
    c = _cache(**bad)
    assert _append(c) == status and _attention(c) == status


def _attention(cache=None, **kw):
    a = dict(q=P, qt=256, qh=64, dt=_lib.BF16, cache=ctypes.byref(_cache() if cache is None else cache), pp=P, prefix=4000,
             table=P, ld=2, lens=P, starts=None, t=3, b=3, heads=4, seq=32, maxq=1, scale=0.1, out=P, ot=256, oh=64, lse=None,
             ws=None, bytes=0, stream=None)
    a.update(kw)
    return _lib.lib().fg_prefix_attention(*a.values())


@pytest.mark.parametrize("bad,why", [(dict(t=2), "query token"), (dict(maxq=2), "query token"), (dict(heads=3), "kv_heads"),
                                     (dict(heads=0), "sizes"), (dict(maxq=0), "sizes"), (dict(prefix=-1), "sizes"),
                                     (dict(seq=33), "page table"), (dict(pp=None), "null"), (dict(lens=None), "null"),
                                     (dict(out=None), "null"), (dict(), "workspace"), (dict(ws=ODD, bytes=1 << 30), "workspace"),
                                     (dict(ws=P, bytes=64), "workspace"), (dict(t=2 ** 30, b=2 ** 30), "32 bits")])
def test_attention_refusals(bad, why):
    assert _attention(**bad) == _lib.EINVAL and why in _lib.last_error()


def test_attention_without_queries_is_no_error():
    assert _attention(t=0, b=0, q=None, out=None) == _lib.OK


def test_workspace_follows_the_plan():
    query = _lib.lib().fg_prefix_attention_workspace_bytes

    def ws(t, b, h, hk, d, *rest):
        return query(t, b, h, hk, d, _lib.BF16, *rest)

    assert ws(0, 4, 8, 2, 64, 100, 100, 1, 1) == 0 and ws(4, 4, 7, 2, 64, 0, 100, 1, 0) == 0
    assert ws(64, 64, 32, 8, 128, 0, 100, 1, 0) == 0  # one part for each sequence: nothing to join
    row = 32 * (128 * 4 + 8)
    assert ws(1, 1, 32, 8, 128, 100, 100, 1, 0) == 0  # few keys: one part with the prefix's in it
    short = ws(1, 1, 32, 8, 128, 400, 100, 1, 0)
    assert short % row == 0 and short // row >= 2  # a longer prefix makes parts of its own
    assert ws(1, 1, 32, 8, 128, 0, 8192, 1, 0) > short
    assert ws(3, 0, 8, 2, 64, 0, 0, 1, 1) > 0  # tokens of no sequence


def test_cache_descriptions():
    k = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)
    ops.PagedKVCache(k, k.clone())
    one = torch.ones(2)
    e4 = torch.zeros(4, 2, 16, 64, dtype=torch.uint8).view(torch.float8_e4m3fn)
    cache = ops.PagedKVCache(e4, e4, one, one)
    assert cache.page_size == 16 and cache._handle()[1:] == (torch.float8_e4m3fn, (4, 2, 16, 64))
    for args in ((k, k[:3]), (k, k.half()), (k.float(), k.float()), (k[0], k[0]), (k, k.transpose(1, 2).contiguous().transpose(1, 2)),
                 (k.transpose(2, 3), k.transpose(2, 3)), (k, k, one, one), (e4, e4), (e4, e4, one), (e4, e4, one, torch.ones(3)),
                 (e4, e4, one, one.double())):
        with pytest.raises(ConfigError):
            ops.PagedKVCache(*args)


def test_allocate():
    c = ops.PagedKVCache.allocate(3, 2, 16, 64, torch.float8_e4m3fn, "cpu")
    assert c.k.shape == (3, 2, 16, 64) and c.k_scale.tolist() == [1, 1] and c.k.float().abs().max() == 0
    assert ops.PagedKVCache.allocate(3, 2, 16, 64, device="cpu").k.dtype == torch.bfloat16


def test_no_cpu_path(monkeypatch):
    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    with pytest.raises(HardwareUnsupported):
        ops.add_rmsnorm(x, None)
    monkeypatch.setenv("FORGE_FORCE_REF", "1")
    with pytest.raises(HardwareUnsupported, match="FORGE_FORCE_REF"):
        ops.add_rmsnorm(x, None)


def test_more_threads_than_a_launch_takes():
    for status in (_norm(m=2 ** 26), _append(t=2 ** 26), _append(t=2 ** 31 - 1, heads=1)):
        assert status == _lib.EHIP and "configuration" in _lib.last_error()
    assert _attention(t=2 ** 24, b=2 ** 24) == _lib.EINVAL and "more work items" in _lib.last_error()
    # 2^26 rows to join in 2^20 work items
    assert _attention(t=2 ** 24, b=2 ** 18, starts=P, maxq=64) == _lib.EINVAL and "more work items" in _lib.last_error()
    assert _attention(t=2 ** 24 - 1, b=2 ** 18, starts=P, maxq=64) == _lib.EINVAL and "workspace" in _lib.last_error()


@pytest.mark.parametrize("token,head,t,h,bad", [(256, 64, 3, 4, False), (64, 192, 3, 4, False), (0, 64, 3, 4, True), (256, 0, 3, 4, True),
                                                (0, 64, 1, 4, False), (256, 32, 3, 4, True), (256, 0, 3, 1, False)])
def test_rows_that_overlap(token, head, t, h, bad):
    assert ops._overlaps(token, head, t, h, 64) is bad


class _Tensors(ops.PagedKVCache):
    """A cache whose tensors move as a program's may: into new memory, to another shape or order."""

    def move(self, **to):
        for t in (self.k, self.v):
            x = torch.zeros(to.get("shape", t.shape), dtype=t.dtype)
            t.set_(x.transpose(1, 2) if to.get("turn") else x)


def _two_heads():
    return _Tensors(*(torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16) for _ in range(2)))


@pytest.mark.parametrize("op", ["append", "attention"])
def test_a_cache_description_lives_through_its_call(op, monkeypatch):
    """The C call reads it without the interpreter's lock, and another thread may have it made again meanwhile."""
    freed = []

    class Watched(_lib.KVCache):
        def __init__(self, *a):
            super().__init__(*a)
            weakref.finalize(self, freed.append, ctypes.addressof(self))

    cache, calls = _two_heads(), []

    class Lib:
        def call(self, *a):
            cache.move()
            cache._handle()  # what another thread's call does
            gc.collect()
            calls.append(list(freed))
            return _lib.OK

        fg_rope_append = fg_prefix_attention = call

        def fg_prefix_attention_workspace_bytes(self, *a):
            return 0

    for owner, name, value in ((_lib, "KVCache", Watched), (_lib, "lib", Lib), (_lib, "stream_of", lambda t: 0),
                               (ops, "_on_gpu", lambda *a: None)):
        monkeypatch.setattr(owner, name, value)
    q, k, i = torch.zeros(3, 4, 64, dtype=torch.bfloat16), torch.zeros(3, 2, 64, dtype=torch.bfloat16), torch.arange(3)
    if op == "append":
        ops.rope_append(q, k, k, i, torch.zeros(4, 64), cache, i)
    else:
        ops.prefix_attention(q, cache, torch.zeros(3, 1, dtype=torch.int32), i.int())
    assert calls == [[]]


def test_a_used_cache_can_be_copied_and_pickled():
    cache = ops.PagedKVCache.allocate(3, 2, 16, 64, torch.float8_e4m3fn, "cpu")
    assert cache._handle()[2] == (3, 2, 16, 64)
    for other in (copy.deepcopy(cache), copy.copy(cache)):
        assert other._handle()[1:] == cache._handle()[1:] and other.k_scale.tolist() == [1, 1]
    assert copy.deepcopy(cache).k.data_ptr() != cache.k.data_ptr()
    cache = ops.PagedKVCache.allocate(3, 2, 16, 64, device="cpu")  # torch unpickles no e4m3 tensors
    assert cache._handle()[1:] == pickle.loads(pickle.dumps(cache))._handle()[1:]


def _described(cache):
    made = cache._handle()[0]._obj
    return [getattr(made, f) for f, _ in _lib.KVCache._fields_]


def test_a_cache_description_follows_its_tensors():
    cache = _two_heads()
    first = _described(cache)
    assert first[4:8] == [2 * 16 * 64, 16 * 64, 64, 4]
    for t in (cache.k, cache.v):  # in place, at the same address
        t.resize_(2, 2, 16, 64)
    assert _described(cache)[:2] == first[:2] and _described(cache)[7] == 2 and cache._handle()[2] == (2, 2, 16, 64)
    cache.move(turn=True, shape=(2, 16, 2, 64))
    assert _described(cache)[4:7] == [2 * 16 * 64, 64, 2 * 64]
    cache.k.resize_(1, 2, 16, 64)
    with pytest.raises(ConfigError):
        cache._handle()


def test_a_query_bound_past_the_queries_is_the_queries():
    """No sequence has more query tokens than there are, so a looser bound asks for no other plan."""
    query = _lib.lib().fg_prefix_attention_workspace_bytes
    for t in (7, 300):
        want = query(t, 3, 8, 2, 64, _lib.BF16, 0, 5000, t, 1)
        for bound in (t + 1, 65536, 2 ** 31 - 2, 2 ** 62):
            assert query(t, 3, 8, 2, 64, _lib.BF16, 0, 5000, bound, 1) == want > 0
    # refused for the workspace, which comes after the sizes
    assert _attention(t=512, b=512, heads=64, ot=4096, starts=P, maxq=65536) == _lib.EINVAL and "workspace" in _lib.last_error()
    assert _attention(t=2 ** 62, b=2, starts=P, maxq=1) == _lib.EINVAL and "32 bits" in _lib.last_error()


def _cover(strides, counts, dim):
    """Whether the rows share an element, by listing all elements."""
    at = torch.zeros(1, dtype=torch.int64)
    for s, n in zip(strides, counts):
        at = (at.view(-1, 1) + s * torch.arange(n)).flatten()
    at = (at.view(-1, 1) + torch.arange(dim)).flatten()
    return len(at.unique()) < len(at)


@pytest.mark.parametrize("token,head,t,h,bad", [(64, 64, 3, 4, True), (192, 64, 3, 4, True), (64, 128, 3, 4, True), (128, 64, 1, 4, False),
                                                (192, 128, 2, 3, False), (192, 128, 2, 2, False), (192, 128, 3, 4, True), (100, 164, 2, 2, False),
                                                (100, 163, 2, 2, True), (63, 1000, 1, 4, False), (64, 256, 5, 4, True)])
def test_rows_that_overlap_across_tokens_and_heads(token, head, t, h, bad):
    assert _cover((token, head), (t, h), 64) is bad
    assert ops._overlaps(token, head, t, h, 64) is bad
    status = _append(t=t, heads=h, qot=token, qoh=head, pos=None)  # refused for its output first, for its positions else
    assert status == _lib.EINVAL and ("overlap" in _lib.last_error()) is bad
    status = _attention(_cache(kv_heads=1), t=t, b=t, heads=h, ot=token, oh=head)
    assert status == _lib.EINVAL and ("overlap" in _lib.last_error()) is bad and (bad or "workspace" in _lib.last_error())


def test_rows_that_overlap_by_their_elements():
    for token in (0, 8, 60, 64, 65, 100, 128, 192, 200):
        for head in (0, 50, 64, 72, 128, 130, 256):
            for t, h in ((1, 1), (1, 3), (2, 2), (3, 2), (2, 4), (5, 3)):
                assert ops._overlaps(token, head, t, h, 64) is _cover((token, head), (t, h), 64), (token, head, t, h)


@pytest.mark.parametrize("strides,pages,bad", [((2048, 0, 64), 4, True), ((0, 1024, 64), 4, True), ((0, 1024, 64), 1, False),
                                               ((1024, 1024, 64), 4, True), ((2048, 64, 128), 4, False), ((2048, 64, 64), 4, True),
                                               ((64, 4096, 256), 4, False), ((64, 2048, 192), 4, True), ((2112, 1056, 64), 4, False),
                                               ((2048, 1056, 64), 4, True)])
def test_caches_whose_rows_overlap_take_no_tokens(strides, pages, bad):
    """Such a cache can be read (keys expanded over heads, say), not written."""
    c = _cache(page_stride=strides[0], head_stride=strides[1], token_stride=strides[2], num_pages=pages)
    assert _cover(strides, (pages, 2, 16), 64) is bad
    assert _append(c, pos=None) == _lib.EINVAL and ("overlap" in _lib.last_error()) is bad
    assert _attention(c) == _lib.EINVAL and "workspace" in _lib.last_error()


@pytest.mark.parametrize("t,b,h,hk,d,prefix,seq,maxq", [(2 ** 24, 2 ** 18, 4, 2, 64, 4000, 32, 64), (2 ** 24, 2 ** 24, 4, 2, 64, 4000, 32, 1),
                                                        (2 ** 20, 2 ** 16, 64, 8, 128, 0, 8192, 511)])
def test_a_plan_that_is_refused_asks_for_no_workspace(t, b, h, hk, d, prefix, seq, maxq):
    """The caller would allocate it in front of the call, tens of GiB."""
    query = _lib.lib().fg_prefix_attention_workspace_bytes
    assert query(t, b, h, hk, d, _lib.BF16, prefix, seq, maxq, 1) == 0
    cache = _cache(kv_heads=hk, head_dim=d, head_stride=16 * d, token_stride=d, page_stride=16 * d * hk)
    status = _attention(cache, t=t, b=b, heads=h, ot=h * d, oh=d, prefix=prefix, seq=seq, ld=-(-seq // 16), starts=P, maxq=maxq)
    assert status == _lib.EINVAL and "more work items" in _lib.last_error()


@pytest.mark.parametrize("expanded", [False, True])
def test_one_page_list_for_all_sequences(expanded, monkeypatch):
    """A page table expanded over the sequences goes to the C call as rows of its own width, as any other."""
    seen = []

    class Lib:
        def fg_prefix_attention(self, *a):
            seen.append((a[7], a[8], a[14]))
            return _lib.OK

        def fg_prefix_attention_workspace_bytes(self, *a):
            return 0

    for owner, name, value in ((_lib, "lib", Lib), (_lib, "stream_of", lambda t: 0), (ops, "_on_gpu", lambda *a: None)):
        monkeypatch.setattr(owner, name, value)
    ops._attention_workspace.cache_clear()
    one = torch.arange(2, dtype=torch.int32).view(1, 2)
    table = one.expand(3, 2) if expanded else one.repeat(3, 1)
    q = torch.zeros(3, 4, 64, dtype=torch.bfloat16)
    ops.prefix_attention(q, _two_heads(), table, torch.full((3,), 20, dtype=torch.int32))
    assert len(seen) == 1 and seen[0][1] == 2 and seen[0][2] == 32
    ops._attention_workspace.cache_clear()


@pytest.mark.parametrize("bad,why", [(dict(y=1), "y"), (dict(y=1, ydt=_lib.BF16, ldy=72), "y"), (dict(y=2), "y"), (dict(y=2, ydt=_lib.BF16, rdt=_lib.F32), "y"),
                                     (dict(ro=2, ldro=72), "residual_out"), (dict(ro=1, rdt=_lib.F32), "residual_out"),
                                     (dict(y=3, ydt=_lib.BF16), "y"), (dict(y=3), "y")])
def test_norm_outputs_in_the_place_of_other_rows(bad, why):
    """An output in an input's place needs its type and stride: else a row lands where another, unread one stands."""
    place = {i: ctypes.c_void_p(4096 * i) for i in (1, 2, 3, 4)}  # of x, the residual, residual_out, y
    kw = dict(x=place[1], r=place[2], ro=place[3], y=place[4])
    kw.update({k: place[v] if k in ("y", "ro") else v for k, v in bad.items()})
    assert _norm(**kw) == _lib.EINVAL and f"{why} in the place of" in _lib.last_error()


@pytest.mark.parametrize("bad", [dict(qot=512), dict(qot=64, qoh=192), dict(qoh=72, qot=512)])
def test_rotated_queries_in_the_place_of_other_rows(bad):
    """In place means the rows' own strides: else a token lands where another, unread one stands."""
    assert _append(pos=None, **bad) == _lib.EINVAL and "in the place of" in _lib.last_error()
    assert _append(pos=None, qo=ctypes.c_void_p(4096), **bad) == _lib.EINVAL and "null" in _lib.last_error()
    assert _append(pos=None, t=1, qot=512) == _lib.EINVAL and "null" in _lib.last_error()
