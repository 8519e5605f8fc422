"""A paged cache in 4 or 8 bits with a power-of-two scale for each 32 columns, the way into it, back out of it, and the attention
that reads it, computed by libforge_mi355x.so only.

* :class:`MXKVCache`: keys and values in the OCP microscaling formats, e2m1 (4 bits) or e4m3 (8 bits) codes with e8m0 scales;
* :func:`mx_append`: rotation by positions of one or several axes, and the new tokens' codes and scales;
* :func:`mx_read`: tokens of the cache as 16-bit values;
* :func:`mx_attention`: attention over this cache, with a tanh cap on the scores and a window.

Beside :class:`ops_decoder.PagedKVCache`, whose e4m3 form has one given scale per head, this cache takes its scales from the values
as they are written.  As in ``ops_decoder`` every op is one call into the C ABI (``include/forge_mi355x.h``) on the current
stream, raises where it cannot run, neither synchronises nor reads lengths on the host, and takes outputs and workspaces from
torch's caching allocator, so a layer can be captured in a HIP graph.
"""
from __future__ import annotations

import functools
from dataclasses import dataclass

import torch

from . import _lib
from .errors import ConfigError
from .ops_decoder import _elsewhere, _index, _result
from .ops_gemm import _check, _done, _on_gpu

_CODE = _lib.DTYPE_CODE
BLOCK = 32  # columns that share a scale
_BITS = {"mxfp4": 4, "mxfp8": 8}


@dataclass(frozen=True)
class MXKVCache:
    """Keys and values of many sequences in pages of block-scaled codes: ``k`` and ``v`` are uint8
    ``[pages, kv_heads, page_size, head_dim * bits / 8]`` (``bits`` 4: e2m1, two columns a byte, the even one low; 8: e4m3), ``k_scale``
    and ``v_scale`` uint8 ``[pages, kv_heads, page_size, head_dim / 32]``, the exponents of each 32 columns' scale (e8m0: byte b is
    ``2^(b - 127)``, 255 NaN).  ``head_dim`` is a multiple of 32.  All strides are ``k``'s (columns adjacent, 16-byte aligned), the
    scales' in proportion, as they are for tensors of one order (:meth:`allocate`) and for the same slices of them."""

    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor

    def __post_init__(self) -> None:
        k, s = self.k, self.k_scale
        for t in (k, self.v, s, self.v_scale):
            if t.dim() != 4 or t.dtype is not torch.uint8 or t.device != k.device:
                raise ConfigError("MXKVCache: codes and scales are 4-dimensional uint8 tensors on one device")
        if k.shape != self.v.shape or s.shape != self.v_scale.shape or k.shape[:3] != s.shape[:3]:
            raise ConfigError("MXKVCache: k and v, their scales and their tokens need the same shape")
        if k.stride() != self.v.stride() or s.stride() != self.v_scale.stride() or k.stride(3) != 1 or \
                (s.stride(3) != 1 and s.shape[3] > 1):
            raise ConfigError("MXKVCache: k and v, and their scales, need the same strides and adjacent columns")
        width, blocks = k.shape[3], s.shape[3]
        if blocks == 0 or width not in (16 * blocks, 32 * blocks):
            raise ConfigError("MXKVCache: rows of 16 (4 bits) or 32 (8 bits) bytes of codes for each scale")
        per = width // blocks
        if any(n > 1 and a != per * b for n, a, b in zip(k.shape[:3], k.stride(), s.stride())):
            raise ConfigError(f"MXKVCache: the scales' strides must be the codes' divided by {per}")

    @classmethod
    def allocate(cls, num_pages: int, kv_heads: int, page_size: int, head_dim: int, fmt: str = "mxfp4",
                 device: str | torch.device = "cuda") -> MXKVCache:
        """A cache of zeros; ``fmt`` is ``"mxfp4"`` or ``"mxfp8"``."""
        if fmt not in _BITS:
            raise ConfigError(f"MXKVCache: unknown format {fmt!r}: use mxfp4 or mxfp8")
        if head_dim % BLOCK or head_dim <= 0:
            raise ConfigError(f"MXKVCache: head_dim must be a multiple of {BLOCK}, got {head_dim}")
        shape = (num_pages, kv_heads, page_size)
        k, v = (torch.zeros((*shape, head_dim * _BITS[fmt] // 8), dtype=torch.uint8, device=device) for _ in range(2))
        ks, vs = (torch.ones((*shape, head_dim // BLOCK), dtype=torch.uint8, device=device) for _ in range(2))
        return cls(k, v, ks, vs)

    @property
    def page_size(self) -> int:
        return self.k.shape[2]

    @property
    def bits(self) -> int:
        return self.k.shape[3] // self.k_scale.shape[3] // 4

    @property
    def head_dim(self) -> int:
        return self.k_scale.shape[3] * BLOCK

    def _handle(self) -> tuple[object, int, int, int, int]:
        """The C description (made on first use, and again where a tensor's memory, shape or order has changed) as the reference
        that the C call takes and keeps alive, key heads, page size, head columns, bits."""
        k, v, ks, vs = self.k, self.v, self.k_scale, self.v_scale
        now = (k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), k.shape, k.stride(), ks.stride())
        got = self.__dict__.get("_made")
        if got is None or got[0] != now:
            self.__post_init__()
            pages, hk, page, _ = k.shape
            dim, bits = self.head_dim, self.bits
            # a dimension of one has no stride
            strides = [s if n > 1 else 0 for n, s in zip(k.shape[:3], k.stride())]
            made = _lib.MXCache(_lib.ptr(k), _lib.ptr(v), _lib.ptr(ks), _lib.ptr(vs), *strides, pages, bits, hk, page, dim)
            got = self.__dict__["_made"] = (now, (_lib.ctypes.byref(made), hk, page, dim, bits))
        return got[1]

    def __getstate__(self) -> dict:
        """What a copy or a pickle holds: the tensors.  The description is of this object's memory."""
        return {n: t for n, t in self.__dict__.items() if n != "_made"}


def _heads(op: str, name: str, t: torch.Tensor, dim: int) -> torch.Tensor:
    """``t [tokens, heads, dim]`` with adjacent columns (copied only if they are not)."""
    if t.dim() != 3 or t.shape[2] != dim:
        raise ConfigError(f"{op}: {name} must be [tokens, heads, {dim}], got {list(t.shape)}")
    if t.dtype is not torch.bfloat16 and t.dtype is not torch.float16:
        raise ConfigError(f"{op}: {name} must be fp16 or bf16")
    return t if t.stride(2) == 1 else t.contiguous()


# ================================================================================================ into the cache
def mx_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor, cos_sin: torch.Tensor,
              cache: MXKVCache, slots: torch.Tensor, *, sections: tuple[int, ...] | None = None, interleaved: bool = False,
              q_out: torch.Tensor | None = None) -> torch.Tensor:
    """Rotate ``q [T, heads, dim]`` and ``k [T, kv_heads, dim]`` by ``positions``, write ``k``'s and ``v``'s codes and scales to the
    cache's ``slots [T]`` (``page * page_size + token``; one outside the cache, as -1, is padding) and return the rotated ``q`` (in
    ``q_out``, which may be ``q``, or a new tensor).  What a slot given to two tokens then holds is undefined: codes of the one may stand
    beside scales of the other.

    ``cos_sin``, the pairs and ``interleaved`` are those of :func:`ops_decoder.rope_append`.  ``positions`` is ``[T]`` or, with
    ``sections``, ``[axes, T]`` (up to four, as time, height and width of an image's tokens): the first ``sections[0]`` pairs turn
    by the first axis, the next ``sections[1]`` by the second and so on, ``rot / 2`` in all.  Queries are rotated in fp32; a rotated
    key is rounded to fp32 once and then to its code.  A block of 32 columns takes the smallest scale (from 2^-126 on) for which no
    code is off by more than half its step; one with a NaN or an infinity, or a position outside the table, reads as NaN.
    """
    op = "mx_append"
    _on_gpu(q, op)
    handle, hk, _, dim, _ = cache._handle()
    _elsewhere(op, q, k, v, positions, cos_sin, slots, cache.k, q_out)
    q = _heads(op, "q", q, dim)
    dt, shape = q.dtype, q.shape
    t, h, _ = shape
    if k.shape != (t, hk, dim) or v.shape != (t, hk, dim) or k.dtype is not dt or v.dtype is not dt:
        raise ConfigError(f"{op}: k and v must be [{t}, {hk}, {dim}] of q's type")
    table = cos_sin.shape
    if len(table) != 2 or cos_sin.dtype is not torch.float32:
        raise ConfigError(f"{op}: cos_sin must be fp32 [positions, rot]")
    max_pos, rot = table
    if rot % 2 or not 2 <= rot <= dim:
        raise ConfigError(f"{op}: cos_sin's rot must be even and up to {dim}, got {rot}")
    axes, ends = 1, None
    if sections is None:
        positions = _index(op, "positions", positions, t)
    else:
        axes = len(sections)
        if not 1 <= axes <= 4 or min(sections) < 0 or sum(sections) != rot // 2:
            raise ConfigError(f"{op}: sections are up to four numbers of pairs, {rot // 2} in all, got {sections}")
        if positions.shape != (axes, t) or positions.dtype not in (torch.int32, torch.int64):
            raise ConfigError(f"{op}: positions must be an int32 or int64 tensor of [{axes}, {t}]")
        if not positions.is_contiguous():
            positions = positions.contiguous()
        ends = (_lib.ctypes.c_int32 * axes)(*sections)
    slots = _index(op, "slots", slots, t)
    if k.stride(2) != 1:
        k = k.contiguous()
    if v.stride(2) != 1:
        v = v.contiguous()
    ld, column = cos_sin.stride()
    if column != 1 or max_pos <= 1:
        cos_sin, ld = cos_sin.contiguous(), rot
    q_out, o0, o1 = _result(op, "q_out", q_out, q, shape)
    if t and h:
        q0, q1, _ = q.stride()
        k0, k1, _ = k.stride()
        v0, v1, _ = v.stride()
        status = _lib.lib().fg_mx_append(
            q.data_ptr(), q0, q1, k.data_ptr(), k0, k1, v.data_ptr(), v0, v1, q_out.data_ptr(), o0, o1, _CODE[dt],
            positions.data_ptr(), positions.dtype is torch.int64, t, axes, ends, cos_sin.data_ptr(), ld, max_pos, rot, interleaved,
            slots.data_ptr(), slots.dtype is torch.int64, handle, t, h, _lib.stream_of(q))
        if status:
            _check(status, "fg_mx_append")
    _done(op)
    return q_out


# ================================================================================================ out of the cache
def mx_read(cache: MXKVCache, slots: torch.Tensor, *, dtype: torch.dtype = torch.bfloat16) -> tuple[torch.Tensor, torch.Tensor]:
    """The keys and values in the cache's ``slots [n]`` as ``[n, kv_heads, head_dim]`` each, in fp16 or bf16, exact where the type can
    hold the value (bf16 does from 2^-126 on).  A slot outside the cache gives zeros."""
    op = "mx_read"
    _on_gpu(cache.k, op)
    handle, hk, _, dim, _ = cache._handle()
    _elsewhere(op, cache.k, slots)
    if dtype is not torch.bfloat16 and dtype is not torch.float16:
        raise ConfigError(f"{op}: the values are fp16 or bf16")
    if slots.dim() != 1:
        raise ConfigError(f"{op}: slots must be an int32 or int64 tensor of [n]")
    n = slots.shape[0]
    slots = _index(op, "slots", slots, n)
    k, v = (torch.empty((n, hk, dim), dtype=dtype, device=slots.device) for _ in range(2))
    if n:
        status = _lib.lib().fg_mx_read(handle, slots.data_ptr(), slots.dtype is torch.int64, k.data_ptr(), v.data_ptr(), _CODE[dtype], n,
                                       _lib.stream_of(slots))
        if status:
            _check(status, "fg_mx_read")
    _done(op)
    return k, v


# ================================================================================================ attention
def mx_attention(q: torch.Tensor, cache: MXKVCache, page_table: torch.Tensor, seq_lens: torch.Tensor, *,
                 query_start: torch.Tensor | None = None, max_query_len: int = 1, max_seq_len: int | None = None,
                 scale: float | None = None, softcap: float | None = None, window: int | None = None, return_lse: bool = False,
                 out: torch.Tensor | None = None) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """Attention of ``q [T, heads, dim]`` over the cache, for B sequences: each query token sees its sequence's tokens up to itself,
    with ``window`` the last ``window`` of them (its own included).  Scores are ``scale * q.k`` or, with ``softcap``,
    ``softcap * tanh(scale * q.k / softcap)``.  Returns ``[T, heads, dim]`` in ``q``'s type, with ``return_lse`` also the logarithm of
    each row's softmax sum, fp32 ``[T, heads]``.

    ``page_table``, ``seq_lens``, ``query_start``, ``max_query_len``, ``max_seq_len``, ``scale`` and ``out`` are those of
    :func:`ops_decoder.prefix_attention`, as is what tokens of no sequence, rows that see no token (zeros, lse -inf), query tokens
    past ``max_query_len`` (NaN) and page ids outside the cache (no tokens) give.

    Codes become ``q``'s type exactly, but for fp16 queries over values past 65504 (infinite) or below 2^-24.  Scores, softmax and
    sums are fp32, a capped score within ``2^-20 * softcap``; the probabilities are rounded to ``q``'s type for the product with the
    values.  A NaN block that some query token of a sequence sees can show in that sequence's earlier query tokens too.
    """
    op = "mx_attention"
    _on_gpu(q, op)
    handle, hk, page, dim, bits = cache._handle()
    _elsewhere(op, q, page_table, seq_lens, query_start, cache.k, out)
    q = _heads(op, "q", q, dim)
    shape = q.shape
    t, h, _ = shape
    if h % hk or h == 0:
        raise ConfigError(f"{op}: {h} query heads are no multiple of {hk} key heads")
    pages = page_table.shape
    if len(pages) != 2 or page_table.dtype is not torch.int32:
        raise ConfigError(f"{op}: page_table must be int32 [sequences, pages]")
    b, width = pages
    if seq_lens.shape != (b,) or seq_lens.dtype is not torch.int32:
        raise ConfigError(f"{op}: seq_lens must be int32 [{b}]")
    ragged = query_start is not None
    if ragged and (query_start.shape != (b + 1,) or query_start.dtype is not torch.int32):
        raise ConfigError(f"{op}: query_start must be int32 [{b + 1}]")
    if not ragged and (t != b or max_query_len != 1):
        raise ConfigError(f"{op}: without query_start each of the {b} sequences has one query token, got {t}")
    if max_query_len < 1:
        raise ConfigError(f"{op}: max_query_len must be positive")
    if max_seq_len is None:
        max_seq_len = width * page
    elif not 0 <= max_seq_len <= width * page:
        raise ConfigError(f"{op}: max_seq_len {max_seq_len} is past the page table's {width} pages of {page}")
    if window is None:
        window = 0
    elif window < 1:
        raise ConfigError(f"{op}: window must be positive (None: all tokens)")
    if softcap is None:
        softcap = 0.0
    elif not softcap > 0:
        raise ConfigError(f"{op}: softcap must be positive (None: no cap)")
    out, o0, o1 = _result(op, "out", out, q, shape)
    lse = q.new_empty((t, h), dtype=torch.float32) if return_lse else None
    if t:
        q0, q1, _ = q.stride()
        ld, column = page_table.stride()
        if column != 1 or b <= 1 or ld < width:
            page_table, ld = page_table.contiguous(), width
        if not seq_lens.is_contiguous():
            seq_lens = seq_lens.contiguous()
        query_start = query_start.contiguous() if ragged else None
        need = _attention_workspace(q.get_device(), t, b, h, hk, dim, bits, max_seq_len, max_query_len, window, ragged)
        ws = q.new_empty((need,), dtype=torch.uint8) if need else None
        status = _lib.lib().fg_mx_attention(
            q.data_ptr(), q0, q1, _CODE[q.dtype], handle, page_table.data_ptr(), ld, seq_lens.data_ptr(), _lib.ptr(query_start), t, b, h,
            max_seq_len, max_query_len, dim ** -0.5 if scale is None else scale, softcap, window, out.data_ptr(), o0, o1, _lib.ptr(lse),
            _lib.ptr(ws), need, _lib.stream_of(q))
        if status:
            _check(status, "fg_mx_attention")
    _done(op)
    return (out, lse) if return_lse else out


@functools.lru_cache(maxsize=1024)
def _attention_workspace(_device: int, t: int, b: int, h: int, hk: int, dim: int, bits: int, max_seq_len: int, max_query_len: int,
                         window: int, ragged: bool) -> int:
    """Bytes of a call's partial sums, which follow from its sizes (and the GPU's CUs) alone."""
    return _lib.lib().fg_mx_attention_workspace_bytes(t, b, h, hk, dim, bits, max_seq_len, max_query_len, window, ragged)
