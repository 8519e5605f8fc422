"""The operators of a serving decoder layer between its quantised linears, computed by libforge_mi355x.so only.

* :func:`add_rmsnorm`: the residual's addition, the RMSNorm and, if asked for, the 8-bit codes and scales that
  ``ops_gemm.int8_linear`` / ``fp8_linear`` take;
* :func:`rope_append`: the rotation of a projection's queries and keys by their positions, and the keys' and values' way
  into a :class:`PagedKVCache`;
* :func:`prefix_attention`: the attention that reads this cache, for a batch whose sequences share a prefix.

The reference runs these steps around its linears (``forge/models/attention.py:245-256``, ``forge/models/layers.py:167-173``).
As in ``ops_gemm`` every op is one call into the C ABI (``include/forge_mi355x.h``) on the current stream, raises where it
cannot run, neither synchronises nor reads lengths on the host, and takes outputs and workspaces from torch's caching
allocator, so a layer can be captured in a HIP graph.
"""
from __future__ import annotations

import functools
from dataclasses import dataclass
from typing import NamedTuple

import torch

from . import _lib
from .errors import ConfigError
from .ops_gemm import _as_rows, _check, _done, _ld, _on_gpu

_16BIT = (torch.float16, torch.bfloat16)
_FLOATS = (torch.float32, *_16BIT)
_CODE = _lib.DTYPE_CODE
_QUANT = {None: None, "int8": torch.int8, "fp8": torch.float8_e4m3fn, "fp8_block": torch.float8_e4m3fn}


def _elsewhere(op: str, x: torch.Tensor, *tensors: torch.Tensor | None) -> None:
    """Raise if one of ``tensors`` is not on ``x``'s GPU."""
    dev = x.get_device()
    for t in tensors:
        if t is not None and t.get_device() != dev:
            raise ConfigError(f"{op}: a tensor is on {t.device}, the call is on {x.device}")


# ================================================================================================ norm
def _rows(t: torch.Tensor, k: int) -> tuple[torch.Tensor, int]:
    """``t [..., k]`` as rows of adjacent columns that do not overlap (copied only if they are not), and their stride."""
    if t.dim() == 2:
        ld, column = t.stride()
        if column == 1 and ld >= k:
            return t, ld
    t = _as_rows(t)
    return t, _ld(t)


class NormOutput(NamedTuple):
    y: torch.Tensor
    scale: torch.Tensor | None
    residual: torch.Tensor


def add_rmsnorm(x: torch.Tensor, weight: torch.Tensor | None, residual: torch.Tensor | None = None, *,
                eps: float = 1e-5, quant: str | None = None, block: int = 128,
                residual_out: torch.Tensor | None = None) -> NormOutput:
    """``h = x + residual`` and ``y = h / sqrt(mean(h^2) + eps) * weight`` over the last dimension, in one pass.

    ``h`` is rounded to the residual's type (``x``'s or fp32), is the new residual stream and is what is normed; it goes to
    ``residual_out`` (may be ``residual`` itself: in place) or a new tensor.  Without a residual ``h`` is ``x``.
    ``quant``: ``None`` gives ``y`` in ``x``'s type and no scale, ``"int8"`` / ``"fp8"`` codes with one fp32 scale per row
    (``[M]``), ``"fp8_block"`` e4m3 codes with one per 1 x ``block`` columns (``[M, ceil(K / block)]``, the scales of a
    block of columns next to each other, as ``fp8_linear`` reads them fastest): what ``int8_linear`` does to its input,
    and what ``fp8_linear`` takes as ``x`` and ``x_scale``.

    ``ops_gemm.quantize_act_fp8(rms_eps=...)`` norms and quantises per token too, without a residual and with the weight
    after 1 / rms; here ``h * weight`` comes first, so codes and scales of the two can differ in their last step.  A row
    whose squares overflow fp32 gives zeros.
    """
    _on_gpu(x, "add_rmsnorm")
    if quant not in _QUANT:
        raise ConfigError(f"add_rmsnorm: unknown quant {quant!r}: use None, int8, fp8 or fp8_block")
    xdt = x.dtype
    if xdt not in _FLOATS:
        raise ConfigError("add_rmsnorm: x must be an fp32, fp16 or bf16 tensor")
    shape = x.shape
    if not shape:
        raise ConfigError("add_rmsnorm: x needs a last dimension to norm")
    k = shape[-1]
    _elsewhere("add_rmsnorm", x, weight, residual, residual_out)
    if weight is not None:
        if weight.shape != (k,) or weight.dtype not in _FLOATS:
            raise ConfigError(f"add_rmsnorm: weight must be an fp32, fp16 or bf16 tensor of [{k}]")
        if not weight.is_contiguous():
            weight = weight.contiguous()
    x2, ldx = _rows(x, k)
    m = x2.shape[0]
    r2 = ro2 = rdt = None
    ldr = ldro = 0
    if residual is not None:
        rdt = residual.dtype
        if residual.shape != shape or (rdt is not xdt and rdt is not torch.float32):
            raise ConfigError("add_rmsnorm: residual must have x's shape and x's type or fp32")
        r2, ldr = _rows(residual, k)
        if residual_out is None:
            residual_out, ldro = residual.new_empty(shape), k
            ro2 = residual_out  # contiguous: the address and k say all
        elif residual_out.shape != shape or residual_out.dtype is not rdt:
            raise ConfigError("add_rmsnorm: residual_out must be like residual")
        else:
            ro2, ldro = _rows(residual_out, k)
            if m and ro2.data_ptr() != residual_out.data_ptr():
                raise ConfigError("add_rmsnorm: residual_out must be rows of adjacent columns that do not overlap")
    elif residual_out is not None:
        raise ConfigError("add_rmsnorm: residual_out without a residual")
    ydt = _QUANT[quant] or xdt
    y = x.new_empty((m, k), dtype=ydt)
    scale, s_row, s_block = None, 0, 0
    if quant == "fp8_block":
        if block < 8 or block > 512 or block & (block - 1):
            raise ConfigError("add_rmsnorm: block is a power of two from 8 to 512")
        scale = x.new_empty((-(-k // block), m), dtype=torch.float32).t()
        s_row, s_block = 1, max(m, 1)
    elif quant is not None:
        scale, s_row = x.new_empty((m,), dtype=torch.float32), 1
    if m and k:
        status = _lib.lib().fg_add_rmsnorm(
            x2.data_ptr(), ldx, _CODE[xdt], _lib.ptr(r2), ldr, _lib.ptr(ro2), ldro, 0 if rdt is None else _CODE[rdt],
            _lib.ptr(weight), 0 if weight is None else _CODE[weight.dtype], eps, y.data_ptr(), k, _CODE[ydt], _lib.ptr(scale),
            s_row, s_block, block if quant == "fp8_block" else 0, m, k, _lib.stream_of(x2))
        if status:
            _check(status, "fg_add_rmsnorm")
    _done("add_rmsnorm")
    return NormOutput(y if x2 is x else y.view(shape), scale, x if residual is None else residual_out)


# ================================================================================================ paged cache
@dataclass(frozen=True)
class PagedKVCache:
    """Keys and values of many sequences in pages: ``k`` and ``v`` are ``[pages, kv_heads, page_size, head_dim]`` (any
    strides of whole 16-byte units, the same for both, columns adjacent) in fp16, bf16 or float8_e4m3fn; an e4m3 value
    stands for ``code * k_scale[head]`` (``v_scale``), fp32 ``[kv_heads]``, of any sign.  A page holds each key head's tokens
    next to each other (:meth:`allocate`), the order in which attention reads them.  Rows that share memory, as those of keys
    expanded over heads, can be read but not appended to."""

    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor | None = None
    v_scale: torch.Tensor | None = None

    def __post_init__(self) -> None:
        k, v = self.k, self.v
        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype or k.device != v.device:
            raise ConfigError("PagedKVCache: k and v are [pages, kv_heads, page_size, head_dim] of one type on one device")
        if k.dtype not in (*_16BIT, torch.float8_e4m3fn):
            raise ConfigError("PagedKVCache: fp16, bf16 or float8_e4m3fn")
        if k.stride() != v.stride() or k.stride(3) != 1:
            raise ConfigError("PagedKVCache: k and v need the same strides and adjacent columns")
        for name in ("k_scale", "v_scale"):
            s = getattr(self, name)
            if (s is not None) != (k.dtype == torch.float8_e4m3fn):
                raise ConfigError("PagedKVCache: k_scale and v_scale belong to a float8_e4m3fn cache, and to no other")
            if s is not None and (s.shape != (k.shape[1],) or s.dtype != torch.float32 or not s.is_contiguous()
                                  or s.device != k.device):
                raise ConfigError(f"PagedKVCache: {name} must be contiguous fp32 of [{k.shape[1]}] on the cache's device")

    @classmethod
    def allocate(cls, num_pages: int, kv_heads: int, page_size: int, head_dim: int, dtype: torch.dtype = torch.bfloat16,
                 device: str | torch.device = "cuda", k_scale: torch.Tensor | None = None,
                 v_scale: torch.Tensor | None = None) -> PagedKVCache:
        """An empty cache; scales of an e4m3 cache default to 1."""
        shape = (num_pages, kv_heads, page_size, head_dim)
        if dtype == torch.float8_e4m3fn:
            k_scale, v_scale = (torch.ones(kv_heads, device=device) if s is None else s for s in (k_scale, v_scale))
        return cls(torch.zeros(shape, dtype=torch.uint8, device=device).view(dtype) if dtype == torch.float8_e4m3fn
                   else torch.zeros(shape, dtype=dtype, device=device),
                   torch.zeros(shape, dtype=torch.uint8, device=device).view(dtype) if dtype == torch.float8_e4m3fn
                   else torch.zeros(shape, dtype=dtype, device=device), k_scale, v_scale)

    @property
    def page_size(self) -> int:
        return self.k.shape[2]

    def _handle(self) -> tuple[object, torch.dtype, tuple[int, ...]]:
        """The C description (made on first use, and again where a tensor's memory, shape or order has changed), type and
        shape (``v`` has ``k``'s: of the two, ``k``'s are compared).  The description comes as the reference that the C call
        takes, which keeps it alive: another thread may make it again during the call."""
        k, v, ks, vs = self.k, self.v, self.k_scale, self.v_scale
        now = (k.data_ptr(), v.data_ptr(), k.shape, k.stride(), None if ks is None else (ks.data_ptr(), vs.data_ptr()))
        got = self.__dict__.get("_made")
        if got is None or got[0] != now:
            self.__post_init__()
            shape, (sp, sh, st, _) = tuple(k.shape), k.stride()
            made = _lib.KVCache(_lib.ptr(k), _lib.ptr(v), _lib.ptr(ks), _lib.ptr(vs), sp, sh, st, shape[0], _CODE[k.dtype],
                                *shape[1:])
            got = self.__dict__["_made"] = (now, (_lib.ctypes.byref(made), k.dtype, shape))
        return got[1]

    def __getstate__(self) -> dict:
        """What a copy or a pickle holds: the tensors.  The description is of this object's memory."""
        return {n: t for n, t in self.__dict__.items() if n != "_made"}


def _overlaps(token: int, head: int, t: int, h: int, dim: int) -> bool:
    """Whether rows of ``dim`` columns at these strides (expanded from fewer, or windows that slide, say) share elements."""
    if head >= dim and token >= (h - 1) * head + dim:
        return False  # a token steps over its heads
    if (t > 1 and token < dim) or (h > 1 and head < dim):
        return True
    if t <= 1 or h <= 1:
        return False
    (n, few), (m, many) = sorted(((t, token), (h, head)))
    # steps of the short axis, and the nearest step of the long one
    return any(abs(i * few - min((i * few + many // 2) // many, m - 1) * many) < dim for i in range(1, n))


def _index(op: str, name: str, t: torch.Tensor, n: int) -> torch.Tensor:
    if t.shape != (n,) or (t.dtype is not torch.int64 and t.dtype is not torch.int32):
        raise ConfigError(f"{op}: {name} must be an int32 or int64 tensor of [{n}]")
    return t if t.is_contiguous() else t.contiguous()


def _queries(op: str, q: torch.Tensor, cdt: torch.dtype, dim: int) -> tuple[torch.Tensor, torch.Size]:
    """``q`` as ``[tokens, heads, dim]`` with adjacent columns (copied only if they are not), of a type that the cache takes,
    and its shape."""
    shape = q.shape
    if len(shape) != 3 or shape[2] != dim:
        raise ConfigError(f"{op}: q must be [tokens, heads, {dim}], got {list(shape)}")
    dt = q.dtype
    if dt is not torch.bfloat16 and dt is not torch.float16:
        raise ConfigError(f"{op}: q must be fp16 or bf16")
    if cdt is not dt and cdt is not torch.float8_e4m3fn:
        raise ConfigError(f"{op}: a {cdt} cache does not take {dt} queries")
    return q if q.stride(2) == 1 or dim == 1 else q.contiguous(), shape


def _result(op: str, name: str, out: torch.Tensor | None, q: torch.Tensor, shape: torch.Size) -> tuple[torch.Tensor, int, int]:
    """``out``, or a new tensor like ``q``, and its strides of tokens and heads."""
    t, h, dim = shape
    if out is None:
        return q.new_empty(shape), h * dim, dim
    if out.shape != shape or out.dtype is not q.dtype or (out.stride(2) != 1 and dim > 1):
        raise ConfigError(f"{op}: {name} must be like q, with adjacent columns")
    token, head, _ = out.stride()
    if t and _overlaps(token, head, t, h, dim):
        raise ConfigError(f"{op}: {name}'s rows overlap")
    return out, token, head


# ================================================================================================ rotation and append
def rope_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor, cos_sin: torch.Tensor,
                cache: PagedKVCache, slots: torch.Tensor, *, interleaved: bool = False,
                q_out: torch.Tensor | None = None) -> torch.Tensor:
    """Rotate ``q [T, heads, dim]`` and ``k [T, kv_heads, dim]`` by ``positions [T]``, write ``k`` and ``v`` to the cache's
    ``slots [T]`` (``page * page_size + token``; one outside the cache, as -1, is padding) and return the rotated ``q``
    (in ``q_out``, which may be ``q``, or a new tensor).

    ``cos_sin``: fp32 ``[max_position, rot]``, the cosines of the ``rot / 2`` pairs, then their sines; the first ``rot``
    columns of a head turn, in pairs ``(i, i + rot / 2)`` or, ``interleaved``, ``(2 i, 2 i + 1)``; the others pass through.
    The rotation is fp32, rounded once to the result's type; an e4m3 cache takes ``value / scale`` of its key head, clamped
    to +-448.  ``q``, ``k``, ``v`` may be views of one projection's output.  A position outside the table gives NaN.  What a
    slot given to two tokens then holds is undefined: each head's columns may come from either.
    """
    op = "rope_append"
    _on_gpu(q, op)
    handle, cdt, (_, hk, _, dim) = cache._handle()
    _elsewhere(op, q, k, v, positions, cos_sin, slots, cache.k, q_out)
    q, shape = _queries(op, q, cdt, dim)
    dt = q.dtype
    t, h, _ = shape
    if k.shape != (t, hk, dim) or v.shape != (t, hk, dim) or k.dtype is not dt or v.dtype is not dt:
        raise ConfigError(f"{op}: k and v must be [{t}, {hk}, {dim}] of q's type")
    table = cos_sin.shape
    if len(table) != 2 or cos_sin.dtype is not torch.float32:
        raise ConfigError(f"{op}: cos_sin must be fp32 [positions, rot]")
    max_pos, rot = table
    if rot % 2 or not 2 <= rot <= dim:
        raise ConfigError(f"{op}: cos_sin's rot must be even and up to {dim}, got {rot}")
    positions, slots = _index(op, "positions", positions, t), _index(op, "slots", slots, t)
    (k0, k1, kc), (v0, v1, vc), (ld, tc) = k.stride(), v.stride(), cos_sin.stride()
    if kc != 1 or vc != 1 or tc != 1 or max_pos <= 1:
        k, v, cos_sin = k.contiguous() if kc != 1 else k, v.contiguous() if vc != 1 else v, cos_sin.contiguous()
        (k0, k1, _), (v0, v1, _), ld = k.stride(), v.stride(), rot
    q_out, o0, o1 = _result(op, "q_out", q_out, q, shape)
    if t:
        q0, q1, _ = q.stride()
        status = _lib.lib().fg_rope_append(
            q.data_ptr(), q0, q1, k.data_ptr(), k0, k1, v.data_ptr(), v0, v1, q_out.data_ptr(), o0, o1, _CODE[dt],
            positions.data_ptr(), positions.dtype is torch.int64, cos_sin.data_ptr(), ld, max_pos, rot, interleaved,
            slots.data_ptr(), slots.dtype is torch.int64, handle, t, h, _lib.stream_of(q))
        if status:
            _check(status, "fg_rope_append")
    _done(op)
    return q_out


# ================================================================================================ attention
def prefix_attention(q: torch.Tensor, cache: PagedKVCache, page_table: torch.Tensor, seq_lens: torch.Tensor, *,
                     prefix_pages: torch.Tensor | None = None, prefix_len: int = 0,
                     query_start: torch.Tensor | None = None, max_query_len: int = 1, max_seq_len: int | None = None,
                     scale: float | None = None, return_lse: bool = False,
                     out: torch.Tensor | None = None) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """Attention of ``q [T, heads, dim]`` over the cache, for B sequences that share a prefix (which is read once for all):
    each query token sees the prefix and its own sequence's tokens up to itself.  Returns ``[T, heads, dim]`` in ``q``'s
    type, with ``return_lse`` also the logarithm of each row's softmax sum, fp32 ``[T, heads]``.

    * ``prefix_pages`` int32 ``[n]``, ``prefix_len``: the pages of the shared prefix, and its tokens (a host integer; 0: none);
    * ``page_table`` int32 ``[B, pages]``, ``seq_lens`` int32 ``[B]``: each sequence's own pages after the prefix, and how many
      tokens they hold, those of the queries included (appended before, with :func:`rope_append`).  Entries past the length,
      and what stands in their slots, are not read;
    * ``query_start`` int32 ``[B + 1]``: sequence b's queries are tokens ``query_start[b] .. query_start[b + 1]`` of ``q`` (offsets
      outside ``q`` count as its begin or end), and the last of its tokens; ``max_query_len`` bounds their number.  ``None``: one
      query token per sequence (decoding);
    * ``max_seq_len``: a host bound of ``seq_lens`` (default: what the page table can hold), by which the work is split;
    * ``heads`` is a multiple of the cache's ``kv_heads``; ``scale`` defaults to ``1 / sqrt(dim)``.

    Lengths are read on the GPU only.  Scores, softmax and sums are fp32; the probabilities are rounded to ``q``'s type for
    the product with the values, which adds about a third to the result's own rounding (fp16 keeps keys down to 2^-32 of the
    largest weight).  A row that sees no token gives zeros (lse -inf), as do query tokens of no sequence.  A query token past
    ``max_query_len`` gives NaN.  A NaN or infinity in a value that some query token of a sequence sees can show in that
    sequence's earlier query tokens too.
    """
    op = "prefix_attention"
    _on_gpu(q, op)
    handle, cdt, (_, hk, page, dim) = cache._handle()
    _elsewhere(op, q, page_table, seq_lens, prefix_pages, query_start, cache.k, out)
    q, shape = _queries(op, q, cdt, dim)
    dt = q.dtype
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
    if max_query_len < 1 or prefix_len < 0:
        raise ConfigError(f"{op}: max_query_len must be positive and prefix_len not negative")
    if max_seq_len is None:
        max_seq_len = width * page
    elif not 0 <= max_seq_len <= width * page:
        raise ConfigError(f"{op}: max_seq_len {max_seq_len} is past the page table's {width} pages of {page}")
    if prefix_len and (prefix_pages is None or prefix_pages.dim() != 1 or prefix_pages.dtype is not torch.int32
                       or prefix_pages.shape[0] * page < prefix_len):
        raise ConfigError(f"{op}: a prefix of {prefix_len} tokens needs int32 prefix_pages that hold them")
    out, o0, o1 = _result(op, "out", out, q, shape)
    lse = q.new_empty((t, h), dtype=torch.float32) if return_lse else None
    if t:
        q0, q1, _ = q.stride()
        ld, column = page_table.stride()
        if column != 1 or b <= 1 or ld < width:
            page_table, ld = page_table.contiguous(), width
        if not seq_lens.is_contiguous():
            seq_lens = seq_lens.contiguous()
        prefix_pages = prefix_pages.contiguous() if prefix_len else None
        query_start = query_start.contiguous() if ragged else None
        need = _attention_workspace(q.get_device(), t, b, h, hk, dim, prefix_len, max_seq_len, max_query_len, ragged, cdt)
        ws = q.new_empty((need,), dtype=torch.uint8) if need else None
        status = _lib.lib().fg_prefix_attention(
            q.data_ptr(), q0, q1, _CODE[dt], handle, _lib.ptr(prefix_pages), prefix_len, page_table.data_ptr(), ld,
            seq_lens.data_ptr(), _lib.ptr(query_start), t, b, h, max_seq_len, max_query_len,
            dim ** -0.5 if scale is None else scale, out.data_ptr(), o0, o1, _lib.ptr(lse), _lib.ptr(ws), need,
            _lib.stream_of(q))
        if status:
            _check(status, "fg_prefix_attention")
    _done(op)
    return (out, lse) if return_lse else out


@functools.lru_cache(maxsize=1024)
def _attention_workspace(_device: int, t: int, b: int, h: int, hk: int, dim: int, prefix_len: int, max_seq_len: int,
                         max_query_len: int, ragged: bool, cdt: torch.dtype) -> int:
    """Bytes of a call's partial sums, which follow from its sizes (and the GPU's CUs) alone."""
    return _lib.lib().fg_prefix_attention_workspace_bytes(t, b, h, hk, dim, _CODE[cdt], prefix_len, max_seq_len, max_query_len,
                                                          ragged)
