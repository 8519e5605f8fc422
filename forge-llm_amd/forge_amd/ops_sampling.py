"""The next tokens from their logits, computed by libforge_mi355x.so only.

:func:`sample_tokens`: temperature, top-k, top-p, min-p and the draw by given random numbers, for a batch of rows whose settings may
differ.  As in ``ops_decoder`` it is one call into the C ABI (``include/forge_mi355x.h``) on the current stream, raises where it
cannot run, does not synchronise or read settings on the host, and takes its results and workspace from torch's caching allocator,
so a decoding step can be captured in a HIP graph with it.
"""
from __future__ import annotations

import functools

import torch

from . import _lib
from .errors import ConfigError
from .ops_decoder import _elsewhere
from .ops_gemm import _check, _done, _on_gpu

_FLOATS = (torch.float32, torch.float16, torch.bfloat16)


def _setting(name: str, x: float | int | torch.Tensor | None, none: float | int, b: int, dtype: torch.dtype) -> tuple[torch.Tensor | None, float | int]:
    """A setting as a tensor of the rows, or as one number for all."""
    if x is None:
        return None, none
    if not isinstance(x, torch.Tensor):
        return None, x
    if x.shape != (b,) or x.dtype is not dtype:
        raise ConfigError(f"sample_tokens: {name} must be a number or a {dtype} tensor of [{b}]")
    return (x if x.is_contiguous() else x.contiguous()), none


def sample_tokens(logits: torch.Tensor, uniform: torch.Tensor, *, temperature: float | torch.Tensor = 1.0,
                  top_k: int | torch.Tensor | None = None, top_p: float | torch.Tensor | None = None,
                  min_p: float | torch.Tensor | None = None,
                  return_logprobs: bool = False) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """A token for each row of ``logits [B, V]`` (fp32, fp16 or bf16) by the random numbers ``uniform`` (fp32 ``[B]``, in [0, 1)): int64
    ``[B]``, with ``return_logprobs`` also the logarithm of ``softmax(logits)`` at it (fp32 ``[B]``; of all tokens, at temperature 1).

    Settings are numbers, or tensors of a number for each row (fp32, ``top_k`` int32).  A row's tokens weigh
    ``exp(logit / temperature)``.  Kept are the ``top_k`` tokens of the largest logits (equal ones by their index; 0 or None: all), of
    these the fewest most probable ones that have ``top_p`` of their weight (1 or None: all; 0: one), and of these the ones that
    weigh ``min_p`` times the most probable one at least.  The token is the first, by index, at which the kept ones' weights
    sum up to more than ``uniform`` times their total.  Temperature 0 gives the first of the largest logits.

    Logits of -inf (or NaN) are masked: a row of nothing else gives token -1 (logprob -inf).  Weights are fp64 and summed exactly
    in units of 2^-46 of the largest (past 2^16 tokens twice that, past 2^17 four times, and so on): the same inputs give the same
    tokens whatever else runs, and a token of less than half a unit is not drawn.  Up to 65535 rows a call.  A row with a logit of +inf draws among such (its logprob is NaN).
    """
    op = "sample_tokens"
    _on_gpu(logits, op)
    if logits.dim() != 2 or logits.dtype not in _FLOATS or logits.shape[1] == 0:
        raise ConfigError(f"{op}: logits must be an fp32, fp16 or bf16 tensor of [rows, tokens]")
    b, v = logits.shape
    if uniform.shape != (b,) or uniform.dtype is not torch.float32:
        raise ConfigError(f"{op}: uniform must be fp32 [{b}]")
    t, t_all = _setting("temperature", temperature, 1.0, b, torch.float32)
    k, k_all = _setting("top_k", top_k, 0, b, torch.int32)
    p, p_all = _setting("top_p", top_p, 1.0, b, torch.float32)
    m, m_all = _setting("min_p", min_p, 0.0, b, torch.float32)
    if not t_all >= 0 or k_all < 0 or not p_all >= 0 or not m_all >= 0:
        raise ConfigError(f"{op}: temperature, top_k, top_p and min_p must not be negative")
    _elsewhere(op, logits, uniform, t, k, p, m)
    ld, column = logits.stride()
    if column != 1 and v > 1:
        logits, ld = logits.contiguous(), v
    elif ld < 0 or b <= 1:
        ld = v
    if not uniform.is_contiguous():
        uniform = uniform.contiguous()
    token = logits.new_empty((b,), dtype=torch.int64)
    logprob = logits.new_empty((b,), dtype=torch.float32) if return_logprobs else None
    if b:
        need = _workspace(logits.get_device(), b, v)
        ws = logits.new_empty((need,), dtype=torch.uint8)
        status = _lib.lib().fg_sample_tokens(
            logits.data_ptr(), ld, _lib.DTYPE_CODE[logits.dtype], uniform.data_ptr(), _lib.ptr(t), t_all, _lib.ptr(k), min(k_all, 2 ** 31 - 1),
            _lib.ptr(p), p_all, _lib.ptr(m), m_all, token.data_ptr(), _lib.ptr(logprob), b, v, ws.data_ptr(), need, _lib.stream_of(logits))
        if status:
            _check(status, "fg_sample_tokens")
    _done(op)
    return (token, logprob) if return_logprobs else token


@functools.lru_cache(maxsize=256)
def _workspace(_device: int, b: int, v: int) -> int:
    """Bytes of a call's histograms and lists, which follow from its sizes (and the GPU's CUs) alone."""
    return _lib.lib().fg_sample_workspace_bytes(b, v)
