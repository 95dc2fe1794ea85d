"""Attention over a K / V cache in one pass: a sliding window with first tokens that stay visible, and a shared prefix.

The patched attention of the reference multiplies, normalises and multiplies again (``manual_sdpa``, src/module.py:93-117),
which the quantised attention probabilities need; ``QLlamaAttention`` does the same with ``softmax_quantize``.  Where the
probabilities are not quantised, and for the tokens of a decode step, the functions here read queries, keys and values once
and write the output: no score leaves the chip.  They read the cache as ``write_k_cache`` / ``write_v_cache`` leave it
(``[B, Hkv, S, D]``) and give the rows that the output projection reads (``[B, L, H, D]``).
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional

import torch

from . import _lib
from .quantizer import _dtype_code, _ptr, _stream_ptr
from .rotary import _check_devices, _check_no_gradient, _check_out, _strides, _TYPES


def _ready(t: torch.Tensor) -> torch.Tensor:
    """The tensor as the kernels read it: last axis dense, 16-byte aligned rows, every token a row of its own; a copy where it
    is not."""
    ok = (t.shape[-1] == 1 or t.stride(-1) == 1) and t.data_ptr() % 16 == 0 and all(s % 8 == 0 for s in _strides(t, 0)) and \
        (t.shape[-2] <= 1 or t.stride(-2) > 0)
    return t if ok else t.clone(memory_format=torch.contiguous_format)


def _counts(name: str, t: Optional[torch.Tensor], B: int) -> Optional[torch.Tensor]:
    if t is None:
        return None
    if t.dtype not in (torch.int32, torch.int64) or tuple(t.shape) != (B,):
        raise ValueError(f"{name} must be int32 or int64 [{B}]; got {t.dtype} {tuple(t.shape)}")
    return t


def _run(what: str, q, k, v, prefix_k, prefix_v, window: int, sinks: int, scale: Optional[float], lengths, starts, out) -> torch.Tensor:
    if scale is None:
        scale = 1.0 / math.sqrt(q.shape[-1]) if q.dim() == 4 and q.shape[-1] else 1.0
    if out is None and q.is_cuda and window >= 0 and sinks >= 0 and scale > 0 and math.isfinite(scale):
        y = _lib.host().attention(q, k, v, prefix_k, prefix_v, window, sinks, scale, lengths, starts)
        if isinstance(y, torch.Tensor):
            return y
        if y is not None and y not in (_lib.ERR_ALIGN, _lib.ERR_UNSUPPORTED):
            _lib.check(y, what)
    if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape or k.shape[0] != q.shape[0] or k.shape[3] != q.shape[3]:
        raise ValueError(f"{what}: q must be [B, L, H, D], k and v [B, Hkv, S, D]; got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    if q.dtype not in _TYPES or k.dtype != q.dtype or v.dtype != q.dtype:
        raise NotImplementedError(f"{what}: q, k and v must all be fp16 or all bf16; got {q.dtype}, {k.dtype}, {v.dtype}")
    B, L, H, D = q.shape
    Hkv, S = k.shape[1], k.shape[2]
    if Hkv == 0 or H % Hkv:
        raise ValueError(f"{what}: {H} query heads are not a multiple of {Hkv} key heads")
    if D % 8 or not 8 <= D <= 128:
        raise NotImplementedError(f"{what}: head lengths are multiples of 8 up to 128; got {D}")
    P = 0
    if prefix_k is not None:
        if prefix_k.dim() != 3 or prefix_k.shape != prefix_v.shape or prefix_k.shape[0] != Hkv or prefix_k.shape[2] != D:
            raise ValueError(f"{what}: k_prefix and v_prefix must be [{Hkv}, P, {D}]; got {tuple(prefix_k.shape)} and {tuple(prefix_v.shape)}")
        if prefix_k.dtype != q.dtype or prefix_v.dtype != q.dtype:
            raise NotImplementedError(f"{what}: the prefix must have q's type")
        P = prefix_k.shape[1]
    if window < 0 or sinks < 0:
        raise ValueError(f"{what}: window and sinks are counts of tokens; got {window} and {sinks}")
    if not (scale > 0 and math.isfinite(scale)):
        raise ValueError(f"{what}: scale must be positive and finite; got {scale}")
    lengths, starts = _counts("lengths", lengths, B), _counts("starts", starts, B)
    if out is not None:
        _check_out("out", out, q, q.shape)
        if out.numel() and any(t is not None and t.numel() and t.data_ptr() == out.data_ptr() for t in (q, k, v, prefix_k, prefix_v)):
            raise ValueError(f"{what}: out must not be an input")
    _check_no_gradient(what, q, k, v, prefix_k, prefix_v, out)
    _check_devices(what, q, k, v, prefix_k, prefix_v, lengths, starts, out)
    if out is None:
        out = torch.empty((B, L, H, D), dtype=q.dtype, device=q.device)
    if out.numel() == 0:
        return out
    # (a length or start beyond 32 bits is beyond every cache: the nearest value means the same)
    lengths, starts = (t if t is None else (t.clamp(-2 ** 31, 2 ** 31 - 1) if t.dtype == torch.int64 else t).to(torch.int32).contiguous()
                       for t in (lengths, starts))
    q, k, v, prefix_k, prefix_v = (t if t is None else _ready(t) for t in (q, k, v, prefix_k, prefix_v))
    i3, i2 = ctypes.c_int64 * 3, ctypes.c_int64 * 2
    a = _lib.Attention(_ptr(q), _ptr(k), _ptr(v), _ptr(out), B, L, H, Hkv, S, D, i3(*_strides(q, 3)), i3(*_strides(k, 3)), i3(*_strides(v, 3)),
                       i3(*_strides(out, 3)), _ptr(lengths), _ptr(starts), _ptr(prefix_k), _ptr(prefix_v), P,
                       i2(*(_strides(prefix_k, 2) if P else (0, 0))), i2(*(_strides(prefix_v, 2) if P else (0, 0))), window, sinks, scale, _dtype_code(q))
    lib = _lib.lib()
    with _lib.device_guard(q.device):
        n = int(lib.hbq_attention_workspace_bytes(ctypes.byref(a)))
        ws = torch.empty(n, dtype=torch.uint8, device=q.device) if n > 0 else None
        _lib.check(lib.hbq_attention_run(ctypes.byref(a), _ptr(ws), n, _stream_ptr(q.device)), what)
    return out


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: int = 0, sinks: int = 0, scale: Optional[float] = None,
                     lengths: Optional[torch.Tensor] = None, starts: Optional[torch.Tensor] = None,
                     out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention of the newest tokens over a cache, with a sliding window and visible first tokens.

    ``q`` ``[B, L, H, D]``, ``k`` and ``v`` ``[B, Hkv, S, D]`` (fp16 or bf16, ``H`` a multiple of ``Hkv``, ``D`` a multiple of 8 up to
    128, any strides) -> ``[B, L, H, D]``.  Sequence b has ``lengths[b]`` keys (all ``S`` without ``lengths``) and its row i stands at
    position ``starts[b] + i`` (without ``starts``: its rows are its last L tokens, ``lengths[b] - L + i``).  A row at position p sees
    the keys up to p that are among the last ``window`` ones, itself included, or among the first ``sinks`` of the sequence;
    ``window=0``: all of them.  A row that sees nothing (p below 0), and a row behind its sequence's end (p >= ``lengths[b]``, the
    padding of a batch of prompts), is 0.  What the cache holds behind a sequence's end, or where a row's mask hides it, does
    not matter, infinities and NaNs among it; an infinity that a row sees reaches its result however small its weight.  Scores, softmax and
    sums are held in 32 bits.  Where the tensor-core kernel takes the call (many rows) each weight is rounded to the tensors' type before
    its product, and the result's error is 1.2 to 1.4 times that of its own rounding.  ``L = 1`` is a decode step.  ``scale`` defaults to ``1 / sqrt(D)``.  The result may be given as
    ``out``, of any strides with a dense last axis, which overlaps no input."""
    # (a count beyond any cache, held to 64 bits)
    return _run("window_attention", q, k, v, None, None, min(int(window), 2 ** 62), min(int(sinks), 2 ** 62), scale, lengths, starts, out)


def shared_prefix_attention(q: torch.Tensor, k_prefix: torch.Tensor, v_prefix: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                            scale: Optional[float] = None, lengths: Optional[torch.Tensor] = None,
                            starts: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of a batch whose sequences all begin with the same tokens, read once for all of them.

    ``k_prefix`` and ``v_prefix`` ``[Hkv, P, D]`` are the keys and values of the shared beginning; ``q``, ``k``, ``v``, ``lengths`` and
    ``starts`` are those of ``window_attention`` for what each sequence has of its own, counted from the end of the prefix.  A row
    sees the whole prefix and its sequence's own keys up to its position; with no own key yet (p below 0) the prefix alone;
    rows behind their sequence's end are 0.  Weights are held as ``window_attention``'s, those of the prefix in the tensors' type
    but for calls of a few rows and keys."""
    if k_prefix is None or v_prefix is None:
        raise ValueError("shared_prefix_attention needs the prefix; window_attention is the operator without one")
    return _run("shared_prefix_attention", q, k, v, k_prefix, v_prefix, 0, 0, scale, lengths, starts, out)
