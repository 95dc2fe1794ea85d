"""Rotary positions of projected heads for every layout and scaling, alone or behind a norm of each head.

``kvcache.rope_heads`` and ``write_k_cache`` turn whole heads in the half layout by fp16 tables, as the patched blocks do
(``apply_rotary_pos_emb``, src/module.py:157).  ``rope_rotate`` and ``qk_norm_rope`` take the angles from positions and
frequencies instead, in 64 bits: pairs side by side or half a head apart, the whole head or its first part, positions
anywhere in a long context, frequencies scaled for it (``rope_frequencies``).  The arithmetic is in 32 bits and rounded
once, where the separate ops on fp16 tensors round the table, both products and the sum.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional, Tuple

import torch

from . import _lib
from .quantizer import _dtype_code, _ptr, _stream_ptr

_TYPES = (torch.float16, torch.bfloat16)


def rope_frequencies(rotary_dim: int, theta: float, scaling: Optional[dict] = None, device=None) -> Tuple[torch.Tensor, float]:
    """``(inv_freq, factor)``: the angle per position of each of the ``rotary_dim / 2`` pairs (fp64) and what cosine and sine
    are multiplied by.  ``scaling`` holds a ``"type"`` and its constants, by the names of a model's configuration file:

    ``linear``   ``factor``: every pair turns ``factor`` times slower.
    ``ntk``      ``factor``: a base of ``theta * factor^(r / (r - 2))``, so that only the slowest pair turns that much slower.
    ``llama3``   ``factor``, ``low_freq_factor``, ``high_freq_factor``, ``original_max_position_embeddings``: pairs that turn
                 fewer than ``low`` times over the original context slow down by ``factor``, those that turn more than
                 ``high`` times stay, a ramp in the number of turns lies between.
    ``yarn``     ``factor``, ``beta_fast`` (32), ``beta_slow`` (1), ``original_max_position_embeddings``,
                 ``attention_factor`` (``0.1 ln(factor) + 1``): the ramp runs over the pairs' indices, from the pair that
                 turns ``beta_fast`` times over the original context to the one that turns ``beta_slow`` times.
    """
    r = int(rotary_dim)
    if r < 2 or r % 2:
        raise ValueError(f"rotary_dim must be even and at least 2; got {rotary_dim}")
    if not theta > 0:
        raise ValueError(f"theta must be positive; got {theta}")
    kind = "none" if scaling is None else scaling.get("type", scaling.get("rope_type", "none"))
    scale, multiplier = 1.0, 1.0
    if kind not in ("none", "default"):
        scale = float(scaling["factor"])
        if not scale > 0:
            raise ValueError(f"the scaling factor must be positive; got {scale}")
    if kind == "ntk":
        if r == 2:
            raise ValueError("ntk scaling needs more than one pair")
        theta = theta * scale ** (r / (r - 2))
    f = torch.pow(torch.tensor(float(theta), dtype=torch.float64), -torch.arange(0, r, 2, dtype=torch.float64) / r)
    if kind == "linear":
        f = f / scale
    elif kind == "llama3":
        low, high = float(scaling.get("low_freq_factor", 1.0)), float(scaling.get("high_freq_factor", 4.0))
        if not high > low:
            raise ValueError("high_freq_factor must be larger than low_freq_factor")
        turns = float(scaling["original_max_position_embeddings"]) * f / (2 * math.pi)
        keep = ((turns - low) / (high - low)).clamp(0.0, 1.0)
        f = keep * f + (1 - keep) * f / scale
    elif kind == "yarn":
        context = float(scaling["original_max_position_embeddings"])

        def pair_of(turns: float) -> float:
            return r * math.log(context / (turns * 2 * math.pi)) / (2 * math.log(theta))
        low = max(math.floor(pair_of(float(scaling.get("beta_fast", 32.0)))), 0)
        high = min(math.ceil(pair_of(float(scaling.get("beta_slow", 1.0)))), r - 1)
        keep = 1 - ((torch.arange(r // 2, dtype=torch.float64) - low) / max(high - low, 0.001)).clamp(0.0, 1.0)
        f = keep * f + (1 - keep) * f / scale
        multiplier = scaling.get("attention_factor")
        multiplier = (0.1 * math.log(scale) + 1.0 if scale > 1 else 1.0) if multiplier is None else float(multiplier)
    elif kind not in ("none", "default", "ntk"):
        raise ValueError(f"unknown rotary scaling {kind!r}")
    return f.to(device) if device is not None else f, float(multiplier)


def _check_heads(name: str, x: torch.Tensor) -> None:
    if x.dim() not in (3, 4):
        raise ValueError(f"{name} must be [T, H, D] or [B, T, H, D]; got {tuple(x.shape)}")
    if x.dtype not in _TYPES:
        raise NotImplementedError(f"{name} must be fp16 or bf16; got {x.dtype}")


def _check_no_gradient(what: str, *tensors) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise NotImplementedError(f"{what} records no gradient: call it under torch.no_grad()")


def _check_rotary(x: torch.Tensor, inv_freq: torch.Tensor, positions: torch.Tensor) -> None:
    T, D = x.shape[-3], x.shape[-1]
    if inv_freq.dtype != torch.float64 or inv_freq.dim() != 1 or not 2 <= 2 * inv_freq.numel() <= D:
        raise ValueError(f"inv_freq must be fp64 with one to D / 2 = {D // 2} values; got {inv_freq.dtype} {tuple(inv_freq.shape)}")
    ok = [(T,)] + ([(1, T), (x.shape[0], T)] if x.dim() == 4 else [(1, T)])
    if positions.dtype not in (torch.int32, torch.int64) or tuple(positions.shape) not in ok:
        raise ValueError(f"positions must be int32 or int64, one per token ({ok[0]} or {ok[-1]}); got {positions.dtype} {tuple(positions.shape)}")


def _check_devices(what: str, x: torch.Tensor, *others) -> None:
    if not x.is_cuda:
        raise _lib.HbqError(f"{what} needs CUDA tensors (there is no CPU fallback)")
    if any(t is not None and t.device != x.device for t in others):
        raise ValueError(f"{what}: all tensors must be on {x.device}")


def _check_out(name: str, out: torch.Tensor, x: torch.Tensor, shape) -> None:
    if tuple(out.shape) != tuple(shape) or out.dtype != x.dtype:
        raise ValueError(f"{name} must be {x.dtype} {tuple(shape)}; got {out.dtype} {tuple(out.shape)}")
    if any(s == 0 and n > 1 for s, n in zip(out.stride(), out.shape)) or (out.shape[-1] > 1 and out.stride(-1) != 1):
        raise ValueError(f"{name} must be a tensor of separate elements with a dense last axis")


def _strides(t: torch.Tensor, n: int):
    s = [t.stride(i) if t.shape[i] > 1 else 0 for i in range(t.dim() - 1)]
    return [0] * (n - len(s)) + s


def _heads(x: torch.Tensor, out: torch.Tensor, weight=None) -> _lib.Heads:
    i3 = ctypes.c_int64 * 3
    return _lib.Heads(_ptr(x), _ptr(out), _ptr(weight), x.shape[-2], i3(*_strides(x, 3)), i3(*_strides(out, 3)))


def _rotary(x: torch.Tensor, inv_freq: torch.Tensor, positions: torch.Tensor, interleaved: bool, factor: float) -> _lib.Rotary:
    pb = positions.stride(0) if positions.dim() == 2 and positions.shape[0] > 1 else 0
    return _lib.Rotary(_ptr(inv_freq), _ptr(positions), (ctypes.c_int64 * 2)(pb, positions.stride(-1)), 2 * inv_freq.numel(), int(bool(interleaved)),
                       int(positions.dtype == torch.int64), float(factor))


def _dense(x: torch.Tensor) -> torch.Tensor:
    return x if x.shape[-1] == 1 or x.stride(-1) == 1 else x.contiguous()


def _sizes(x: torch.Tensor):
    return (x.shape[0] if x.dim() == 4 else 1), x.shape[-3], x.shape[-1]


def rope_rotate(x: torch.Tensor, inv_freq: torch.Tensor, positions: torch.Tensor, interleaved: bool = False, factor: float = 1.0,
                out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Turn pair i of every head of ``x`` (``[T, H, D]`` or ``[B, T, H, D]``, any strides with a dense last axis, fp16 or bf16)
    by ``positions * inv_freq[i]``; values behind the first ``2 * inv_freq.numel()`` of a head stay as they are.

    ``inv_freq`` (fp64) and ``factor`` come from ``rope_frequencies``; ``positions`` is int32 or int64, ``[T]`` or ``[B, T]``.
    ``interleaved``: pairs ``(2 i, 2 i + 1)``, else ``(i, i + rotary_dim / 2)``.  ``out``: a tensor of x's shape to write into
    -- ``x`` itself, or one that overlaps nothing of it, a slice of a cache in any layout for instance."""
    if out is None:
        y = _lib.host().rope_rotate(x, inv_freq, positions, interleaved, factor) if x.is_cuda else None
        if isinstance(y, torch.Tensor):
            return y
        if y is not None:
            _lib.check(y, "hbq_rope_rotate")
    _check_heads("x", x)
    _check_rotary(x, inv_freq, positions)
    if out is not None:
        _check_out("out", out, x, x.shape)
    _check_no_gradient("rope_rotate", x, inv_freq, out)
    _check_devices("rope_rotate", x, inv_freq, positions, out)
    xd, f = _dense(x), inv_freq.contiguous()
    if out is None:
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    B, T, D = _sizes(x)
    h, r = _heads(xd, out), _rotary(x, f, positions, interleaved, factor)
    with _lib.device_guard(x.device):
        _lib.check(_lib.lib().hbq_rope_rotate(ctypes.byref(h), ctypes.byref(r), _dtype_code(x), B, T, D, _stream_ptr(x.device)), "hbq_rope_rotate")
    return out


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor, eps: float, inv_freq: torch.Tensor,
                 positions: torch.Tensor, interleaved: bool = False, factor: float = 1.0,
                 out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """``rope_rotate`` of ``x * rsqrt(mean(x^2) + eps) * weight`` over each head of ``q`` and ``k``, both in one launch.

    ``q`` ``[.., T, H, D]`` and ``k`` ``[.., T, Hkv, D]`` may be views of one packed projection; ``q_weight`` / ``k_weight`` are
    ``[D]`` of their type.  ``out``: the pair of tensors to write into, as for ``rope_rotate``."""
    if out is None:
        y = _lib.host().qk_norm_rope(q, k, q_weight, k_weight, eps, inv_freq, positions, interleaved, factor) if q.is_cuda else None
        if isinstance(y, tuple):
            return y
        if y is not None:
            _lib.check(y, "hbq_qk_norm_rope")
    _check_heads("q", q)
    _check_heads("k", k)
    if k.dim() != q.dim() or k.dtype != q.dtype or k.shape[-1] != q.shape[-1] or k.shape[:-2] != q.shape[:-2]:
        raise ValueError(f"q and k must agree in type, tokens and head length; got {q.dtype} {tuple(q.shape)} and {k.dtype} {tuple(k.shape)}")
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w.dtype != q.dtype or tuple(w.shape) != (q.shape[-1],):
            raise ValueError(f"{name} must be {q.dtype} [{q.shape[-1]}]; got {w.dtype} {tuple(w.shape)}")
    _check_rotary(q, inv_freq, positions)
    oq, ok = out if out is not None else (None, None)
    for name, o, x in (("out[0]", oq, q), ("out[1]", ok, k)):
        if o is not None:
            _check_out(name, o, x, x.shape)
    _check_no_gradient("qk_norm_rope", q, k, q_weight, k_weight, inv_freq, oq, ok)
    _check_devices("qk_norm_rope", q, k, q_weight, k_weight, inv_freq, positions, oq, ok)
    qd, kd, f, wq, wk = _dense(q), _dense(k), inv_freq.contiguous(), q_weight.contiguous(), k_weight.contiguous()
    oq = torch.empty(q.shape, dtype=q.dtype, device=q.device) if oq is None else oq
    ok = torch.empty(k.shape, dtype=k.dtype, device=k.device) if ok is None else ok
    B, T, D = _sizes(q)
    hq, hk, r = _heads(qd, oq, wq), _heads(kd, ok, wk), _rotary(q, f, positions, interleaved, factor)
    with _lib.device_guard(q.device):
        _lib.check(_lib.lib().hbq_qk_norm_rope(ctypes.byref(hq), ctypes.byref(hk), ctypes.byref(r), _dtype_code(q), B, T, D, float(eps),
                                               _stream_ptr(q.device)), "hbq_qk_norm_rope")
    return oq, ok
