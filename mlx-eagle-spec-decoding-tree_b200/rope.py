"""Tree-position RoPE operator with the reference's call signature.

``rope_positions(inp, offsets, inv_freqs, scaling_factor)`` follows
``mlx_arrayed_rope_kernel.py:46-152``: ``inp`` is ``(B, H, L, D)``, ``offsets`` holds
one integer position per (batch, token), ``inv_freqs`` is ``(D/2,)`` fp32; layout is
non-traditional (element i pairs with i + D/2), math in fp32, output in the input
dtype.  Inside the decode loop the same rotation runs fused with the KV-cache
append (``b200_rope_kv_append``); this stand-alone form is the drop-in operator.

``rotate`` is the general form: either order of the pairs, part of the head, 16- and 32-bit types, strided rows, angles that keep
fp32's precision at far positions, and the inverse.  ``frequencies`` gives its frequencies for plain models and for ones stretched to longer contexts.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional, Tuple

import torch

from . import _lib


def rope_positions(inp: torch.Tensor, offsets: torch.Tensor, inv_freqs: torch.Tensor, scaling_factor: float = 1.0,
                   verbose: bool = False) -> torch.Tensor:
    out = _lib.ops().rope_positions(inp, offsets, inv_freqs, scaling_factor)
    if out is not None:
        return out
    _lib.require_cuda(inp, offsets, inv_freqs)
    if inp.dtype != torch.float16 or inp.dim() != 4:
        raise _lib.B200Error("rope_positions expects a float16 (B, H, L, D) tensor")
    B, H, L, D = inp.shape
    if offsets.numel() != B * L or inv_freqs.numel() != D // 2:
        raise _lib.B200Error("offsets must be (B, L) and inv_freqs (D/2,)")
    x = inp.contiguous()
    out = torch.empty_like(x)
    rc = _lib.lib().b200_rope_positions(_lib.ptr(x), _lib.ptr(offsets.to(torch.int32).contiguous()),
                                        _lib.ptr(inv_freqs.float().contiguous()), float(scaling_factor),
                                        _lib.ptr(out), B, H, L, D, _lib.stream_ptr(inp.device))
    _lib.check(rc, "b200_rope_positions")
    return out


def frequencies(rotary_dim: int, base: float = 10000.0, rope_scaling: Optional[dict] = None, device=None) -> Tuple[torch.Tensor, float, float]:
    """``(inv_freqs, scaling_factor, magnitude)`` for :func:`rotate` and ``paged.append``: ``base ** (-2 i / rotary_dim)`` in fp32, rescaled as a
    model's ``rope_scaling`` dict says (``type`` or ``rope_type``):

    ``default``  as they are;
    ``linear``   positions divided by ``factor``;
    ``llama3``   frequencies that turn less than ``low_freq_factor`` times in ``original_max_position_embeddings`` rows divided by ``factor``, those
                 that turn more than ``high_freq_factor`` times kept, linear in the number of turns between;
    ``yarn``     the same with ``beta_slow`` (1) and ``beta_fast`` (32) turns, linear in the pair's index between the pairs that turn so often
                 (rounded outwards), and a magnitude of ``attention_factor`` or ``1 + 0.1 ln(factor)`` on rotated queries and keys.
    """
    if rotary_dim < 2 or rotary_dim % 2 or not base > 0.0:
        raise _lib.B200Error("rotary_dim must be even and positive, base positive")
    f = float(base) ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim)
    rs = rope_scaling or {}
    kind = rs.get("type") or rs.get("rope_type", "default")
    scaling = magnitude = 1.0
    needs = dict(linear=("factor",), llama3=("factor",), yarn=("factor", "original_max_position_embeddings")).get(kind, ())
    if any(not float(rs.get(n) or 0.0) > 0.0 for n in needs):
        raise _lib.B200Error(f"rope_scaling of type {kind} needs {' and '.join(needs)}, positive")
    if kind == "linear":
        scaling = 1.0 / float(rs["factor"])
    elif kind == "llama3":
        lo, hi = float(rs.get("low_freq_factor", 1.0)), float(rs.get("high_freq_factor", 4.0))
        if not hi > lo:
            raise _lib.B200Error("high_freq_factor must be more than low_freq_factor")
        turns = float(rs.get("original_max_position_embeddings", 8192)) * f / (2 * math.pi)
        keep = ((turns - lo) / (hi - lo)).clamp(0.0, 1.0)
        f = f * (keep + (1.0 - keep) / float(rs["factor"]))
    elif kind == "yarn":
        if not base > 1.0 or any(rs.get(n) is not None for n in ("mscale", "mscale_all_dim")) or not rs.get("truncate", True):
            raise _lib.B200Error("yarn takes a base above 1, its magnitude by attention_factor, not mscale, and borders rounded outwards")
        factor, length = float(rs["factor"]), float(rs["original_max_position_embeddings"])

        def index(turns):                                 # of the pair that turns so often (not whole)
            return rotary_dim * math.log(length / (2 * math.pi * turns)) / (2 * math.log(base))

        lo = max(math.floor(index(float(rs.get("beta_fast", 32.0)))), 0)
        hi = min(math.ceil(index(float(rs.get("beta_slow", 1.0)))), rotary_dim - 1)
        stretch = ((torch.arange(rotary_dim // 2, dtype=torch.float64) - lo) / max(hi - lo, 1e-3)).clamp(0.0, 1.0)
        f = f * (1.0 - stretch + stretch / factor)
        magnitude = float(rs["attention_factor"]) if rs.get("attention_factor") is not None else (1.0 + 0.1 * math.log(factor) if factor > 1.0 else 1.0)
    elif kind != "default":
        raise _lib.B200Error("rope_scaling type must be default, linear, llama3 or yarn")
    return f.float().to(device), scaling, magnitude


def _rotary(positions, inv_freqs, dim, tokens, like, scaling_factor, magnitude, interleaved, inverse=False) -> _lib.Rotary:
    """The descriptor of a rotation, its tensors looked over."""
    _lib.require_tensor("inv_freqs", inv_freqs, (torch.float32,), (None,), like)
    if not 2 <= 2 * inv_freqs.numel() <= dim:
        raise _lib.B200Error(f"inv_freqs must hold 1 to {dim // 2} frequencies for a head of {dim}, not {inv_freqs.numel()}")
    if positions is not None:
        _lib.require_tensor("positions", positions, (torch.int32, torch.int64), (tokens,), like)
    return _lib.Rotary(_lib.ptr(positions), _lib.ptr(inv_freqs), float(scaling_factor), float(magnitude),
                       int(positions is not None and positions.dtype == torch.int64), 2 * inv_freqs.numel(), int(bool(interleaved)), int(bool(inverse)))


def rotate(x: torch.Tensor, positions: torch.Tensor, inv_freqs: torch.Tensor, *, scaling_factor: float = 1.0, magnitude: float = 1.0,
           interleaved: bool = False, inverse: bool = False, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x (tokens, heads, dim)`` rotated by ``positions (tokens,)`` times ``scaling_factor * inv_freqs``: the pairs ``(x[i], x[i + R/2])``, or
    ``interleaved`` ``(x[2i], x[2i + 1])``, of the first ``R = 2 * len(inv_freqs)`` dims become ``magnitude * (a cos - b sin, a sin + b cos)``; the rest
    passes through.  float16, bfloat16 or float32, fp32 inside, rounded once; tokens and heads may be strided (a slice of a fused
    projection).  Positions are int32 or int64; an angle is off by less than 2^-23 radians up to 2^37 rows, and by twice that a doubling beyond.

    ``inverse`` rotates by the negative angle: the gradient of a rotation with respect to ``x`` is the rotation of the result's gradient
    with ``inverse`` and the same magnitude.  ``out`` may be ``x`` itself; other overlaps are undefined.  No gradient is recorded."""
    if out is None:
        y = _lib.ops().rotate(x, positions, inv_freqs, scaling_factor, magnitude, interleaved, inverse)
        if y is not None:
            return y
    _lib.require_tensor("x", x, tuple(_lib.DTYPES), (None, None, None), packed=False)
    tokens, heads, dim = x.shape
    if dim > 2048 or heads > 65535 or tokens > 0x7fffffff:
        raise _lib.B200Error("rotate takes heads of at most 2048 dims, at most 65535 of them, and at most 2^31 - 1 tokens")
    if positions is None:
        raise _lib.B200Error("rotate needs positions")
    r = _rotary(positions, inv_freqs, dim, tokens, x, scaling_factor, magnitude, interleaved, inverse)
    if out is None:
        out = torch.empty(tokens, heads, dim, dtype=x.dtype, device=x.device)
    else:
        _lib.require_tensor("out", out, (x.dtype,), x.shape, x, packed=False)
        _lib.require_writable("out", out)
    with _lib.on_device(x):
        rc = _lib.lib().b200_rotate(ctypes.byref(r), _lib.ptr(x), x.stride(0), x.stride(1), _lib.ptr(out), out.stride(0), out.stride(1),
                                    _lib.DTYPES[x.dtype], tokens, heads, dim, _lib.stream_ptr(x.device))
    _lib.check(rc, "b200_rotate")
    return out
