"""Rotary positions: pairs of a head's elements turned by an angle that grows with
the token's position.

``rotate_positions`` turns the queries and keys of packed prompts before
``prompt_attention``; ``append_tokens`` does the same on the way into the pages
of a cache.  The plan that a program keeps is one tensor of frequencies
(``rotary_frequencies``).

Inference only: no gradient is recorded.  The sm_100a kernel lives in
``csrc/rotary.cu``; CPU tensors raise.
"""
from __future__ import annotations

import math

import torch

from . import _lib
from .prompt_attention import _rows

_pack = _lib.words_of("grs_rotate_positions").pack
_entry = None


def rotary_frequencies(
    rotated: int,
    *,
    base: float = 10000.0,
    stretch: float = 1.0,
    trained: int | None = None,
    keep: tuple[float, float] = (1.0, 4.0),
    device="cuda",
) -> torch.Tensor:
    """Radians per position of each pair of a head's first ``rotated`` elements,
    fp64 [rotated // 2] on ``device``: ``base ** (-2 i / rotated)``.

    ``stretch`` > 1 scales them for contexts that many times longer than the
    model was trained on.  Without ``trained`` every frequency is divided by it.
    With ``trained``, the positions of a training context, pairs that turn at
    most ``keep[0]`` times within it are divided, pairs that turn ``keep[1]``
    times or more are kept, and those between are mixed in proportion.  (A
    larger ``base`` is a third way; a model that also lengthens its queries and
    keys gives ``magnitude`` to the calls.)
    """
    if rotated < 2 or rotated % 2:
        raise ValueError("rotated must be even and positive")
    if not (base > 0 and math.isfinite(base) and stretch > 0 and math.isfinite(stretch)):
        raise ValueError("base and stretch must be positive")
    f = base ** (-torch.arange(rotated // 2, dtype=torch.float64) * 2 / rotated)
    if trained is None:
        f = f / stretch
    else:
        low, high = keep
        if trained <= 0 or not high > low:
            raise ValueError("trained must be positive, keep an ascending pair")
        kept = ((trained * f / (2 * math.pi) - low) / (high - low)).clamp(0.0, 1.0)
        f = f * (kept + (1.0 - kept) / stretch)
    return f.to(device)


def _frequencies(frequencies: torch.Tensor, device: int, width: int) -> int:
    """Number of pairs of a frequency tensor that fits heads of this width."""
    if (frequencies.dtype is not torch.float64 or frequencies.dim() != 1
            or not frequencies.is_contiguous() or frequencies.get_device() != device):
        _lib.require_cuda(frequencies)
        raise ValueError("frequencies must be contiguous fp64 [pairs] on the inputs' device")
    pairs = frequencies.numel()
    if 2 * pairs > width:
        raise ValueError("more pairs than the heads hold")
    return pairs


def _positions(positions: torch.Tensor, device: int, tokens: int) -> int:
    """1 for int64 positions, 0 for int32."""
    if (positions.dtype not in (torch.int32, torch.int64) or positions.shape != (tokens,)
            or not positions.is_contiguous() or positions.get_device() != device):
        _lib.require_cuda(positions)
        raise ValueError("positions must be contiguous int32 or int64 [tokens]")
    return int(positions.dtype is torch.int64)


def _turned_out(name: str, out: torch.Tensor | None, like: torch.Tensor, device: int,
                dtype: torch.dtype, stride: tuple, *others: torch.Tensor | None):
    """An output of like's shape (a new one, like itself, or one that is none of
    the others) and its strides."""
    if out is None:
        out = torch.empty_like(like)          # half the time of asking for the format
        step = out.stride()
        if step[0] < step[1]:
            out = torch.empty_like(like, memory_format=torch.contiguous_format)
            step = out.stride()
        return out, step
    step = _rows(name, out, device, dtype, like.shape)
    need = 1
    for size, s in sorted(zip(like.shape, step), key=lambda p: p[1]):
        if size > 1 and s < need:
            raise ValueError(f"{name} must not overlap itself")
        need = max(need, s * size)
    at = out.data_ptr()
    if out.numel():
        if at == like.data_ptr() and any(
                a != b for a, b, n in zip(step, stride, like.shape) if n > 1):
            raise ValueError(f"{name} must be the input itself or not overlap it")
        if any(t is not None and t.data_ptr() == at for t in others):
            raise ValueError(f"{name} must not be another input")
    return out, step


def _check_magnitude(magnitude: float) -> float:
    magnitude = float(magnitude)
    if not abs(magnitude) <= 3.4e38:          # NaN too
        raise ValueError("magnitude must be finite in fp32")
    return magnitude


def rotate_positions(
    query: torch.Tensor,
    key: torch.Tensor | None,
    positions: torch.Tensor,
    frequencies: torch.Tensor,
    *,
    interleaved: bool = False,
    magnitude: float = 1.0,
    query_out: torch.Tensor | None = None,
    key_out: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor | None]:
    """Query [T, H, D] and key [T, Hkv, D] (or None) turned by their tokens'
    positions, int32 or int64 [T] (any value; a negative one turns back).

    bf16 or fp32, D <= 256 and contiguous, any other strides.  frequencies fp64
    [R / 2], R <= D even, radians per position: pair i is elements i and
    i + R / 2 of a head, or 2 i and 2 i + 1 when ``interleaved``; (a, b) becomes
    ``magnitude * (a cos - b sin, a sin + b cos)``.  Elements from R on are
    copied.  Angles are exact modulo whole turns at any position; the rest is
    fp32, rounded once.

    Outputs are new, or the given ones: the inputs themselves (in place) or
    memory that overlaps neither.  The call does not synchronise and can be
    captured into a CUDA graph.
    """
    global _entry
    device = query.get_device()
    if device < 0:
        _lib.require_cuda(query)
    place = _lib.elsewhere(device)
    if place is not None:
        with place:
            return rotate_positions(query, key, positions, frequencies, interleaved=interleaved,
                                    magnitude=magnitude, query_out=query_out, key_out=key_out)
    shape, dtype = query.shape, query.dtype
    keys = None if key is None else key.shape
    if len(shape) != 3 or (key is not None and len(keys) != 3):
        raise ValueError("query must be [tokens, heads, D], key [tokens, kv_heads, D]")
    tokens, heads, width = shape
    code = _lib.DTYPE_CODES.get(dtype)
    if code is None:
        raise ValueError("rotation takes bf16 or fp32")
    if not 1 <= width <= 256:
        raise ValueError("head widths from 1 to 256 are supported")
    if tokens >= 1 << 30 or not 0 < heads < 1 << 30:
        raise ValueError("at most 2^30 tokens and heads, and one head at least")
    q = query.stride()
    if q[2] != 1 and width > 1:
        raise ValueError("query needs a contiguous head width")
    k, kv_heads = (0, 0), 0
    if key is not None:
        kv_heads = keys[1]
        if not 0 < kv_heads < 1 << 30:
            raise ValueError("at most 2^30 heads, and one at least")
        k = _rows("key", key, device, dtype, (tokens, kv_heads, width))
    elif key_out is not None:
        raise ValueError("key_out comes with a key")
    wide = _positions(positions, device, tokens)
    pairs = _frequencies(frequencies, device, width)
    magnitude = _check_magnitude(magnitude)
    query_out, qo = _turned_out("query_out", query_out, query, device, dtype, q, key)
    key_at = key_to = 0
    ko = (0, 0)
    if key is not None:
        key_out, ko = _turned_out("key_out", key_out, key, device, dtype, k, query, query_out)
        key_at, key_to = key.data_ptr(), key_out.data_ptr()
    if not tokens:
        return query_out, key_out
    if not pairs:
        raise ValueError("no frequencies")
    if _entry is None:
        _entry = _lib.words_entry("grs_rotate_positions")
    status = _entry(_pack(
        code, query.data_ptr(), q[0], q[1], key_at, k[0], k[1], positions.data_ptr(), wide,
        frequencies.data_ptr(), pairs, bool(interleaved), magnitude, query_out.data_ptr(), qo[0],
        qo[1], key_to, ko[0], ko[1], tokens, heads, kv_heads, width, _lib.stream_on(device)))
    if status:
        _lib.check(status, "rotate_positions")
    return query_out, key_out
