"""Causal attention over whole prompts: packed sequences, grouped heads.

``paged_attention`` decodes one token at a time; ``prompt_attention`` computes
every row of one or many prompts at once, so a prompt fills its keys and
values in one pass of the model.  The rows of a prompt that a beam search
continues are the prefix of ``shared_prefix_attention``.

Inference only: no gradient is recorded.  The sm_100a kernels live in
``csrc/grouped_attention_tc.cu`` (bf16, tensor cores) and
``csrc/grouped_attention.cu`` (fp32, and bf16 layouts that the tensor-core
kernel does not take); CPU tensors raise.
"""
from __future__ import annotations

import math

import torch

from . import _lib
from .paged_attention import _status_word


def _status_for(device: torch.device, status: torch.Tensor | None) -> torch.Tensor:
    """The caller's status word, or the device's (``check_decode_status``)."""
    if status is not None:
        if status.dtype != torch.int32 or status.numel() != 1 or status.device != device:
            raise ValueError("status must be one int32 on the query's device")
        return status
    return _status_word(device)


def _check_rows(name: str, t: torch.Tensor, like: torch.Tensor, shape: tuple) -> None:
    if t.device != like.device or t.dtype != like.dtype:
        raise ValueError(f"{name} must have the query's device and dtype")
    if tuple(t.shape) != shape:
        raise ValueError(f"{name} must be {list(shape)}, not {list(t.shape)}")
    if t.numel() and t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{name} needs a contiguous head width")


def _check_out(out: torch.Tensor, query: torch.Tensor, *inputs: torch.Tensor) -> None:
    _check_rows("out", out, query, tuple(query.shape))
    need = 1
    for size, stride in sorted(zip(out.shape, out.stride()), key=lambda p: p[1]):
        if size > 1 and stride < need:
            raise ValueError("out must not overlap itself")
        need = max(need, stride * size)
    if out.numel() and any(out.data_ptr() == t.data_ptr() for t in (query, *inputs)):
        raise ValueError("out must not be one of the inputs")


def _check_heads(query: torch.Tensor, kv_heads: int) -> None:
    if query.dtype not in _lib.DTYPE_CODES:
        raise ValueError("attention takes bf16 or fp32 queries")
    heads, width = query.shape[1:]
    if not 1 <= width <= 256:
        raise ValueError("head widths from 1 to 256 are supported")
    if not kv_heads or heads % kv_heads:
        raise ValueError("query heads must be a multiple of the key/value heads")


def _check_scale(scale: float | None, width: int) -> float:
    scale = 1.0 / math.sqrt(width) if scale is None else float(scale)
    if not math.isfinite(scale):
        raise ValueError("scale must be finite")
    return scale


def prompt_attention(
    query: torch.Tensor,
    key: torch.Tensor,
    value: torch.Tensor,
    offsets: torch.Tensor,
    *,
    scale: float | None = None,
    out: torch.Tensor | None = None,
    status: torch.Tensor | None = None,
) -> torch.Tensor:
    """Causal softmax attention of packed sequences.

    query [T, H, D], key and value [T, Hkv, D], bf16 or fp32, D <= 256 and
    contiguous (any other strides: slices of one projection's output are
    fine); query head i reads K/V head ``i // (H // Hkv)``.  offsets int32
    [N + 1], ascending, on the device: sequence j holds the tokens
    ``offsets[j]:offsets[j + 1]`` (possibly none), each of which attends to its
    own sequence up to itself.  ``scale`` defaults to ``1 / sqrt(D)``.

    Rows of tokens that lie in no sequence (behind the last one) are left as
    they were in a given ``out`` and zero in a new one; whatever they hold in
    query, key and value reaches no other row.  ``out`` must not overlap the
    inputs.  The call neither synchronises nor reads ``offsets`` on the host,
    so it can be captured into a CUDA graph.
    """
    _lib.require_cuda(query, key, value, offsets, out, status)
    if query.dim() != 3 or key.dim() != 3:
        raise ValueError("query must be [tokens, heads, D], key and value [tokens, kv_heads, D]")
    tokens, heads, width = query.shape
    kv_heads = key.shape[1]
    _check_heads(query, kv_heads)
    _check_rows("query", query, query, tuple(query.shape))
    _check_rows("key", key, query, (tokens, kv_heads, width))
    _check_rows("value", value, query, (tokens, kv_heads, width))
    if (offsets.dtype != torch.int32 or offsets.dim() != 1 or not offsets.numel()
            or not offsets.is_contiguous() or offsets.device != query.device):
        raise ValueError("offsets must be a contiguous int32 [sequences + 1] on the query's device")
    fresh = out is None
    if fresh:
        out = torch.empty(query.shape, dtype=query.dtype, device=query.device)
    else:
        _check_out(out, query, key, value)
    if not out.numel():
        return out
    scale = _check_scale(scale, width)
    word = _status_for(query.device, status)
    with _lib.on_device(query):
        code = _lib.lib().grs_prompt_attention(
            _lib.DTYPE_CODES[query.dtype], query.data_ptr(), query.stride(0), query.stride(1),
            key.data_ptr(), key.stride(0), key.stride(1), value.data_ptr(), value.stride(0),
            value.stride(1), offsets.data_ptr(), offsets.numel() - 1, out.data_ptr(),
            out.stride(0), out.stride(1), tokens, heads, kv_heads, width,
            scale, int(fresh),
            word.data_ptr(), _lib.stream_of(query))
    _lib.check(code, "prompt attention")
    return out
