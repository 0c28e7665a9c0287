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
from .paged_attention import _STATUS, _status_word

_pack = _lib.words_of("grs_prompt_attention").pack
_entry = None
_STATUS_AT: dict[int, int] = {}          # device index -> address of its status word
_LARGEST_SCALE = 3.4e38 / math.log2(math.e)


def _status_for(query: torch.Tensor, device: int, status: torch.Tensor | None) -> int:
    """Address of the caller's status word, or of the device's
    (``check_decode_status``)."""
    if status is not None:
        if (status.dtype is not torch.int32 or status.numel() != 1
                or status.get_device() != device):
            _lib.require_cuda(status)
            raise ValueError("status must be one int32 on the query's device")
        return status.data_ptr()
    word = _STATUS.get(query.device)
    if word is None:
        # made under capture it would live in that graph's memory
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("make one call before capturing the first, or pass status=")
        word = _status_word(query.device)
    _STATUS_AT[device] = word.data_ptr()     # the word lives as long as the process
    return _STATUS_AT[device]


def _refuse(name: str, t: torch.Tensor, device: int, dtype: torch.dtype, shape: tuple) -> None:
    _lib.require_cuda(t)
    if t.get_device() != device or t.dtype is not dtype:
        raise ValueError(f"{name} must have the query's device and dtype")
    if t.shape != shape:
        raise ValueError(f"{name} must be {list(shape)}, not {list(t.shape)}")
    raise ValueError(f"{name} needs a contiguous head width")


def _rows(name: str, t: torch.Tensor, device: int, dtype: torch.dtype, shape: tuple) -> tuple:
    """Strides of t, rows of the query's device and dtype and the given shape
    with a contiguous last dimension."""
    stride = t.stride()
    if (t.get_device() != device or t.dtype is not dtype or t.shape != shape
            or (stride[-1] != 1 and shape[-1] > 1)):
        _refuse(name, t, device, dtype, shape)
    return stride


def _out_rows(out: torch.Tensor, device: int, dtype: torch.dtype, shape: tuple,
              *inputs: torch.Tensor | None) -> tuple:
    stride = _rows("out", out, device, dtype, shape)
    need = 1
    for size, step in sorted(zip(shape, stride), key=lambda p: p[1]):
        if size > 1 and step < need:
            raise ValueError("out must not overlap itself")
        need = max(need, step * size)
    at = out.data_ptr()
    if out.numel() and any(t is not None and t.data_ptr() == at for t in inputs):
        raise ValueError("out must not be one of the inputs")
    return stride


def _check_heads(query: torch.Tensor, heads: int, kv_heads: int, width: int) -> int:
    """Type code of a query whose heads and width are supported."""
    code = _lib.DTYPE_CODES.get(query.dtype)
    if code is None:
        raise ValueError("attention takes bf16 or fp32 queries")
    if not 1 <= width <= 256:
        raise ValueError("head widths from 1 to 256 are supported")
    if not kv_heads or not heads or heads % kv_heads:
        raise ValueError("query heads must be a multiple of the key/value heads")
    if heads >= 1 << 30:
        raise ValueError("at most 2^30 heads")
    return code


def _check_scale(scale: float | None, width: int) -> float:
    scale = 1.0 / math.sqrt(width) if scale is None else float(scale)
    if not abs(scale) <= _LARGEST_SCALE:      # NaN too
        raise ValueError("scale * log2(e) must be finite in fp32")
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
    global _entry
    device = query.get_device()
    if device < 0:
        _lib.require_cuda(query)
    place = _lib.elsewhere(device)
    if place is not None:
        with place:
            return prompt_attention(query, key, value, offsets, scale=scale, out=out,
                                    status=status)
    if query.dim() != 3 or key.dim() != 3:
        raise ValueError("query must be [tokens, heads, D], key and value [tokens, kv_heads, D]")
    shape = query.shape
    tokens, heads, width = shape
    kv_heads = key.shape[1]
    if tokens >= 1 << 30:
        raise ValueError("at most 2^30 tokens")
    code, dtype = _check_heads(query, heads, kv_heads, width), query.dtype
    q = query.stride()
    if q[2] != 1 and width > 1:
        raise ValueError("query needs a contiguous head width")
    k = _rows("key", key, device, dtype, (tokens, kv_heads, width))
    v = _rows("value", value, device, dtype, (tokens, kv_heads, width))
    if (offsets.dtype is not torch.int32 or offsets.dim() != 1 or not offsets.numel()
            or not offsets.is_contiguous() or offsets.get_device() != device):
        _lib.require_cuda(offsets)
        raise ValueError("offsets must be a contiguous int32 [sequences + 1] on the query's device")
    if offsets.numel() > 1 << 30:
        raise ValueError("at most 2^30 offsets")
    scale = _check_scale(scale, width)
    fresh = out is None
    if fresh:
        out = torch.empty_like(query, memory_format=torch.contiguous_format)
        o = (heads * width, width)
    else:
        o = _out_rows(out, device, dtype, shape, query, key, value)
    if not tokens:
        return out
    word = None if status is not None else _STATUS_AT.get(device)
    if word is None:
        word = _status_for(query, device, status)
    if _entry is None:
        _entry = _lib.words_entry("grs_prompt_attention")
    code = _entry(_pack(
        code, query.data_ptr(), q[0], q[1], key.data_ptr(), k[0], k[1], value.data_ptr(), v[0],
        v[1], offsets.data_ptr(), offsets.numel() - 1, out.data_ptr(), o[0], o[1], tokens, heads,
        kv_heads, width, scale, fresh, word, _lib.stream_on(device)))
    if code:
        _lib.check(code, "prompt attention")
    return out
