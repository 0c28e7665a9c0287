"""Decode attention over a paged cache held in 8 bits.

``paged_attention`` and ``shared_prefix_attention`` read pages of the model's
own type; ``quantized_attention`` reads pages of e4m3 codes with a scale for
each page and head, as ``append_tokens`` writes them: half of bf16's bytes, which
is what bounds a decode step over long contexts.

Inference only: no gradient is recorded.  The sm_100a kernels live in
``csrc/quantized_attention.cu``; CPU tensors raise.
"""
from __future__ import annotations

from functools import lru_cache

import torch

from . import _lib
from .prompt_attention import _STATUS_AT, _check_heads, _check_scale, _out_rows, _status_for

_pack = _lib.words_of("grs_quantized_attention").pack
_entry = None
_E4M3 = torch.float8_e4m3fn


@lru_cache(maxsize=4096)
def _workspace_bytes(*sizes: int) -> int:
    return _lib.lib().grs_quantized_attention_workspace_bytes(*sizes)


def _scales(key_scale: torch.Tensor, value_scale: torch.Tensor, device: int, pages: int,
            kv_heads: int) -> int:
    """Row stride of fp32 key and value scales [pages, kv_heads] of one layout."""
    row = None
    for name, t in (("key_scale", key_scale), ("value_scale", value_scale)):
        stride = t.stride()
        if (t.dtype is not torch.float32 or t.shape != (pages, kv_heads)
                or t.get_device() != device or (stride[1] != 1 and kv_heads > 1)):
            _lib.require_cuda(t)
            raise ValueError(f"{name} must be fp32 [pages, kv_heads] with contiguous rows on the "
                             "inputs' device")
        if row is not None and stride[0] != row and pages > 1:
            raise ValueError("key/value scales must share a layout")
        row = stride[0]
    return row


def _table(name: str, t: torch.Tensor, device: int, rows: int) -> tuple[int, int]:
    """Columns and row stride of an int32 block table."""
    shape, stride = t.shape, t.stride()
    if (t.dtype is not torch.int32 or len(shape) != 2 or shape[0] != rows
            or t.get_device() != device or (stride[1] != 1 and shape[1] > 1)):
        _lib.require_cuda(t)
        raise ValueError(f"{name} must be int32 [sequences, columns] with contiguous rows on the "
                         "inputs' device")
    return shape[1], stride[0]


def _lengths(t: torch.Tensor, device: int, rows: int) -> int:
    if (t.dtype is not torch.int32 or t.shape != (rows,) or not t.is_contiguous()
            or t.get_device() != device):
        _lib.require_cuda(t)
        raise ValueError("lengths must be contiguous int32 [sequences] on the inputs' device")
    return t.data_ptr()


def _cache(key_cache: torch.Tensor, value_cache: torch.Tensor, shape: tuple, device: int,
           dtype: torch.dtype, kv_heads: int, width: int) -> tuple:
    """Strides of a key cache of that shape, [pages, page, kv_heads, D], and a value
    cache of its layout."""
    stride = key_cache.stride()
    if (key_cache.dtype is not dtype or value_cache.dtype is not dtype
            or key_cache.get_device() != device or value_cache.get_device() != device):
        _lib.require_cuda(key_cache, value_cache)
        raise ValueError(f"caches must be {dtype} on the inputs' device")
    if value_cache.shape != shape or shape[2] != kv_heads or shape[3] != width:
        raise ValueError(f"caches must be [pages, page, {kv_heads}, {width}]")
    if stride[3] != 1 and width > 1:
        raise ValueError("caches need a contiguous head width")
    other = value_cache.stride()
    if stride != other and any(a != b for a, b, n in zip(stride, other, shape) if n > 1):
        raise ValueError("key/value caches must share a layout")
    if shape[0] >= 1 << 31 or not 0 < shape[1] < 1 << 30:
        raise ValueError("at most 2^31 pages of 1 to 2^30 tokens")
    return stride


def quantized_attention(
    query: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    key_scale: torch.Tensor,
    value_scale: torch.Tensor,
    block_table: torch.Tensor,
    lengths: torch.Tensor,
    *,
    scale: float | None = None,
    out: torch.Tensor | None = None,
    status: torch.Tensor | None = None,
) -> torch.Tensor:
    """Softmax attention of one query per sequence, query [B, H, D] (bf16 or
    fp32), to the first ``lengths[b]`` tokens of its pages.

    key_cache/value_cache float8_e4m3fn [pages, page, Hkv, D] of one layout,
    D <= 256 and contiguous; key_scale/value_scale fp32 [pages, Hkv], positive
    and finite: a code stands for code * scale.  block_table int32 [B, columns],
    lengths int32 [B].  Query head i reads K/V head ``i // (H // Hkv)``;
    ``scale`` defaults to ``1 / sqrt(D)``.  Rows without any key are zero; what
    pages hold behind a sequence's last token reaches no row.  Several new
    tokens of one sequence are as many rows of an expanded table, each with the
    length up to its own token.

    The products run on the tensor cores with sums and softmax in fp32: weights
    are rounded to f16 for bf16 queries; fp32 queries and weights go in two f16
    parts, 22 bits (errors of 4e-7 to 8e-7 of the norm, up to 5e-6 over 20000
    tokens and more or at width 256).  Tables no wider than the longest sequence
    are fastest where sequences are short: the kernel is chosen by their width.

    Page ids outside the cache are skipped and lengths beyond the table are
    cut; both are recorded in ``status`` (default: the device word that
    ``check_decode_status`` reads).  ``out`` must not overlap the inputs.  The
    call does not synchronise and can be captured into a CUDA graph.
    """
    global _entry
    device = query.get_device()
    if device < 0:
        _lib.require_cuda(query)
    place = _lib.elsewhere(device)
    if place is not None:
        with place:
            return quantized_attention(query, key_cache, value_cache, key_scale, value_scale,
                                       block_table, lengths, scale=scale, out=out, status=status)
    shape, dtype, pool = query.shape, query.dtype, key_cache.shape
    if len(shape) != 3 or len(pool) != 4:
        raise ValueError("query must be [batch, heads, D], caches [pages, page, kv_heads, D]")
    batch, heads, width = shape
    pages, page, kv_heads, _ = pool
    if batch >= 1 << 30:
        raise ValueError("at most 2^30 sequences")
    code = _check_heads(query, heads, kv_heads, width)
    q = query.stride()
    if q[2] != 1 and width > 1:
        raise ValueError("query needs a contiguous head width")
    c = _cache(key_cache, value_cache, pool, device, _E4M3, kv_heads, width)
    s = _scales(key_scale, value_scale, device, pages, kv_heads)
    columns, row = _table("block_table", block_table, device, batch)
    past = _lengths(lengths, device, batch)
    if columns * page >= 1 << 30:
        raise ValueError("a block table row holds at most 2^30 tokens")
    scale = _check_scale(scale, width)
    if out is None:
        out = torch.empty_like(query)         # half the time of asking for the format
        o = out.stride()
        if o[0] < o[1]:
            out = torch.empty_like(query, memory_format=torch.contiguous_format)
            o = out.stride()
    else:
        o = _out_rows(out, device, dtype, shape, query)
    if not batch:
        return out
    word = None if status is not None else _STATUS_AT.get(device)
    if word is None:
        word = _status_for(query, device, status)
    if _entry is None:
        _entry = _lib.words_entry("grs_quantized_attention")
    work, need = 0, _workspace_bytes(batch, heads, kv_heads, width, columns * page)
    if need:
        scratch = _lib.scratch(query, need)
        work = scratch.data_ptr()
    code = _entry(_pack(
        code, query.data_ptr(), q[0], q[1], key_cache.data_ptr(), value_cache.data_ptr(), c[0],
        c[1], c[2], key_scale.data_ptr(), value_scale.data_ptr(), s, block_table.data_ptr(), row,
        columns, past, pages, page, out.data_ptr(), o[0], o[1], batch, heads, kv_heads, width,
        scale, work, need, word, _lib.stream_on(device)))
    if code:
        _lib.check(code, "quantized attention")
    return out
