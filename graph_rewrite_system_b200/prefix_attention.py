"""Decode attention of a batch that shares a long prefix.

``paged_attention(shared_key=...)`` holds a prefix of a few hundred keys in the
shared memory of every group of beams (head width 32, one K/V head per query
head).  ``shared_prefix_attention`` is the form for long prefixes, grouped
heads and wider heads: the prefix is read once for the whole batch on the
tensor cores and joined with each beam's own pages and current token.

Inference only: no gradient is recorded.  The sm_100a kernels live in
``csrc/prefix_attention.cu`` and the grouped attention sources beside it; CPU
tensors raise.
"""
from __future__ import annotations

import torch

from . import _lib
from .prompt_attention import _check_heads, _check_out, _check_rows, _check_scale, _status_for


def shared_prefix_attention(
    query: torch.Tensor,
    prefix_key: torch.Tensor,
    prefix_value: torch.Tensor,
    key_cache: torch.Tensor | None = None,
    value_cache: torch.Tensor | None = None,
    block_table: torch.Tensor | None = None,
    lengths: torch.Tensor | None = None,
    *,
    current_key: torch.Tensor | None = None,
    current_value: torch.Tensor | None = None,
    current_valid: torch.Tensor | None = None,
    scale: float | None = None,
    out: torch.Tensor | None = None,
    status: torch.Tensor | None = None,
) -> torch.Tensor:
    """Attention of one query per beam, query [B, H, D], to the prefix
    prefix_key/prefix_value [N, Hkv, D] that every beam shares (N may be 0),
    then to the first ``lengths[b]`` tokens of the beam's pages, then to its
    current token.

    key_cache/value_cache [pages, page, Hkv, D] of one layout, block_table
    int32 [B, columns] and lengths int32 [B] come together (a
    ``PagedKVCache`` layer) or not at all; current_key/current_value
    [B, Hkv, D] of one layout come together, current_valid bool or uint8 [B]
    defaults to all valid.  bf16 or fp32, D <= 256 and contiguous; query head
    i reads K/V head ``i // (H // Hkv)``; ``scale`` defaults to
    ``1 / sqrt(D)``.  Beams without any key are zero.

    Page ids outside the cache are skipped and lengths beyond the table are
    cut; both are recorded in ``status`` (default: the device word that
    ``check_decode_status`` reads).  ``out`` must not overlap the inputs.  The
    call does not synchronise and can be captured into a CUDA graph.
    """
    _lib.require_cuda(query, prefix_key, prefix_value, key_cache, value_cache, block_table,
                      lengths, current_key, current_value, current_valid, out, status)
    if query.dim() != 3 or prefix_key.dim() != 3:
        raise ValueError("query must be [batch, heads, D], the prefix [keys, kv_heads, D]")
    batch, heads, width = query.shape
    num_prefix, kv_heads = prefix_key.shape[:2]
    _check_heads(query, kv_heads)
    _check_rows("query", query, query, tuple(query.shape))
    _check_rows("prefix_key", prefix_key, query, (num_prefix, kv_heads, width))
    _check_rows("prefix_value", prefix_value, query, (num_prefix, kv_heads, width))
    paged = (key_cache, value_cache, block_table, lengths)
    if any(t is None for t in paged) != all(t is None for t in paged):
        raise ValueError("caches, block table and lengths must be supplied together")
    columns = pages = page = 0
    strides = (0, 0, 0)
    if key_cache is not None:
        if key_cache.dim() != 4:
            raise ValueError("caches must be [pages, page, kv_heads, D]")
        pages, page = key_cache.shape[:2]
        _check_rows("key_cache", key_cache, query, (pages, page, kv_heads, width))
        _check_rows("value_cache", value_cache, query, (pages, page, kv_heads, width))
        if key_cache.stride() != value_cache.stride():
            raise ValueError("key/value caches must share a layout")
        strides = key_cache.stride()[:3]
        if (block_table.dtype != torch.int32 or block_table.dim() != 2
                or block_table.shape[0] != batch or block_table.device != query.device
                or (block_table.shape[1] > 1 and block_table.stride(1) != 1)):
            raise ValueError("block_table must be int32 [batch, columns] with contiguous rows")
        if (lengths.dtype != torch.int32 or tuple(lengths.shape) != (batch,)
                or not lengths.is_contiguous() or lengths.device != query.device):
            raise ValueError("lengths must be contiguous int32 [batch]")
        columns = block_table.shape[1] if page else 0
        if columns * page >= 1 << 30:
            raise ValueError("a block table row holds at most 2^30 tokens")
    if (current_key is None) != (current_value is None):
        raise ValueError("current key/value must be supplied together")
    cur_strides = (0, 0)
    if current_key is not None:
        _check_rows("current_key", current_key, query, (batch, kv_heads, width))
        _check_rows("current_value", current_value, query, (batch, kv_heads, width))
        if current_key.stride() != current_value.stride():
            raise ValueError("current key/value must share a layout")
        cur_strides = current_key.stride()[:2]
    if current_valid is not None:
        if current_key is None:
            raise ValueError("current_valid comes with the current key/value")
        if (current_valid.dtype not in (torch.bool, torch.uint8)
                or tuple(current_valid.shape) != (batch,) or not current_valid.is_contiguous()
                or current_valid.device != query.device):
            raise ValueError("current_valid must be contiguous bool or uint8 [batch]")
    if out is None:
        out = torch.empty(query.shape, dtype=query.dtype, device=query.device)
    else:
        inputs = (prefix_key, prefix_value, key_cache, value_cache, current_key, current_value)
        _check_out(out, query, *(t for t in inputs if t is not None and t.numel()))
    if not out.numel():
        return out
    scale = _check_scale(scale, width)
    word = _status_for(query.device, status)
    lib = _lib.lib()
    with _lib.on_device(query):
        stream = _lib.stream_of(query)
        need = lib.grs_shared_prefix_workspace_bytes(batch, heads, kv_heads, width, num_prefix)
        work = _lib.scratch(need, query.device, stream)
        code = lib.grs_shared_prefix_attention(
            _lib.DTYPE_CODES[query.dtype], query.data_ptr(), query.stride(0), query.stride(1),
            prefix_key.data_ptr(), prefix_key.stride(0), prefix_key.stride(1),
            prefix_value.data_ptr(), prefix_value.stride(0), prefix_value.stride(1), num_prefix,
            _lib.ptr(key_cache), _lib.ptr(value_cache), *strides, _lib.ptr(block_table),
            0 if block_table is None else block_table.stride(0), columns, _lib.ptr(lengths),
            pages, page, _lib.ptr(current_key), _lib.ptr(current_value), *cur_strides,
            _lib.ptr(current_valid), out.data_ptr(), out.stride(0), out.stride(1), batch, heads,
            kv_heads, width, scale,
            work.data_ptr(), work.numel(), word.data_ptr(), stream)
    _lib.check(code, "shared-prefix attention")
    return out
