"""Decode attention of a batch that shares a long prefix.

``paged_attention(shared_key=...)`` holds a prefix of a few hundred keys in the
shared memory of every group of beams (head width 32, one K/V head per query
head).  ``shared_prefix_attention`` is the form for long prefixes, grouped
heads and wider heads: a long prefix is read once for the whole batch (bf16 on
the tensor cores) and joined with each beam's own pages and current token; a
short one, up to 256 keys, is read with the beam's own keys in one launch.

Inference only: no gradient is recorded.  The sm_100a kernels live in
``csrc/prefix_attention.cu`` and the grouped attention sources beside it; CPU
tensors raise.
"""
from __future__ import annotations

from functools import lru_cache

import torch

from . import _lib
from .prompt_attention import (_STATUS_AT, _check_heads, _check_scale, _out_rows, _rows,
                               _status_for)

_pack = _lib.words_of("grs_shared_prefix_attention").pack
_entry = None


@lru_cache(maxsize=4096)
def _workspace_bytes(*sizes: int) -> int:
    return _lib.lib().grs_shared_prefix_workspace_bytes(*sizes)


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
    global _entry
    device = query.get_device()
    if device < 0:
        _lib.require_cuda(query)
    place = _lib.elsewhere(device)
    if place is not None:
        with place:
            return shared_prefix_attention(
                query, prefix_key, prefix_value, key_cache, value_cache, block_table, lengths,
                current_key=current_key, current_value=current_value,
                current_valid=current_valid, scale=scale, out=out, status=status)
    if query.dim() != 3 or prefix_key.dim() != 3:
        raise ValueError("query must be [batch, heads, D], the prefix [keys, kv_heads, D]")
    shape = query.shape
    batch, heads, width = shape
    num_prefix, kv_heads, _ = prefix_key.shape
    if batch >= 1 << 30 or num_prefix >= 1 << 30:
        raise ValueError("at most 2^30 beams and prefix keys")
    code, dtype = _check_heads(query, heads, kv_heads, width), query.dtype
    q = query.stride()
    if q[2] != 1 and width > 1:
        raise ValueError("query needs a contiguous head width")
    pk = _rows("prefix_key", prefix_key, device, dtype, (num_prefix, kv_heads, width))
    pv = _rows("prefix_value", prefix_value, device, dtype, (num_prefix, kv_heads, width))

    columns = pages = page = table_row = 0
    c = (0, 0, 0)
    keys = values = table = past = 0
    if key_cache is None or value_cache is None or block_table is None or lengths is None:
        if not (key_cache is value_cache is block_table is lengths):
            raise ValueError("caches, block table and lengths must be supplied together")
    else:
        if key_cache.dim() != 4:
            raise ValueError("caches must be [pages, page, kv_heads, D]")
        pages, page = key_cache.shape[:2]
        c = _rows("key_cache", key_cache, device, dtype, (pages, page, kv_heads, width))
        if c != _rows("value_cache", value_cache, device, dtype, (pages, page, kv_heads, width)):
            raise ValueError("key/value caches must share a layout")
        if (block_table.dtype is not torch.int32 or block_table.dim() != 2
                or block_table.get_device() != device):
            _lib.require_cuda(block_table)
            raise ValueError("block_table must be int32 [batch, columns] on the query's device")
        rows, columns = block_table.shape
        table_row, step = block_table.stride()
        if rows != batch or (columns > 1 and step != 1):
            raise ValueError("block_table must be [batch, columns] with contiguous rows")
        if (lengths.dtype is not torch.int32 or lengths.shape != (batch,)
                or not lengths.is_contiguous() or lengths.get_device() != device):
            _lib.require_cuda(lengths)
            raise ValueError("lengths must be contiguous int32 [batch] on the query's device")
        if columns * page >= 1 << 30 or pages >= 1 << 31 or columns >= 1 << 30 or page >= 1 << 30:
            raise ValueError("a block table row holds at most 2^30 tokens")
        columns = columns if page else 0
        keys, values = key_cache.data_ptr(), value_cache.data_ptr()
        table, past = block_table.data_ptr(), lengths.data_ptr()

    cur = (0, 0)
    cur_key = cur_value = valid = 0
    if (current_key is None) != (current_value is None):
        raise ValueError("current key/value must be supplied together")
    if current_key is not None:
        cur = _rows("current_key", current_key, device, dtype, (batch, kv_heads, width))
        if cur != _rows("current_value", current_value, device, dtype, (batch, kv_heads, width)):
            raise ValueError("current key/value must share a layout")
        cur_key, cur_value = current_key.data_ptr(), current_value.data_ptr()
    if current_valid is not None:
        if current_key is None:
            raise ValueError("current_valid comes with the current key/value")
        if (current_valid.dtype not in (torch.bool, torch.uint8)
                or current_valid.shape != (batch,) or not current_valid.is_contiguous()
                or current_valid.get_device() != device):
            _lib.require_cuda(current_valid)
            raise ValueError("current_valid must be contiguous bool or uint8 [batch]")
        valid = current_valid.data_ptr()
    scale = _check_scale(scale, width)
    if out is None:
        out = torch.empty_like(query, memory_format=torch.contiguous_format)
        o = (heads * width, width)
    else:
        o = _out_rows(out, device, dtype, shape, query, prefix_key, prefix_value, key_cache,
                      value_cache, current_key, current_value)
    if not batch:
        return out
    word = None if status is not None else _STATUS_AT.get(device)
    if word is None:
        word = _status_for(query, device, status)
    if _entry is None:
        _entry = _lib.words_entry("grs_shared_prefix_attention")
    work, need = 0, _workspace_bytes(batch, heads, kv_heads, width, num_prefix, columns * page)
    if need:
        scratch = _lib.scratch(query, need)
        work = scratch.data_ptr()
    code = _entry(_pack(
        code, query.data_ptr(), q[0], q[1], prefix_key.data_ptr(), pk[0], pk[1],
        prefix_value.data_ptr(), pv[0], pv[1], num_prefix, keys, values, c[0], c[1], c[2], table,
        table_row, columns, past, pages, page, cur_key, cur_value, cur[0], cur[1], valid,
        out.data_ptr(), o[0], o[1], batch, heads, kv_heads, width, scale, work, need, word,
        _lib.stream_on(device)))
    if code:
        _lib.check(code, "shared-prefix attention")
    return out
