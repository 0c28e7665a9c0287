"""Keys and values of a token model in pages: as they are, or in 8 bits.

``PagedKVCache`` appends one token to every layer of every beam at once, with
the rollout's action states beside it.  ``append_tokens`` writes the keys and
values of one layer as the model makes them - one token per sequence or whole
packed prompts - and turns keys and queries by their positions on the way; pages
may be bf16 or fp32 like the inputs, or e4m3 with a scale for each page and
head.  ``TokenKVCache`` owns such pages for all layers: the rollout cache's free
list, reference counts and forks.

Inference only: no gradient is recorded.  The sm_100a kernels live in
``csrc/token_cache.cu`` and ``csrc/paged_cache.cu``; CPU tensors raise.
"""
from __future__ import annotations

from contextlib import nullcontext

import torch

from . import _lib
from .paged_cache import PagePool
from .prefix_attention import shared_prefix_attention
from .prompt_attention import _STATUS_AT, _rows, _status_for
from .quantized_attention import (_E4M3, _cache, _lengths, _scales, _table, quantized_attention)
from .rotary import _check_magnitude, _frequencies, _positions, _turned_out

_pack = _lib.words_of("grs_append_tokens").pack
_entry = None
_GUARDED = 2                                  # GRS_APPEND_GUARDED


def append_tokens(
    key: torch.Tensor,
    value: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    block_table: torch.Tensor,
    lengths: torch.Tensor,
    *,
    key_scale: torch.Tensor | None = None,
    value_scale: torch.Tensor | None = None,
    offsets: torch.Tensor | None = None,
    source_table: torch.Tensor | None = None,
    frequencies: torch.Tensor | None = None,
    interleaved: bool = False,
    magnitude: float = 1.0,
    positions: torch.Tensor | None = None,
    query: torch.Tensor | None = None,
    query_out: torch.Tensor | None = None,
    status: torch.Tensor | None = None,
) -> torch.Tensor | None:
    """Write key and value [T, Hkv, D] (bf16 or fp32, D <= 256 and contiguous)
    behind the ``lengths[b]`` tokens that each sequence has in its pages; returns
    the turned query [T, H, D], if one is given.

    key_cache/value_cache [pages, page, Hkv, D] of one layout, block_table int32
    [B, columns], lengths int32 [B] (before the call).  offsets int32 [B + 1],
    ascending: sequence b has the tokens ``offsets[b]:offsets[b + 1]``, possibly
    none; without offsets one each (T = B).  With ``frequencies`` keys and
    queries are turned as by ``rotate_positions``, at the place in the sequence
    or at ``positions`` (int32 or int64 [T]; behind a shared prefix, for
    instance, ``lengths`` plus its length).

    Caches have the inputs' dtype, or float8_e4m3fn with key_scale/value_scale
    fp32 [pages, Hkv], which the call writes: a code stands for code * scale.
    The scale of a page and head is the smallest power of two (from 2^-118 to
    2^119) that holds the largest finite value of its new rows within 448 (for
    turned keys the value before turning, times max(1, sqrt(2) * |magnitude|)),
    or the page's old scale if rows are there and it is larger; rows
    that are there move to a new scale.  Infinite values are held as NaN.  The
    rows of a page behind the new ones are left as they were.

    source_table (int32 [B, any columns that hold the lengths]): the rows that a sequence has in
    its first page to receive tokens are copied from the page that this table
    names there - the parent's, after a fork - as are their scales.  No page may
    receive tokens of two sequences, or receive tokens and be another's source;
    the caches overlap none of the inputs; pages that are not 8-bit hold less than
    2^31 elements a head.

    Tokens whose pages lie outside the cache or whose place the table does not
    hold are not written (kept rows without a source stay unspecified), which ``status`` records (default: the device word
    that ``check_decode_status`` reads).  Query rows of no sequence are left as
    they were in a given ``query_out`` and zero in a new one; ``query_out`` may
    be the query itself.  The call does not synchronise and can be captured into
    a CUDA graph.
    """
    global _entry
    device = key.get_device()
    if device < 0:
        _lib.require_cuda(key)
    place = _lib.elsewhere(device)
    if place is not None:
        with place:
            return append_tokens(
                key, value, key_cache, value_cache, block_table, lengths, key_scale=key_scale,
                value_scale=value_scale, offsets=offsets, source_table=source_table,
                frequencies=frequencies, interleaved=interleaved, magnitude=magnitude,
                positions=positions, query=query, query_out=query_out, status=status)
    shape, dtype = key.shape, key.dtype
    code = _lib.DTYPE_CODES.get(dtype)
    if code is None or len(shape) != 3:
        raise ValueError("keys must be bf16 or fp32 [tokens, kv_heads, D]")
    tokens, kv_heads, width = shape
    if not 1 <= width <= 256:
        raise ValueError("head widths from 1 to 256 are supported")
    if tokens >= 1 << 30 or not 0 < kv_heads < 1 << 30:
        raise ValueError("at most 2^30 tokens and heads, and one head at least")
    k = key.stride()
    if k[2] != 1 and width > 1:
        raise ValueError("key needs a contiguous head width")
    v = _rows("value", value, device, dtype, shape)
    pool = key_cache.shape
    if len(pool) != 4:
        raise ValueError("caches must be [pages, page, kv_heads, D]")
    pages, page = pool[:2]
    cache_code, scale_row, key_at, value_at = code, 0, 0, 0
    if key_cache.dtype is _E4M3:
        if key_scale is None or value_scale is None:
            raise ValueError("8-bit caches come with key and value scales")
        cache_code = 2
        c = _cache(key_cache, value_cache, pool, device, _E4M3, kv_heads, width)
        scale_row = _scales(key_scale, value_scale, device, pages, kv_heads)
        if pages > 1 and scale_row < kv_heads:
            raise ValueError("scales must not overlap themselves")
        key_at, value_at = key_scale.data_ptr(), value_scale.data_ptr()
        if key_at == value_at and pages:
            raise ValueError("key and value scales must not be one tensor")
    else:
        if key_scale is not None or value_scale is not None:
            raise ValueError("scales come with 8-bit caches")
        c = _cache(key_cache, value_cache, pool, device, dtype, kv_heads, width)
        if source_table is not None and page * width >= 1 << 31:
            raise ValueError("rows are copied between pages of less than 2^31 elements a head")
    if c[2] < width or c[1] < c[2] * kv_heads or c[0] < c[1] * page:
        need = 1                              # not pages of rows of heads: any order will do
        for size, step in sorted(zip(pool, c), key=lambda p: p[1]):
            if size > 1 and step < need:
                raise ValueError("a cache must not overlap itself")
            need = max(need, step * size)
    keys_at, values_at = key_cache.data_ptr(), value_cache.data_ptr()
    if keys_at == values_at and keys_at:
        raise ValueError("key and value caches must not be one tensor")
    rows = lengths.numel()
    past = _lengths(lengths, device, rows)
    if rows >= 1 << 29:
        raise ValueError("at most 2^29 sequences")
    columns, row = _table("block_table", block_table, device, rows)
    if columns * page >= 1 << 30:
        raise ValueError("a block table row holds at most 2^30 tokens")
    source = source_row = source_columns = 0
    if source_table is not None:
        source_columns, source_row = _table("source_table", source_table, device, rows)
        source = source_table.data_ptr()
    begins = 0
    if offsets is not None:
        if (offsets.dtype is not torch.int32 or offsets.shape != (rows + 1,)
                or not offsets.is_contiguous() or offsets.get_device() != device):
            _lib.require_cuda(offsets)
            raise ValueError("offsets must be contiguous int32 [sequences + 1] on the inputs' "
                             "device")
        begins = offsets.data_ptr()
    elif tokens != rows:
        raise ValueError("without offsets every sequence has one token")
    pairs = turns = 0
    if frequencies is not None:
        pairs, turns = _frequencies(frequencies, device, width), frequencies.data_ptr()
    elif query is not None or positions is not None:
        raise ValueError("query and positions come with frequencies")
    magnitude = _check_magnitude(magnitude)
    places = wide = 0
    if positions is not None:
        wide, places = _positions(positions, device, tokens), positions.data_ptr()
    heads = query_at = query_to = 0
    q = qo = (0, 0)
    fresh = query_out is None
    if query is not None:
        asked = query.shape
        if len(asked) != 3:
            raise ValueError("query must be [tokens, heads, D]")
        heads = asked[1]
        if not 0 < heads < 1 << 30 or heads % kv_heads:
            raise ValueError("query heads must be a multiple of the key/value heads")
        q = _rows("query", query, device, dtype, (tokens, heads, width))
        query_out, qo = _turned_out("query_out", query_out, query, device, dtype, q, key, value)
        query_at, query_to = query.data_ptr(), query_out.data_ptr()
    elif not fresh:
        raise ValueError("query_out comes with a query")
    if not tokens:
        return query_out
    flags = int(fresh)
    word = None if status is not None else _STATUS_AT.get(device)
    if word is None:
        if status is not None and status.shape == (2,) and status.is_contiguous():
            status, flags = status[:1], flags | _GUARDED
        word = _status_for(key, device, status)
    if _entry is None:
        _entry = _lib.words_entry("grs_append_tokens")
    code = _entry(_pack(
        code, cache_code, query_at, q[0], q[1], query_to, qo[0], qo[1], flags, key.data_ptr(),
        k[0], k[1], value.data_ptr(), v[0], v[1], keys_at, values_at,
        c[0], c[1], c[2], key_at, value_at, scale_row, block_table.data_ptr(), row, source,
        source_row, source_columns, columns, past, begins, places, wide, turns, pairs, bool(interleaved),
        magnitude, tokens, rows, heads, kv_heads, width, pages, page, word,
        _lib.stream_on(device)))
    if code:
        _lib.check(code, "append_tokens")
    return query_out


class TokenKVCache(PagePool):
    """Pages of a token model's keys and values, one arena per layer.

    ``keys`` and ``values`` [layers, capacity, page, heads, head_width] of
    ``dtype`` (bf16, fp32 or float8_e4m3fn); ``key_scales`` and
    ``value_scales`` fp32 [layers, capacity, heads] of 8-bit pages, else None.
    Block tables and lengths are device tensors, as in ``PagedKVCache``'s
    device-native API; nothing synchronises but ``check_status``.

    A decode step of beams, parents gathered by the search::

        table = cache.fork_device(parent_table, lengths)
        for layer in range(layers):
            ...
            query = cache.append(layer, key, value, table, lengths, source_table=parent_table,
                                 query=query, frequencies=frequencies)
            context = cache.attend(layer, query, table, lengths + 1)
        cache.check_status()
        cache.release_device(old_table, old_lengths)       # the parents' own rows

    A fork, allocation or release that fails shuts the pages: until
    ``check_status`` raises its error, later forks make no children and ``append``
    writes nothing, so a step that ran out of pages leaves its parents as they were.
    Every layer's ``append`` reads the parents' last pages: released before the last
    of them, they must not be given out again until then.
    """

    def __init__(self, *, layers: int, capacity: int, page_size: int, heads: int,
                 head_width: int, device, dtype: torch.dtype):
        if min(layers, capacity, page_size, heads, head_width) <= 0:
            raise ValueError("all cache dimensions must be positive")
        if dtype not in (torch.bfloat16, torch.float32, _E4M3):
            raise ValueError("TokenKVCache arenas are bf16, fp32 or float8_e4m3fn")
        device = torch.device(device)
        if device.type == "cuda" and device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        super().__init__(capacity, page_size, device)
        self.layers, self.heads, self.head_width, self.dtype = layers, heads, head_width, dtype
        self.key_scales = self.value_scales = None
        with self._here():
            self.keys = torch.empty(layers, capacity, page_size, heads, head_width,
                                    device=self.device, dtype=dtype)
            self.values = torch.empty_like(self.keys)
            if dtype is _E4M3:
                self.key_scales = torch.ones(layers, capacity, heads, device=self.device)
                self.value_scales = torch.ones_like(self.key_scales)
            # errors of append and attend, and of the pool's own calls, which guard the append
            self._words = torch.zeros(2, device=self.device, dtype=torch.int32)
        self._calls, self._status = self._words[:1], self._words[1:]

    # All that the cache does, its making among it, goes where append and attend go: to
    # the stream that this thread pinned on the device, with memory of that stream.
    def _stream(self) -> int:
        return _lib.stream_on(self.device.index)

    def _here(self):
        return _lib.elsewhere(self.device.index) or nullcontext()

    def reset(self) -> None:
        with self._here():
            self._calls.zero_()
            super().reset()

    def status_tensor(self) -> torch.Tensor:
        """An error recorded so far (int32 [1], 0 = ok) without synchronising."""
        with self._here():
            return self._words.amin(0, keepdim=True)

    def check_status(self) -> None:
        """Raise an error recorded by a kernel since the last check, the pool's first."""
        with self._here():
            calls, pool = self._words.tolist()
            if calls or pool:
                self._words.zero_()
                _lib.check(pool or calls, type(self).__name__)

    def _layer(self, layer: int) -> tuple:
        scales = (None, None)
        if self.key_scales is not None:
            scales = self.key_scales[layer], self.value_scales[layer]
        return self.keys[layer], self.values[layer], *scales

    def fork_device(self, parent_table: torch.Tensor, parent_lengths: torch.Tensor,
                    columns: int | None = None) -> torch.Tensor:
        """The block table of one child per parent row, int32 [n, columns]
        (default: one more than the parents'), before its next token: it shares
        the parent's full pages and owns a page of the free list for the token.
        parent_table int32 [n, cols], parent_lengths int32 [n].  The kept rows of
        the parent's last page follow with ``append(source_table=parent_table)``
        in every layer.

        All children or none: where a parent's table does not hold its length
        or names a page that is not allocated, ``columns`` leave a child no
        room or the pages run out - or an error is recorded that
        ``check_status`` has not raised yet - no page is shared or taken and the
        rows name none (-1; zeros where the parent's own length is the error).
        Once ``check_status`` has raised it, the fork can be tried again."""
        n = parent_lengths.shape[0]
        width, row = _table("parent_table", parent_table, self.device.index, n)
        past = _lengths(parent_lengths, self.device.index, n)
        columns = columns or width + 1
        with self._here():
            table = torch.empty(n, columns, device=self.device, dtype=torch.int32)
            if n:
                _lib.check(_lib.lib().grs_cache_fork(
                    self._refcounts.data_ptr(), self._free.data_ptr(),
                    self._free_count.data_ptr(), self.capacity, parent_table.data_ptr(), row,
                    width, past, n, self.page_size, table.data_ptr(), columns, None, columns,
                    self._status.data_ptr(), self._stream()), "fork")
        return table

    def append(self, layer: int, key: torch.Tensor, value: torch.Tensor,
               block_table: torch.Tensor, lengths: torch.Tensor, **options):
        """``append_tokens`` into one layer's pages (its keyword arguments)."""
        keys, values, key_scale, value_scale = self._layer(layer)
        return append_tokens(key, value, keys, values, block_table, lengths, key_scale=key_scale,
                             value_scale=value_scale, status=self._words, **options)

    def attend(self, layer: int, query: torch.Tensor, block_table: torch.Tensor,
               lengths: torch.Tensor, *, scale: float | None = None,
               out: torch.Tensor | None = None) -> torch.Tensor:
        """Attention of one query per row to its pages in one layer:
        ``quantized_attention``, or ``shared_prefix_attention`` without a prefix
        over pages of the query's type."""
        keys, values, key_scale, value_scale = self._layer(layer)
        if key_scale is not None:
            return quantized_attention(query, keys, values, key_scale, value_scale, block_table,
                                       lengths, scale=scale, out=out, status=self._calls)
        none = keys.new_empty(0, self.heads, self.head_width)
        return shared_prefix_attention(query, none, none, keys, values, block_table, lengths,
                                       scale=scale, out=out, status=self._calls)
