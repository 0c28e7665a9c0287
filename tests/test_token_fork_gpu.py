"""Forks of a TokenKVCache that cannot succeed, and what is done after them."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, FP32, E4M3 = torch.bfloat16, torch.float32, torch.float8_e4m3fn
LARGEST = (1 << 31) - 1


@pytest.mark.parametrize("page", [1, 4, 16, 1 << 20])
def test_lengths_near_2_to_the_31(cuda_device, page):
    """A length whose sum with the page size passes 32 bits is reported; nothing
    beside the child's row is written."""
    from graph_rewrite_system_b200 import _lib

    dev = cuda_device
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)
    for length in (LARGEST, LARGEST - 1, LARGEST - page + 2, LARGEST - page + 1, LARGEST // 2):
        refs, free, count = i32(1, 0, 0, 0), i32(3, 2, 1, 0), i32(3)
        room = torch.full((64, 3), 7, dtype=torch.int32, device=dev)
        table, lengths, child_lengths, status = i32(0, 0), i32(min(length, LARGEST)), i32(5), i32(0)
        _lib.check(_lib.lib().grs_cache_fork(
            refs.data_ptr(), free.data_ptr(), count.data_ptr(), 4, table.data_ptr(), 2, 2,
            lengths.data_ptr(), 1, page, room[32].data_ptr(), 3, child_lengths.data_ptr(), 3,
            status.data_ptr(), torch.cuda.current_stream().cuda_stream))
        assert int(status.item()) == -7, length
        assert not room[32].any()
        assert bool((room[:32] == 7).all()) and bool((room[33:] == 7).all())
        assert refs.tolist() == [1, 0, 0, 0]


@pytest.mark.parametrize("page", [1, 16])
def test_lengths_near_2_to_the_31_in_the_rollout_cache(cuda_device, page):
    from graph_rewrite_system_b200.paged_cache import PagedKVCache

    dev = cuda_device
    zeros = lambda *shape: torch.zeros(*shape, dtype=FP32, device=dev)
    for length in (LARGEST, LARGEST - max(page, 2) + 2):
        cache = PagedKVCache(layers=1, capacity=4, page_size=page, heads=1, head_width=4,
                             model_width=4, device=dev, dtype=FP32)
        kept = cache.keys.zero_()
        cache.append_device(torch.zeros(1, 1, dtype=torch.int32, device=dev),
                            torch.tensor([length], dtype=torch.int32, device=dev),
                            zeros(1, 1, 1, 4) + 1, zeros(1, 1, 1, 4) + 1, zeros(1, 4))
        with pytest.raises(ValueError, match="shape"):
            cache.check_status()
        assert not kept.any()


def _cache(dev, capacity=12, dtype=BF16, layers=1, page=4):
    from graph_rewrite_system_b200.token_cache import TokenKVCache

    return TokenKVCache(layers=layers, capacity=capacity, page_size=page, heads=2, head_width=16,
                        device=dev, dtype=dtype)


# what is wrong with a fork of two parents of pages of 4 tokens in tables of two columns
FAILURES = ["negative", "long", "far", "longest", "columns", "outside", "free page", "exhausted"]


def _failing(cache, kind):
    """Parents of 5 and 7 tokens, and the tables, lengths and options of a fork of them
    that cannot succeed, with the error that it records."""
    dev = cache.device
    table = cache.alloc_pages(4).view(2, 2)
    lengths = torch.tensor([5, 7], dtype=torch.int32, device=dev)
    asked, past, options, error = table.clone(), lengths.clone(), {}, "length"
    if kind in ("negative", "long", "far", "longest"):
        past[1] = {"negative": -1, "long": 9, "far": 1 << 30, "longest": LARGEST}[kind]
    elif kind == "columns":
        options, error = dict(columns=1), "shape"
    elif kind == "outside":
        asked[1, 0], error = cache.capacity, "unallocated"
    elif kind == "free page":
        asked[1, 0], error = cache.free[0], "unallocated"
    else:
        cache.alloc_pages(len(cache.free) - 1)
        error = "exhausted"
    return table, lengths, asked, past, options, error


@pytest.mark.parametrize("kind", FAILURES)
def test_failed_forks_change_nothing(cuda_device, kind):
    """Counts and free list as before, rows that name no page, and the fork works
    once its error is raised and its cause is gone."""
    cache = _cache(cuda_device)
    table, lengths, asked, past, options, error = _failing(cache, kind)
    before = cache.refcounts, cache.free, cache.allocated_pages
    child = cache.fork_device(asked, past, **options)
    again = cache.fork_device(table, lengths)            # its error is not raised yet
    assert (cache.refcounts, cache.free, cache.allocated_pages) == before
    own = kind in ("negative", "long", "far", "longest")
    assert bool((child[0] == -1).all()) and bool((child[1] == (0 if own else -1)).all())
    assert bool((again == -1).all())
    with pytest.raises((RuntimeError, ValueError), match=error):
        cache.check_status()
    if kind == "exhausted":
        held = [p for p, n in enumerate(cache.refcounts) if n and p not in table.tolist()[0]
                + table.tolist()[1]]
        cache.release_device(torch.tensor([held], dtype=torch.int32, device=cuda_device),
                             torch.tensor([4 * len(held)], dtype=torch.int32, device=cuda_device))
    child = cache.fork_device(table, lengths)
    cache.check_status()
    assert cache.allocated_pages == 6 and torch.equal(child[:, 0], table[:, 0])
    assert sorted(n for n in cache.refcounts if n) == [1, 1, 1, 1, 2, 2]
    cache.release_device(child, lengths + 1)
    cache.release_device(table, lengths)
    cache.check_status()
    assert cache.allocated_pages == 0 and cache.refcounts == [0] * cache.capacity


def test_forks_without_columns(cuda_device):
    """Parents without tokens in tables without columns."""
    cache = _cache(cuda_device)
    none = torch.zeros(3, 0, dtype=torch.int32, device=cuda_device)
    lengths = torch.zeros(3, dtype=torch.int32, device=cuda_device)
    child = cache.fork_device(none, lengths)
    cache.check_status()
    assert child.shape == (3, 1) and len(set(child.flatten().tolist())) == 3
    assert cache.allocated_pages == 3
    assert bool((cache.fork_device(none, lengths + 1) == 0).all())
    with pytest.raises(RuntimeError, match="length"):
        cache.check_status()
    assert cache.allocated_pages == 3


def _bits(t):
    return t.contiguous().view(torch.uint8).clone()


def _arenas(cache):
    return [_bits(t) for t in (cache.keys, cache.values, cache.key_scales, cache.value_scales)
            if t is not None]


def _fill(cache, seed):
    """Finite rows and scales in every page."""
    g = torch.Generator().manual_seed(seed)
    for t in (cache.keys, cache.values):
        t.copy_(torch.randn(t.shape, generator=g).to(t.dtype))
    if cache.key_scales is not None:
        cache.key_scales.fill_(0.5), cache.value_scales.fill_(2.0)


def _step(cache, table, lengths, source, qkv, frequencies, offsets=None):
    """New tokens of every layer and, for one each, their attention."""
    outs = []
    for layer in range(cache.layers):
        q, k, v = qkv[layer].split([4, 2, 2], 1)
        q = cache.append(layer, k, v, table, lengths, source_table=source, query=q,
                         frequencies=frequencies, offsets=offsets)
        outs.append(q)
        if offsets is None:
            outs.append(cache.attend(layer, q, table, lengths + 1))
    return outs


def _inputs(dev, tokens, dtype, seed=1):
    from graph_rewrite_system_b200.rotary import rotary_frequencies

    g = torch.Generator().manual_seed(seed)
    kind = FP32 if dtype is FP32 else BF16
    return (torch.randn(2, tokens, 8, 16, generator=g).to(kind).to(dev),
            rotary_frequencies(16, device=dev))


@pytest.mark.parametrize("dtype", [BF16, FP32, E4M3])
@pytest.mark.parametrize("kind", FAILURES)
def test_steps_after_failed_forks_write_nothing(cuda_device, kind, dtype):
    """Pages and scales of all layers, bit by bit, page 0 of a living row among them;
    tried again, the step is that of a cache whose fork did not fail."""
    dev = cuda_device
    qkv, f = _inputs(dev, 2, dtype)
    cache, other = (_cache(dev, dtype=dtype, layers=2) for _ in range(2))
    _fill(cache, 3), _fill(other, 3)
    table, lengths, asked, past, options, error = _failing(cache, kind)
    assert int(table.min()) == 0
    before = _arenas(cache)
    child = cache.fork_device(asked, past, **options)
    for columns in (child, torch.nn.functional.pad(child, (0, 2))):
        _step(cache, columns, lengths, table, qkv, f)
        _step(cache, columns, past, asked, qkv, f)
        _step(cache, columns, lengths, None, qkv, f,
              offsets=torch.tensor([0, 0, 2], dtype=torch.int32, device=dev))
    assert all(torch.equal(a, b) for a, b in zip(_arenas(cache), before))
    assert int(cache.status_tensor().item()) < 0
    with pytest.raises((RuntimeError, ValueError), match=error):
        cache.check_status()
    assert int(cache.status_tensor().item()) == 0
    if kind == "exhausted":
        cache.reset()
        assert torch.equal(cache.alloc_pages(4).view(2, 2), table)
    own = other.alloc_pages(4).view(2, 2)
    assert torch.equal(own, table)
    for c in (cache, other):
        child = c.fork_device(table, lengths)
        c.outs = _step(c, child, lengths, table, qkv, f)
        c.check_status()
    assert all(torch.equal(a, b) for a, b in zip(cache.outs, other.outs))
    assert all(torch.equal(a, b) for a, b in zip(_arenas(cache), _arenas(other)))
    assert not all(torch.equal(a, b) for a, b in zip(_arenas(cache), before))


@pytest.mark.parametrize("dtype", [BF16, E4M3])
def test_prompts_after_failed_allocations_write_nothing(cuda_device, dtype):
    dev = cuda_device
    qkv, f = _inputs(dev, 9, dtype)
    cache = _cache(dev, capacity=4, dtype=dtype, layers=2)
    _fill(cache, 4)
    mine = cache.alloc_pages(3).view(1, 3)
    before = _arenas(cache)
    table = cache.alloc_pages(3).view(1, 3)               # one page is left
    zero = torch.zeros(1, dtype=torch.int32, device=dev)
    offsets = torch.tensor([0, 9], dtype=torch.int32, device=dev)
    _step(cache, table, zero, None, qkv, f, offsets)
    assert all(torch.equal(a, b) for a, b in zip(_arenas(cache), before))
    with pytest.raises(RuntimeError, match="exhausted"):
        cache.check_status()
    _step(cache, mine, zero, None, qkv, f, offsets)
    cache.check_status()
    assert not all(torch.equal(a, b) for a, b in zip(_arenas(cache), before))


def test_errors_of_an_append_do_not_shut_the_pages(cuda_device):
    """A row without its page is reported; the others, and later calls, are written."""
    dev = cuda_device
    qkv, f = _inputs(dev, 2, BF16)
    cache = _cache(dev, layers=2)
    _fill(cache, 5)
    table = cache.alloc_pages(2).view(2, 1)
    bad = table.clone()
    bad[0] = -1
    zero = torch.zeros(2, dtype=torch.int32, device=dev)
    _step(cache, bad, zero, None, qkv, f)
    first = _arenas(cache)
    page = int(table[1, 0])
    assert torch.equal(cache.values[:, page, 0], qkv[:, 1, 6:])
    _step(cache, table, zero, None, qkv, f)
    assert not all(torch.equal(a, b) for a, b in zip(_arenas(cache), first))
    with pytest.raises(RuntimeError, match="unallocated"):
        cache.check_status()
    cache.check_status()


def test_a_guard_shuts_the_caches(cuda_device):
    """append_tokens with a status of two words, whatever is set in the second."""
    from graph_rewrite_system_b200.token_cache import append_tokens

    dev = cuda_device
    qkv, f = _inputs(dev, 3, BF16)
    q, k, v = qkv[0].split([4, 2, 2], 1)
    pages = torch.zeros(2, 4, 8, 2, 16, dtype=BF16, device=dev)
    table = torch.arange(3, dtype=torch.int32, device=dev).view(3, 1)
    lengths = torch.zeros(3, dtype=torch.int32, device=dev)
    call = lambda status: append_tokens(k, v, pages[0], pages[1], table, lengths, query=q,
                                        frequencies=f, status=status)
    for guard in (-1, 1, 1 << 30):
        words = torch.tensor([0, guard], dtype=torch.int32, device=dev)
        turned = call(words)
        assert not pages.any() and int(words[0]) == 0
    words = torch.zeros(2, dtype=torch.int32, device=dev)
    assert torch.equal(call(words), turned) and torch.equal(pages[1, :3, 0], v)
