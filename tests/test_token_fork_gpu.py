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
