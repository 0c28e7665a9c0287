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
