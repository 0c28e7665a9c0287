"""Packed prompts whose offsets describe no packing: what is read and written.

The tensors lie inside larger buffers, NaN around the inputs and a mark around
the output; the range of every row is restated on the host."""
from __future__ import annotations

import pytest
import torch

from oracle import grouped_attention as oracle

pytestmark = pytest.mark.gpu

BF16, FP32 = torch.bfloat16, torch.float32
TOKENS, HEADS, KV_HEADS, WIDTH, AROUND, MARK = 100, 4, 2, 64, 96, 7.0


def _ranges(offsets):
    """The keys [begin, end) of every token: of the sequence that a binary search
    finds, clamped to the token; empty behind the last and before the first."""
    out = []
    for p in range(TOKENS):
        lo, hi = 0, len(offsets)
        while lo < hi:
            mid = (lo + hi) // 2
            if offsets[mid] <= p:
                lo = mid + 1
            else:
                hi = mid
        inside = 0 < lo < len(offsets)
        out.append((min(max(offsets[lo - 1], 0), p), p + 1) if inside else (0, 0))
    return out


def _inside(t, fill, dev):
    """t as the middle rows of a buffer of `fill`, and the buffer."""
    room = torch.full((TOKENS + 2 * AROUND,) + tuple(t.shape[1:]), fill, dtype=t.dtype, device=dev)
    part = room[AROUND:AROUND + TOKENS]
    part.copy_(t)
    return part, room


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("offsets", [
    [0, 0], [0], [5, 3, 90], [-7, 40, 400], [200, 100], [2 ** 31 - 1, -2 ** 31],
    [-2 ** 31, 2 ** 31 - 1], [99, 100], [50, 50, 50, 60], [-5, -3, -1], [100, 100],
    [-9] * 400 + [20, 70] + [500] * 400], ids=lambda o: f"{o[0]}..{o[-1]} of {len(o)}")
def test_rows_and_their_surroundings(cuda_device, offsets, dtype):
    from graph_rewrite_system_b200.paged_attention import check_decode_status
    from graph_rewrite_system_b200.prompt_attention import prompt_attention

    g = torch.Generator().manual_seed(len(offsets))
    host = [torch.randn(TOKENS, h, WIDTH, generator=g).to(dtype)
            for h in (HEADS, KV_HEADS, KV_HEADS)]
    (q, _), (k, _), (v, _) = (_inside(t, float("nan"), cuda_device) for t in host)
    out, room = _inside(torch.full((TOKENS, HEADS, WIDTH), MARK, dtype=dtype), MARK, cuda_device)
    at = torch.tensor(offsets, dtype=torch.int32, device=cuda_device)
    prompt_attention(q, k, v, at, out=out)
    check_decode_status(cuda_device)
    assert (room[:AROUND] == MARK).all() and (room[AROUND + TOKENS:] == MARK).all()
    fresh = prompt_attention(q, k, v, at)
    got = out.double().cpu()
    for p, (begin, end) in enumerate(_ranges(offsets)):
        if begin == end:
            assert (got[p] == MARK).all() and not fresh[p].any()
            continue
        # the row alone as the last of its keys
        rows, spread, reach = oracle.prompt_attention(*(t[begin:end] for t in host),
                                                      [0, end - begin])
        bound = oracle.attention_bound(rows[-1:], spread[-1:], reach[-1:], dtype, WIDTH, TOKENS)
        assert float(((got[p] - rows[-1]).abs() / bound[0]).max()) <= 1.0
        assert torch.equal(fresh[p], out[p])
