"""bf16 attention whose scores lie far from zero, vs the fp64 oracle.

Queries and keys hold whole numbers, so that every product and sum of a score
is exact in fp32 and rows with scores of 1e5 still have a soft maximum over
their keys: what is left to test is the softmax alone.
"""
from __future__ import annotations

import math

import pytest
import torch

from oracle import grouped_attention as oracle

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def _inputs(seed, positions, heads, kv_heads, width, far, keys):
    """query [positions, heads, width], key [keys, kv_heads, width] of whole
    numbers whose scores are about f * far, f from -1 to 1 by row, apart by some
    tens among a row's keys and growing along them in some rows."""
    g = torch.Generator().manual_seed(seed)
    whole = lambda low, high, *s: torch.randint(low, high + 1, s, generator=g).float()
    query = whole(-1, 1, positions, heads, width)
    key = whole(-1, 1, keys, kv_heads, width)
    place = torch.tensor([256.0, -256.0, 0.0, 128.0, -3.0, 224.0, -16.0])
    query[:, :, 0] = place[torch.randint(0, 7, (positions, heads), generator=g)]
    key[:, :, 0] = far // 256
    query[:, :, 1] = whole(0, 1, positions, heads) * 4
    key[:, :, 1] = torch.linspace(-60, 60, keys).round()[:, None]
    query, key = query.to(BF16), key.to(BF16)
    assert far // 256 == key[0, 0, 0].item()
    return query, key, torch.randn(keys, kv_heads, width, generator=g).to(BF16)


def _check(got, oracle_out, far, keys, joined):
    """Scores are exact.  A weight is exp2 of c s - b with one rounding: b, about
    the row's maximum, is common to the weights it is taken with, c off by 2^-23
    at most.  What is not below 2^-126 is at most 126 below the maximum and this
    48 beside b: 2^-24 (174 + 2 * 126) in the exponent.  Where parts are joined,
    each part's log2 weight rounds once or, with the score's own product, twice,
    relative to the score.  Then what the oracle's bound counts: the exponential,
    the sums, the weights' and the output's rounding to bf16."""
    out, spread, _ = oracle_out
    exponent = 2.0 ** -24 * (174 + 2 * 126)
    if joined:
        exponent += 2 * 2.0 ** -24 * (1.1 * far + 400) * math.log2(math.e)
    weight = 2 * math.log(2) * exponent + 2 * 2.0 ** -21 + 2 * (keys + 8) * 2.0 ** -24 + 2.0 ** -8
    bound = 1.01 * (weight * spread + 2.0 ** -8 * out.abs()) + 1e-30
    assert torch.isfinite(got).all()
    worst = float(((got.double().cpu() - out).abs() / bound).max())
    assert worst <= 1.0, f"error {worst:.3f} of the bound"


FAR = [19968, 100352, 256]


@pytest.mark.parametrize("width", [32, 40, 64, 128])
@pytest.mark.parametrize("far", FAR)
@pytest.mark.parametrize("heads,kv_heads", [(3, 1), (128, 8)])
def test_prompt(cuda_device, heads, kv_heads, far, width):
    """Single row tiles and (with 128 heads) pairs of them; blocks of keys that a
    row sees in part, sequences that begin inside a tile."""
    from graph_rewrite_system_b200.prompt_attention import prompt_attention

    offsets = [0, 300, 301, 420]
    q, k, v = _inputs(width + heads, 420, heads, kv_heads, width, far, 420)
    dev = cuda_device
    got = prompt_attention(q.to(dev), k.to(dev), v.to(dev),
                           torch.tensor(offsets, dtype=torch.int32, device=dev), scale=1.0)
    _check(got, oracle.prompt_attention(q, k, v, offsets, scale=1.0), far, 300, joined=False)


@pytest.mark.parametrize("width", [32, 40, 64, 128])
@pytest.mark.parametrize("far", FAR)
@pytest.mark.parametrize("batch,group", [(20, 4), (70, 4), (60, 3)])
def test_prefix(cuda_device, batch, group, far, width):
    """Slices that two slots share (up to 128 rows) and slices of two row tiles,
    joined with the beams' own pages and current tokens."""
    from graph_rewrite_system_b200.prefix_attention import shared_prefix_attention

    prefix, page, columns = 1000, 16, 3
    pages = batch * columns
    q, k, v = _inputs(width + batch, batch, 2 * group, 2, width, far,
                      prefix + pages * page + batch)
    # the order in which the scores grow is mixed over the three kinds of keys
    order = torch.randperm(k.shape[0], generator=torch.Generator().manual_seed(5))
    k, v = k[order], v[order]
    parts = [prefix, pages * page, batch]
    (pk, kc, ck), (pv, vc, cv) = k.split(parts), v.split(parts)
    cache = lambda t: t.reshape(pages, page, 2, width).contiguous()
    g = torch.Generator().manual_seed(6)
    args = dict(query=q, prefix_key=pk.contiguous(), prefix_value=pv.contiguous(),
                key_cache=cache(kc), value_cache=cache(vc),
                block_table=torch.randperm(pages, generator=g).to(torch.int32).view(batch, columns),
                lengths=torch.randint(0, page * columns + 1, (batch,), generator=g,
                                      dtype=torch.int32),
                current_key=ck.contiguous(), current_value=cv.contiguous())
    got = shared_prefix_attention(**{n: t.to(cuda_device) for n, t in args.items()}, scale=1.0)
    _check(got, oracle.shared_prefix_attention(**args, scale=1.0), far, prefix + 50, joined=True)


@pytest.mark.parametrize("width", [64, 128])
def test_near_and_far_scales(cuda_device, width):
    """Random rows of growing size at the default scale: from soft rows to rows
    that one key decides; none of them is lost."""
    from graph_rewrite_system_b200.prefix_attention import shared_prefix_attention
    from graph_rewrite_system_b200.prompt_attention import prompt_attention

    g = torch.Generator().manual_seed(width)
    size = torch.logspace(0, 2.5, 300)[:, None, None]
    q = (torch.randn(300, 8, width, generator=g) * size).to(BF16)
    k = (torch.randn(700, 2, width, generator=g) * 90).to(BF16)
    v = torch.randn(700, 2, width, generator=g).to(BF16)
    dev = cuda_device
    for exp, got in (
            (oracle.prompt_attention(q, k[:300], v[:300], [0, 300]),
             prompt_attention(q.to(dev), k[:300].to(dev), v[:300].to(dev),
                              torch.tensor([0, 300], dtype=torch.int32, device=dev))),
            (oracle.shared_prefix_attention(q, k, v),
             shared_prefix_attention(q.to(dev), k.to(dev), v.to(dev)))):
        out, spread, reach = exp
        bound = oracle.attention_bound(out, spread, reach, BF16, width, 700)
        assert torch.isfinite(got).all()
        got = got.double().cpu()
        # a row is a mean of values: at least as large as the oracle's less its bound
        assert ((got - out).abs() <= bound).all()
        assert (got.abs().amax(-1) > 0).all()
