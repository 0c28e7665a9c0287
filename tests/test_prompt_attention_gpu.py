"""Causal attention over packed prompts vs the fp64 oracle."""
from __future__ import annotations

import pytest
import torch

from oracle import grouped_attention as oracle

pytestmark = pytest.mark.gpu


def _inputs(seed, tokens, heads, kv_heads, width, dtype):
    """Slices of one projection's output, as a model holds them."""
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn(tokens, heads + 2 * kv_heads, width, generator=g).to(dtype)
    return qkv.split([heads, kv_heads, kv_heads], 1)


def _offsets(lengths):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return out


def _call(dev, qkv, offsets, **kw):
    from graph_rewrite_system_b200.prompt_attention import prompt_attention

    base = qkv[0]._base if qkv[0]._base is not None else None
    if base is not None:                    # keep the slices' strides on the device
        sizes = [t.shape[1] for t in qkv]
        q, k, v = base.to(dev).split(sizes, 1)
    else:
        q, k, v = (t.to(dev) for t in qkv)
    return prompt_attention(q, k, v, torch.tensor(offsets, dtype=torch.int32, device=dev), **kw)


def _check(got, qkv, offsets, scale=None):
    out, spread, reach = oracle.prompt_attention(*qkv, offsets, scale=scale)
    bound = oracle.attention_bound(out, spread, reach, got.dtype, got.shape[2],
                                   max((b - a for a, b in zip(offsets, offsets[1:])), default=0))
    worst = ((got.double().cpu() - out).abs() / bound).max()
    assert torch.isfinite(got).all()
    assert float(worst) <= 1.0, f"error {float(worst):.3f} of the bound"


BF16, FP32 = torch.bfloat16, torch.float32
LENGTHS = {
    "one": [1], "pair": [1, 1], "tile": [128], "tile+1": [129], "two tiles": [256],
    "odd": [37], "empties": [0, 5, 0, 0, 1, 130, 0], "mixed": [127, 1, 300, 64, 2],
    "many": [3, 17, 1, 9, 0, 31, 33, 2, 64, 5] * 6, "long": [700],
    "hundreds empty": [5] + [0] * 700 + [70, 0, 3], "all empty between": ([0] * 300 + [9]) * 3,
    "thousands": [1, 0, 2] * 900,
}


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("name", list(LENGTHS))
def test_lengths(cuda_device, name, dtype):
    offsets = _offsets(LENGTHS[name])
    qkv = _inputs(len(name), offsets[-1], 4, 2, 64, dtype)
    _check(_call(cuda_device, qkv, offsets), qkv, offsets)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("heads,kv_heads", [(8, 8), (8, 1), (3, 1), (10, 2), (14, 2), (24, 2),
                                            (71, 1), (130, 1)])
def test_head_groups(cuda_device, heads, kv_heads, dtype):
    offsets = _offsets([50, 1, 90])
    qkv = _inputs(heads, offsets[-1], heads, kv_heads, 32, dtype)
    _check(_call(cuda_device, qkv, offsets), qkv, offsets)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("width", [1, 8, 20, 32, 33, 40, 64, 80, 96, 120, 128, 160, 256])
def test_widths(cuda_device, width, dtype):
    offsets = _offsets([70, 140])
    qkv = _inputs(width, offsets[-1], 4, 2, width, dtype)
    _check(_call(cuda_device, qkv, offsets), qkv, offsets)


def test_large_scores(cuda_device):
    # scores of some hundreds: the running maximum moves often and far
    offsets = _offsets([300, 200])
    q, k, v = _inputs(3, offsets[-1], 4, 2, 64, BF16)
    q = (q.float() * torch.linspace(0.1, 12, 500)[:, None, None]).to(BF16)
    _check(_call(cuda_device, (q, k.contiguous(), v.contiguous()), offsets), (q, k, v), offsets)


@pytest.mark.parametrize("scale", [0.0, -0.3, 1.0])
def test_scale(cuda_device, scale):
    offsets = _offsets([150])
    qkv = _inputs(4, 150, 2, 1, 64, BF16)
    _check(_call(cuda_device, qkv, offsets, scale=scale), qkv, offsets, scale)


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_rows_behind_the_last_sequence(cuda_device, dtype):
    """NaN behind the last prompt reaches no row; a given out keeps its rows
    there, a new one has zeros."""
    offsets = _offsets([60, 75])
    base = torch.cat(_inputs(5, 180, 4, 2, 64, dtype), 1)
    clean = base.clone().split([4, 2, 2], 1)
    base[135:] = float("nan")
    base = base.to(cuda_device)
    from graph_rewrite_system_b200.prompt_attention import prompt_attention

    q, k, v = base.split([4, 2, 2], 1)
    off = torch.tensor(offsets, dtype=torch.int32, device=cuda_device)
    got = prompt_attention(q, k, v, off)
    assert not got[135:].any()
    _check(got, clean, offsets)
    out = torch.full_like(got, 7.0)
    assert prompt_attention(q, k, v, off, out=out) is out
    assert (out[135:] == 7).all() and torch.equal(out[:135], got[:135])
    # rows before the first sequence are nobody's either
    out.fill_(7.0)
    prompt_attention(q, k, v, off[1:], out=out)
    assert (out[:60] == 7).all()
    # (another packing: the key blocks start elsewhere, so sums may round apart)
    out[:60] = got[:60]
    out[135:] = 0
    _check(out, clean, offsets)


@pytest.mark.parametrize("width", [32, 64, 128])
@pytest.mark.parametrize("sequences", [0, 1, 40])
def test_long_tails(cuda_device, width, sequences):
    """Whole tiles behind the last sequence, holding NaN, many times over: the
    rows are zero in a new output and untouched in a given one."""
    from graph_rewrite_system_b200.prompt_attention import prompt_attention

    offsets = _offsets([70] * sequences)
    base = torch.cat(_inputs(16, offsets[-1] + 3000, 8, 2, width, BF16), 1).to(cuda_device)
    base[offsets[-1]:] = float("nan")
    q, k, v = base.split([8, 2, 2], 1)
    off = torch.tensor(offsets, dtype=torch.int32, device=cuda_device)
    first = prompt_attention(q, k, v, off)
    out = torch.full_like(first, 3.0)
    for _ in range(20):
        assert torch.equal(prompt_attention(q, k, v, off), first)
        prompt_attention(q, k, v, off, out=out)
    assert not first[offsets[-1]:].any() and torch.isfinite(first).all()
    assert (out[offsets[-1]:] == 3).all() and torch.equal(out[:offsets[-1]], first[:offsets[-1]])


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_bad_values_reach_only_rows_that_see_them(cuda_device, dtype, bad):
    offsets = _offsets([90, 40, 70])
    base = torch.cat(_inputs(6, 200, 4, 2, 64, dtype), 1)
    clean = base.clone().split([4, 2, 2], 1)
    base[110, 6:] = bad                     # value rows of token 20 of the second prompt
    base[110, 4:6] = float("nan")           # and its keys
    got = _call(cuda_device, [t for t in base.split([4, 2, 2], 1)], offsets)
    seeing = torch.zeros(200, dtype=torch.bool)
    seeing[110:130] = True
    assert torch.isnan(got[seeing.to(got.device)]).all()
    out, spread, reach = oracle.prompt_attention(*clean, offsets)
    bound = oracle.attention_bound(out, spread, reach, dtype, 64, 90)
    off = (got.double().cpu() - out).abs() / bound
    assert float(off[~seeing].max()) <= 1.0
    # an infinite value with finite keys: the rows that see it are infinite in it
    if bad == float("inf"):
        base[110, 4:6] = clean[1][110]
        got = _call(cuda_device, [t for t in base.split([4, 2, 2], 1)], offsets)
        assert (got[seeing.to(got.device)] == bad).all()
        assert torch.isfinite(got[~seeing.to(got.device)]).all()


def test_layouts(cuda_device):
    """Head-major tensors, unaligned rows and an out inside a larger buffer."""
    from graph_rewrite_system_b200.prompt_attention import prompt_attention

    offsets = _offsets([80, 33])
    q, k, v = (t.contiguous() for t in _inputs(8, 113, 6, 3, 64, BF16))
    off = torch.tensor(offsets, dtype=torch.int32, device=cuda_device)
    head_major = [t.transpose(0, 1).contiguous().to(cuda_device).transpose(0, 1) for t in (q, k, v)]
    _check(prompt_attention(*head_major, off), (q, k, v), offsets)
    shifted = []
    for t in (q, k, v):
        room = torch.zeros(t.numel() + 1, dtype=BF16, device=cuda_device)
        room[1:] = t.to(cuda_device).reshape(-1)
        shifted.append(room[1:].view(t.shape))
    big = torch.zeros(113, 8, 65, dtype=BF16, device=cuda_device)
    out = big[:, 1:7, :64]
    _check(prompt_attention(*shifted, off, out=out), (q, k, v), offsets)
    assert not big[:, 0].any() and not big[:, 7].any() and not big[:, :, 64].any()
    one = k[:, :1].to(cuda_device).expand(-1, 3, -1)      # one K/V head broadcast to three
    _check(prompt_attention(q.to(cuda_device), one, one, off),
           (q, k[:, :1].expand(-1, 3, -1), k[:, :1].expand(-1, 3, -1)), offsets)


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_far_rows(cuda_device, dtype):
    """Tokens whose rows start past 2^31 elements: q, k, v and out in one
    buffer."""
    from graph_rewrite_system_b200.prompt_attention import prompt_attention

    step = (1 << 20) + 64
    offsets = _offsets([700, 1, 1340, 9])
    tokens = offsets[-1]
    if torch.cuda.mem_get_info()[0] < tokens * step * dtype.itemsize + (1 << 30):
        pytest.skip("needs 10 GB")
    buffer = torch.empty(tokens, step // 64, 64, dtype=dtype, device=cuda_device)
    assert buffer[-1].data_ptr() - buffer.data_ptr() > (1 << 31) * dtype.itemsize
    qkv = _inputs(12, tokens, 4, 2, 64, dtype)
    q, k, v, out = buffer[:, :12].split([4, 2, 2, 4], 1)
    for into, t in zip((q, k, v), qkv):
        into.copy_(t)
    off = torch.tensor(offsets, dtype=torch.int32, device=cuda_device)
    _check(prompt_attention(q, k, v, off, out=out), qkv, offsets)


@pytest.mark.parametrize("values", [[0, 0], [0], [5, 3, 90], [-7, 40, 400], [200, 100],
                                    [2 ** 31 - 1, -2 ** 31]])
def test_any_offsets_are_safe(cuda_device, values):
    """Offsets that describe no packing move no access out of the tensors;
    the rows of no sequence are left as they were."""
    from graph_rewrite_system_b200.paged_attention import check_decode_status

    qkv = _inputs(9, 100, 4, 2, 64, BF16)
    got = _call(cuda_device, qkv, values)
    torch.cuda.synchronize()
    check_decode_status(cuda_device)
    if values in ([0, 0], [0]):
        assert not got.any()


def test_captured_and_on_another_stream(cuda_device):
    """A captured call reads the offsets and rows of its replay; two graphs
    and an eager call on another stream do not disturb each other."""
    from graph_rewrite_system_b200.prompt_attention import prompt_attention

    dev = cuda_device
    sets = []
    for seed, lengths in ((10, [90, 38]), (11, [1, 127])):
        qkv = torch.cat(_inputs(seed, 128, 4, 2, 64, BF16), 1)
        sets.append((qkv, _offsets(lengths)))
    qkv = sets[0][0].to(dev)
    off = torch.tensor(sets[0][1], dtype=torch.int32, device=dev)
    q, k, v = qkv.split([4, 2, 2], 1)
    eager = prompt_attention(q, k, v, off)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(prompt_attention(q, k, v, off))
        graphs.append(g)
    for rows, offsets in sets[::-1]:
        qkv.copy_(rows)
        off.copy_(torch.tensor(offsets, dtype=torch.int32))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = prompt_attention(q, k, v, off)
        for g in graphs:
            g.replay()
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], other)
        _check(outs[0], rows.split([4, 2, 2], 1), offsets)
    assert torch.equal(outs[0], eager)


def test_same_answer_twice(cuda_device):
    qkv = _inputs(12, 600, 8, 2, 128, BF16)
    offsets = _offsets([333, 267])
    assert torch.equal(_call(cuda_device, qkv, offsets), _call(cuda_device, qkv, offsets))
