"""Rotary positions vs the fp64 oracle."""
from __future__ import annotations

import pytest
import torch

from oracle import token_cache as oracle

pytestmark = pytest.mark.gpu

BF16, FP32 = torch.bfloat16, torch.float32


def _freq(rotated, **kw):
    from graph_rewrite_system_b200.rotary import rotary_frequencies

    return rotary_frequencies(rotated, device="cpu", **kw)


def _case(seed, tokens, heads, kv_heads, width, dtype, far=5000, ids=torch.int32):
    g = torch.Generator().manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g).to(dtype)
    positions = torch.randint(-far, far + 1, (tokens,), generator=g, dtype=torch.int64)
    return rand(tokens, heads, width), rand(tokens, kv_heads, width), positions.to(ids)


def _call(dev, q, k, p, f, **kw):
    from graph_rewrite_system_b200.rotary import rotate_positions

    return rotate_positions(q.to(dev), None if k is None else k.to(dev), p.to(dev), f.to(dev), **kw)


def _check(got, x, p, f, interleaved=False, magnitude=1.0):
    out, reach = oracle.turn(x, p, f, interleaved, magnitude)
    bound = oracle.turn_bound(out, reach, x.dtype)
    assert got.dtype is x.dtype and got.shape == x.shape
    off = (got.double().cpu() - out).abs()
    assert bool((off <= bound).all()), float((off - bound).max())


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("width,rotated", [
    (2, 2), (6, 4), (8, 8), (32, 32), (33, 30), (40, 40), (40, 20), (64, 32), (64, 2), (80, 80),
    (96, 48), (100, 50), (128, 128), (128, 96), (256, 256), (256, 64), (255, 254)])
def test_widths(cuda_device, width, rotated, interleaved, dtype):
    q, k, p = _case(width, 7, 3, 2, width, dtype)
    f = _freq(rotated)
    got = _call(cuda_device, q, k, p, f, interleaved=interleaved, magnitude=1.3)
    _check(got[0], q, p, f, interleaved, 1.3)
    _check(got[1], k, p, f, interleaved, 1.3)


@pytest.mark.parametrize("tokens,heads,kv_heads,width", [
    (1, 1, 1, 64), (1, 32, 8, 128), (5, 8, 8, 32), (700, 2, 1, 32), (1200, 1, 1, 8),
    (37, 300, 1, 16), (3000, 1, 1, 2)])
def test_sizes(cuda_device, tokens, heads, kv_heads, width):
    """From one token to several for each CTA, with what is left at the end."""
    q, k, p = _case(tokens, tokens, heads, kv_heads, width, BF16)
    f = _freq(width)
    got = _call(cuda_device, q, k, p, f)
    _check(got[0], q, p, f)
    _check(got[1], k, p, f)
    alone = _call(cuda_device, q, None, p, f)
    assert alone[1] is None and torch.equal(alone[0], got[0])


@pytest.mark.parametrize("far,ids", [(2 ** 31 - 1, torch.int32), (2 ** 40, torch.int64),
                                     (2 ** 62, torch.int64)])
def test_far_positions(cuda_device, far, ids):
    """Angles lose nothing at far positions, on either side of zero."""
    q, k, p = _case(3, 40, 2, 1, 64, FP32, far, ids)
    p[0], p[1], p[2] = far, -far, 0
    f = _freq(64)
    got = _call(cuda_device, q, k, p, f)
    _check(got[0], q, p, f)
    _check(got[1], k, p, f)
    assert torch.equal(got[0][2].cpu(), q[2])


def test_any_frequencies(cuda_device):
    """Zero, negative, beyond a turn per position, tiny."""
    f = torch.tensor([0.0, -1.25, 6.2831853071795864, 1e3, 3.3e-9, 1e-300, 3.0, 0.1],
                     dtype=torch.float64)
    q, k, p = _case(4, 30, 2, 1, 16, FP32, 10 ** 6)
    got = _call(cuda_device, q, k, p, f)
    _check(got[0], q, p, f)


def test_stretched_frequencies(cuda_device):
    plain = _freq(64)
    assert torch.equal(_freq(64, stretch=4.0), plain / 4)
    f = _freq(64, stretch=8.0, trained=4096)
    turns = 4096 * plain / (2 * torch.pi)
    assert torch.equal(f[turns >= 4], plain[turns >= 4])
    assert torch.allclose(f[turns <= 1], plain[turns <= 1] / 8, rtol=1e-15)
    between = (turns > 1) & (turns < 4)
    assert between.any() and bool(((f < plain) & (f > plain / 8))[between].all())


def test_there_and_back(cuda_device):
    q, k, p = _case(5, 50, 4, 2, 64, FP32, 10 ** 6)
    f = _freq(64)
    there = _call(cuda_device, q, k, p, f)
    back = _call(cuda_device, there[0], there[1], -p, f)
    # two turns of (|a| + |b|) <= sqrt(2) of the pair's length, 10 2^-24 each
    bound = 30 * 2.0 ** -24 * q.double().abs().amax()
    assert float((back[0].double().cpu() - q.double()).abs().max()) <= float(bound)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("interleaved", [False, True])
def test_layouts(cuda_device, dtype, interleaved):
    """Slices of one projection, in place, rows off 16 and off 8 bytes, heads
    before tokens, given outputs."""
    from graph_rewrite_system_b200.rotary import rotate_positions

    dev = cuda_device
    q, k, p = _case(6, 21, 6, 2, 64, dtype)
    f = _freq(48)
    exp = _call(dev, q, k, p, f, interleaved=interleaved)
    _check(exp[0], q, p, f, interleaved)
    pd, fd = p.to(dev), f.to(dev)
    for pad in (0, 1, 2, 4):
        room = torch.full((21, 10 * 64 + pad), 7.0, dtype=dtype, device=dev)
        flat = room.flatten()[pad:pad + 20 * (10 * 64 + pad) + 640]
        qkv = flat.as_strided((21, 10, 64), (10 * 64 + pad, 64, 1))
        qkv[:, :6], qkv[:, 6:8], qkv[:, 8:] = q.to(dev), k.to(dev), 5.0
        a, b, _ = qkv.split([6, 2, 2], 1)
        got = rotate_positions(a, b, pd, fd, interleaved=interleaved)
        assert torch.equal(got[0], exp[0]) and torch.equal(got[1], exp[1])
        assert torch.equal(a.cpu(), q)
        got = rotate_positions(a, b, pd, fd, interleaved=interleaved, query_out=a, key_out=b)
        assert got[0] is a and torch.equal(a, exp[0]) and torch.equal(b, exp[1])
        assert bool((qkv[:, 8:] == 5.0).all())
    swapped = q.to(dev).transpose(0, 1).contiguous().transpose(0, 1)
    out = torch.zeros(6, 21, 64, dtype=dtype, device=dev).transpose(0, 1)
    got = rotate_positions(swapped, None, pd, fd, interleaved=interleaved, query_out=out)
    assert got[0] is out and torch.equal(out, exp[0])
    one = q[:, :1].to(dev).expand(21, 6, 64)      # a head read for six
    got = rotate_positions(one, None, pd, fd, interleaved=interleaved)
    _check(got[0], q[:, :1].expand(21, 6, 64), p, f, interleaved)


def test_values_stay_in_their_pair(cuda_device):
    q, k, p = _case(7, 9, 2, 1, 32, FP32)
    f = _freq(16)
    clean = _call(cuda_device, q, k, p, f)[0].cpu()
    q[3, 1, 5], q[4, 0, 30] = float("nan"), float("inf")
    got = _call(cuda_device, q, k, p, f)[0].cpu()
    assert torch.isnan(got[3, 1, 5]) and torch.isnan(got[3, 1, 13]) and got[4, 0, 30] == float("inf")
    for at in ((3, 1, 5), (3, 1, 13), (4, 0, 30)):
        got[at] = clean[at] = 0
    assert torch.equal(got, clean)


def test_no_tokens(cuda_device):
    q, k, p = _case(8, 0, 2, 1, 32, BF16)
    got = _call(cuda_device, q, k, p, _freq(32))
    assert got[0].shape == (0, 2, 32) and got[1].shape == (0, 1, 32)


def test_captured_and_on_another_stream(cuda_device):
    from graph_rewrite_system_b200.rotary import rotate_positions

    q, k, p = (t.to(cuda_device) for t in _case(9, 33, 4, 2, 64, BF16))
    f = _freq(64).to(cuda_device)
    exp = rotate_positions(q, k, p, f)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = rotate_positions(q, k, p, f)
    p += 17
    graph.replay()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = rotate_positions(q, k, p, f)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out[0], other[0]) and torch.equal(out[1], other[1])
    assert not torch.equal(out[0], exp[0])
    _check(out[0], q.cpu(), p.cpu(), f.cpu())


def test_far_rows(cuda_device):
    """Rows whose last starts past 2^31 elements."""
    from graph_rewrite_system_b200.rotary import rotate_positions

    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("needs 10 GB")
    q, k, p = _case(10, 9, 2, 1, 64, BF16)
    room = torch.empty(9, (1 << 31) // 8 + 64, dtype=BF16, device=cuda_device)
    far = room[:, -128:].unflatten(1, (2, 64))
    far.copy_(q)
    f = _freq(64)
    got = rotate_positions(far, None, p.to(cuda_device), f.to(cuda_device), query_out=far)
    _check(got[0], q, p, f)


@pytest.mark.parametrize("far", [1000, 2 ** 45, 2 ** 62])
def test_steps_of_half_a_turn(cuda_device, far):
    """Frequencies whose step rounds to half a turn and whole ones, at positions where
    one unit of the step's last place would be seen."""
    pi = 3.141592653589793
    f = torch.tensor([pi, 5 * pi, 9 * pi, 3 * pi, -pi, -5 * pi, 2 * pi, 7 * pi],
                     dtype=torch.float64)
    q, k, p = _case(11, 30, 2, 1, 16, FP32, far, torch.int64)
    p[0], p[1] = far, -far
    got = _call(cuda_device, q, k, p, f)
    _check(got[0], q, p, f)
    _check(got[1], k, p, f)


def test_frequencies_of_many_turns(cuda_device):
    """Up to 2^60 radians a position; 1 / (2 pi) is held to 2^-108, which leaves them
    2^-40 of a turn at these positions."""
    f = torch.tensor([1e15, 2.0 ** 52 * 7, 1e17, -3e17, 2.0 ** 60, 1e9, 0.3, -1e16],
                     dtype=torch.float64)
    q, k, p = _case(12, 30, 2, 1, 16, FP32, 100)
    got = _call(cuda_device, q, k, p, f)
    _check(got[0], q, p, f)
