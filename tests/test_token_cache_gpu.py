"""Appending keys and values to paged caches vs the fp64 oracle."""
from __future__ import annotations

import pytest
import torch

from oracle import token_cache as oracle

pytestmark = pytest.mark.gpu

BF16, FP32, E4M3 = torch.bfloat16, torch.float32, torch.float8_e4m3fn
KINDS = [(BF16, BF16), (FP32, FP32), (BF16, E4M3), (FP32, E4M3)]


def _freq(rotated):
    from graph_rewrite_system_b200.rotary import rotary_frequencies

    return rotary_frequencies(rotated, device="cpu")


def _case(seed, *, new=None, past, page=16, heads=4, kv_heads=2, width=64, rotated=None,
          dtype=BF16, pages=BF16, fork=False, tail=0, extra=0, interleaved=False, magnitude=1.0,
          query=True):
    """new: tokens per sequence (None: one each without offsets); past: cached
    tokens; fork: every sequence's last page comes from a page of its own."""
    g = torch.Generator().manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g).to(dtype)
    count = new or [1] * len(past)
    tokens = sum(count) + tail
    args = dict(key=rand(tokens, kv_heads, width), value=3 * rand(tokens, kv_heads, width),
                lengths=torch.tensor(past, dtype=torch.int32))
    if new is not None:
        bounds = [0]
        for n in new:
            bounds.append(bounds[-1] + n)
        args["offsets"] = torch.tensor(bounds, dtype=torch.int32)
    columns = max(1, max(-(-(p + n) // page) for p, n in zip(past, count))) + extra
    total = 2 * len(past) * columns + 3
    place = torch.randperm(total, generator=g).to(torch.int32)
    args["block_table"] = place[:len(past) * columns].view(len(past), columns).clone()
    if fork:
        args["source_table"] = place[len(past) * columns:2 * len(past) * columns].view(
            len(past), columns).clone()
    for name in ("key", "value"):
        if pages is E4M3:
            codes = torch.randint(0, 256, (total, page, kv_heads, width), generator=g,
                                  dtype=torch.uint8)
            codes[codes & 127 == 127] = 126          # no NaN
            args[name + "_cache"] = codes.view(E4M3)
            args[name + "_scale"] = torch.exp2(torch.randint(
                -9, -4, (total, kv_heads), generator=g).float())
        else:
            args[name + "_cache"] = rand(total, page, kv_heads, width)
    if rotated != 0:
        args["frequencies"] = _freq(rotated or width)
        args.update(interleaved=interleaved, magnitude=magnitude)
        if query:
            args["query"] = rand(tokens, heads, width)
    return args


def _to(dev, args):
    return {n: t.to(dev) if isinstance(t, torch.Tensor) else t for n, t in args.items()}


def _call(dev, args, **kw):
    """The caches after the call, on the CPU, and the query."""
    from graph_rewrite_system_b200.token_cache import append_tokens

    d = _to(dev, args)
    kw.setdefault("status", torch.zeros(1, dtype=torch.int32, device=dev))
    query = append_tokens(**d, **kw)
    return {n: t.cpu() for n, t in d.items() if isinstance(t, torch.Tensor)}, query


def _spacing(x):
    """Distance of e4m3 values at x."""
    e = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6)))
    return torch.exp2(e - 3)


def _bits(t):
    return t.view(torch.uint8) if t.dtype is E4M3 else t


def _check(after, query, args, code=None):
    exp = oracle.append_tokens(**args)
    dtype = args["key"].dtype
    if "query" in exp:
        out, reach = exp["query"]
        assert bool(((query.double().cpu() - out).abs()
                     <= oracle.turn_bound(out, reach, dtype)).all())
    for name in ("key", "value"):
        cache, fresh, real, reach, scale = exp[name]
        got = after[name + "_cache"]
        # what is not new: kept rows as the oracle moves them, all else as it was
        old = ~fresh
        assert torch.equal(_bits(got)[old], _bits(cache)[old]), name
        x, real, reach = got[fresh].double(), real[fresh], reach[fresh]
        if scale is None:
            assert bool(((x - real).abs() <= oracle.turn_bound(real, reach, got.dtype)).all())
            continue
        assert torch.equal(after[name + "_scale"], scale), name
        # nearest code, at most 448, within the error of the fp32 rotation
        bad = ~torch.isfinite(real)
        assert torch.equal(torch.isnan(x), bad)
        real, x, reach = real[~bad].clamp(-448, 448), x[~bad], reach[~bad]
        off = (x - real).abs()
        near = 0.5 * _spacing(torch.maximum(real.abs(), x.abs())) + 9 * 2.0 ** -24 * reach
        assert bool((off <= near * (1 + 2.0 ** -20)).all()), name
        if name == "value":                           # no arithmetic: the very codes
            assert torch.equal(x, oracle.to_e4m3(real.float()).double())
    return exp


@pytest.mark.parametrize("dtype,pages", KINDS)
@pytest.mark.parametrize("fork", [False, True])
@pytest.mark.parametrize("past", [[0], [15], [16], [37, 0, 5, 16, 31], [3] * 40])
def test_one_token_each(cuda_device, past, fork, dtype, pages):
    args = _case(len(past), past=past, dtype=dtype, pages=pages, fork=fork)
    _check(*_call(cuda_device, args), args)


@pytest.mark.parametrize("dtype,pages", KINDS)
@pytest.mark.parametrize("new,past", [
    ([1], [0]), ([40], [0]), ([5, 0, 17, 1, 0], [0, 7, 30, 16, 0]), ([2] * 33, [15] * 33),
    ([700], [9]), ([100, 3, 250], [16, 1, 100]), ([0, 0, 1], [4, 0, 0])])
def test_prompts(cuda_device, new, past, dtype, pages):
    args = _case(sum(new), new=new, past=past, dtype=dtype, pages=pages, fork=sum(new) % 2 == 0,
                 interleaved=True, magnitude=1.2)
    _check(*_call(cuda_device, args), args)


@pytest.mark.parametrize("pages", [BF16, E4M3])
@pytest.mark.parametrize("page", [1, 2, 3, 8, 17, 64, 300])
def test_pages(cuda_device, page, pages):
    """Pages that end inside a chunk of rows, and of more rows than a chunk."""
    new, past = [5, 33, 1, 0, 400], [0, page - 1, page, 2 * page + 1, 7]
    args = _case(page, new=new, past=past, page=page, pages=pages, width=32, fork=page % 2 == 0)
    _check(*_call(cuda_device, args), args)


@pytest.mark.parametrize("dtype,pages", KINDS)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("width,rotated", [(1, 0), (2, 2), (7, 4), (8, 8), (32, 0), (33, 30),
                                           (40, 40), (40, 20), (64, 32), (96, 48), (128, 128),
                                           (256, 256), (256, 100)])
def test_widths(cuda_device, width, rotated, interleaved, dtype, pages):
    args = _case(width, new=[19, 1], past=[6, 3], width=width, rotated=rotated, dtype=dtype,
                 pages=pages, fork=True, interleaved=interleaved)
    _check(*_call(cuda_device, args), args)


@pytest.mark.parametrize("pages", [BF16, E4M3])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (8, 8), (6, 2), (70, 1), (40, 20)])
def test_heads(cuda_device, heads, kv_heads, pages):
    args = _case(heads, new=[3, 20], past=[2, 0], heads=heads, kv_heads=kv_heads, width=32,
                 pages=pages)
    _check(*_call(cuda_device, args), args)


def test_positions_and_no_query(cuda_device):
    for ids in (torch.int32, torch.int64):
        args = _case(1, past=[5, 9, 0], dtype=FP32, pages=FP32)
        args["positions"] = torch.tensor([1000000, -3, 7], dtype=ids)
        _check(*_call(cuda_device, args), args)
        args = _case(2, past=[5, 9, 0], pages=E4M3, query=False)
        args["positions"] = torch.tensor([100, 2, 7], dtype=ids)
        after, query = _call(cuda_device, args)
        assert query is None
        _check(after, None, args)


def test_scales_grow_and_stay(cuda_device):
    """Token by token: a scale grows with the largest value, the rows that are
    there move with it, and never shrinks inside a page; a new page starts anew."""
    g = torch.Generator().manual_seed(3)
    args = _case(4, past=[0, 0], page=4, pages=E4M3, rotated=0, width=32)
    args["block_table"] = torch.tensor([[2, 5, 1], [7, 0, 3]], dtype=torch.int32)
    sizes = [1.0, 300.0, 1e-3, 9e4, 1e-30, 5.0, 0.0, 1e4, 2e38]
    seen = []
    for t, size in enumerate(sizes):
        args["lengths"] = torch.tensor([t, t], dtype=torch.int32)
        args["key"] = (torch.randn(2, 2, 32, generator=g) * size).to(BF16)
        args["value"] = (torch.randn(2, 2, 32, generator=g) * size / 7).to(BF16)
        after, _ = _call(cuda_device, args)
        _check(after, None, args)
        args = {n: after.get(n, x) for n, x in args.items()}
        seen.append(float(args["key_scale"][[2, 5, 1][t // 4], 0]))
    assert seen[0] < seen[1] == seen[2] < seen[3] and seen[4] < seen[5] == seen[6] < seen[7]


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_borders_of_scales(cuda_device, dtype):
    """Largest values at, just below and just above 448 powers of two, the
    extremes of the scale's range, and rows of zeros."""
    top = [448.0, 450.0, 446.0, 3.5, 3.515625, 0.0, 1e-38, 448 * 2.0 ** -118, 449 * 2.0 ** -118,
           2.0 ** 127, 448 * 2.0 ** 119, 3.3e38]
    args = _case(5, past=[0] * len(top), dtype=dtype, pages=E4M3, rotated=0, width=16)
    for name in ("key", "value"):
        for b, x in enumerate(top):
            args[name][b] = torch.linspace(-1, 1, 16) * x
    _check(*_call(cuda_device, args), args)


@pytest.mark.parametrize("rotated", [0, 32])
def test_infinite_and_nan_values(cuda_device, rotated):
    """Held as NaN, in their own pair, and no part of a scale."""
    args = _case(6, new=[20, 3], past=[3, 0], pages=E4M3, width=64, rotated=rotated,
                 dtype=FP32)
    clean = {n: t.clone() if isinstance(t, torch.Tensor) else t for n, t in args.items()}
    for name in ("key", "value"):
        args[name][2, 0, 40] = float("inf")
        args[name][7, 1, 3] = float("nan")
        args[name][8, 0, 50] = float("-inf")
    after, query = _call(cuda_device, args)
    _check(after, query, args)
    same, _ = _call(cuda_device, clean)
    differ = _bits(after["value_cache"]) != _bits(same["value_cache"])
    assert int(differ.sum()) == 3


def test_bf16_pages_hold_what_came(cuda_device):
    args = _case(7, new=[9], past=[5], rotated=0, width=40)
    args["value"][3, 1, 7] = float("nan")
    args["key"][2, 0, 0] = float("-inf")
    after, _ = _call(cuda_device, args)
    slot = [int(args["block_table"][0, t // 16]) for t in range(5, 14)]
    row = [t % 16 for t in range(5, 14)]
    for name in ("key", "value"):
        got, x = after[name + "_cache"][slot, row], args[name]
        assert torch.equal(torch.isnan(got), torch.isnan(x))
        assert torch.equal(got[~torch.isnan(x)], x[~torch.isnan(x)])


@pytest.mark.parametrize("pages", [BF16, E4M3])
def test_bad_pages_and_lengths(cuda_device, pages):
    """Reported; their tokens are not written, the others are exact, queries turn."""
    for case in range(5):
        args = _case(8, new=[4, 30, 2, 6], past=[3, 10, 0, 20], pages=pages, fork=True)
        code = -2
        if case == 0:
            args["block_table"][1, 1] = 1 << 30
        elif case == 1:
            args["block_table"][0, 0] = -1
        elif case == 2:                       # kept rows cannot come: new ones still do
            args["source_table"][0, 0] = 1 << 20
        elif case == 3:
            args["lengths"][3], code = 1 << 29, -7
        else:
            args["lengths"][1], code = 33, -7
        status = torch.zeros(1, dtype=torch.int32, device=cuda_device)
        after, query = _call(cuda_device, args, status=status)
        assert int(status.item()) == code, case
        exp = oracle.append_tokens(**args)
        if case == 2 and pages is not E4M3:
            assert int(args["block_table"][0, 0]) >= 0
        _check(after, query, args)
        assert "query" in exp
    args = _case(9, past=[3, 4], pages=pages, extra=1)
    args["lengths"][0] = -1
    status = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    after, _ = _call(cuda_device, args, status=status)
    assert int(status.item()) == -7
    args["lengths"][0] = 1 << 30
    args.pop("query")
    exp = oracle.append_tokens(**args)
    for name in ("key", "value"):
        keep = ~exp[name][1]
        assert torch.equal(_bits(after[name + "_cache"])[keep], _bits(exp[name][0])[keep])


@pytest.mark.parametrize("pages", [BF16, E4M3])
@pytest.mark.parametrize("offsets", [[0, 5, 3, 9], [4, 4, 9, 12], [-7, 2, 40, 12], [9, 0, 0, 12],
                                     [0, 1 << 30, -(1 << 30), 3], [12, 12, 12, 12]])
def test_offsets_that_are_no_packing(cuda_device, offsets, pages):
    """Nothing outside the sequences' pages is written, whatever the offsets hold."""
    args = _case(10, new=[4, 4, 4], past=[3, 0, 17], pages=pages, extra=2)
    args["offsets"] = torch.tensor(offsets, dtype=torch.int32)
    before = {n: t.clone() for n, t in args.items() if isinstance(t, torch.Tensor)}
    after, query = _call(cuda_device, args)
    own = set(args["block_table"].flatten().tolist())
    others = [p for p in range(args["key_cache"].shape[0]) if p not in own]
    for name in ("key_cache", "value_cache"):
        assert torch.equal(_bits(after[name])[others], _bits(before[name])[others])
    for name in ("key", "value", "query", "block_table", "lengths", "offsets"):
        assert torch.equal(after[name], before[name])


@pytest.mark.parametrize("tail", [1, 90])
def test_rows_of_no_sequence(cuda_device, tail):
    """Padding behind the last sequence: NaN reaches nothing, query rows are zero
    in a new output and left in a given one."""
    args = _case(11, new=[3, 18], past=[1, 14], tail=tail, pages=E4M3)
    for name in ("query", "key", "value"):
        args[name][-tail:] = float("nan")
    args["offsets"] += 0
    after, query = _call(cuda_device, args)
    assert not query[-tail:].any()
    out = torch.full(args["query"].shape, 5.0, dtype=BF16, device=cuda_device)
    again, same = _call(cuda_device, args, query_out=out)
    assert same is out and bool((out[-tail:] == 5.0).all())
    assert torch.equal(out[:-tail], query[:-tail])
    for name in ("key_cache", "value_cache"):
        assert not torch.isnan(after[name].float()).any()
        assert torch.equal(_bits(after[name]), _bits(again[name]))
    for x in ("query", "key", "value"):
        args[x][-tail:] = 0
    _check(after, query, args)


def test_rows_past_31_bits(cuda_device):
    """A token of no sequence whose query row has 2^31 elements is zeroed."""
    from graph_rewrite_system_b200.token_cache import append_tokens

    heads, width = 1 << 24, 128
    if torch.cuda.mem_get_info()[0] < 3 * 2 * heads * width:
        pytest.skip("needs 13 GB")
    query = torch.ones(1, heads, width, dtype=BF16, device=cuda_device)
    key = torch.ones(1, 1, width, dtype=BF16, device=cuda_device)
    pages = torch.zeros(2, 3, 16, 1, width, dtype=BF16, device=cuda_device)
    none = torch.zeros(0, dtype=torch.int32, device=cuda_device)
    used = torch.ones_like(query)             # its memory serves the next output
    del used
    turned = append_tokens(key, key, pages[0], pages[1], none.view(0, 2), none,
                           offsets=torch.zeros(1, dtype=torch.int32, device=cuda_device),
                           frequencies=_freq(width).to(cuda_device), query=query)
    assert turned.shape == query.shape and not turned.any()
    assert not pages.any()


def test_narrow_source_table(cuda_device):
    """The parents' table ends where their tokens do; kept rows that it does not hold
    are reported, the new ones written."""
    args = _case(21, past=[3, 20, 16, 35], pages=E4M3, fork=True)
    wide = args["source_table"]
    args["source_table"] = torch.cat([wide, torch.full((4, 1), -5, dtype=torch.int32)], 1)[:, :3]
    _check(*_call(cuda_device, args), args)
    d = dict(args, source_table=wide[:, :2].contiguous())
    status = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    after, query = _call(cuda_device, d, status=status)
    assert int(status.item()) == -2
    args["source_table"][3, 2] = -1           # as a page outside the cache
    _check(after, query, args)


def test_no_tokens_and_no_pages(cuda_device):
    args = _case(12, new=[0, 0], past=[3, 0], pages=E4M3)
    after, query = _call(cuda_device, args)
    assert query.shape == (0, 4, 64)
    for name in ("key_cache", "value_cache"):
        assert torch.equal(_bits(after[name]), _bits(args[name]))
    args = _case(13, new=[2, 1], past=[3, 0], pages=E4M3)
    for name in ("key", "value"):
        args[name + "_cache"] = args[name + "_cache"][:0]
        args[name + "_scale"] = args[name + "_scale"][:0]
    status = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    after, query = _call(cuda_device, args, status=status)
    assert int(status.item()) == -2
    _check(after, query, args)
    # all tokens behind no sequence
    args = _case(14, new=[0], past=[3], tail=5)
    after, query = _call(cuda_device, args)
    assert not query.any()


def test_layouts(cuda_device):
    """A layer of stacked arenas, scales of a layer, slices of one projection in
    place, rows off 16 bytes, K and V in one buffer."""
    from graph_rewrite_system_b200.token_cache import append_tokens

    dev = cuda_device
    for pages in (BF16, E4M3):
        args = _case(15, new=[9, 30], past=[7, 0], pages=pages, fork=True)
        after, query = _call(dev, args)
        d = _to(dev, args)
        pool = d["key_cache"].shape[0]
        bits = torch.uint8 if pages is E4M3 else BF16
        both = torch.zeros(2, pool, 16, 2, 2, 64, dtype=bits, device=dev)
        both[1, :, :, 0], both[1, :, :, 1] = _bits(d["key_cache"]), _bits(d["value_cache"])
        d["key_cache"], d["value_cache"] = (both.view(pages)[1, :, :, i] for i in range(2))
        if pages is E4M3:
            scales = torch.zeros(pool, 4, device=dev)
            scales[:, :2], scales[:, 2:] = d["key_scale"], d["value_scale"]
            d["key_scale"], d["value_scale"] = scales[:, :2], scales[:, 2:]
        qkv = torch.cat([d["query"], d["key"], d["value"]], 1)
        d["query"], d["key"], d["value"] = qkv.split([4, 2, 2], 1)
        got = append_tokens(**d, query_out=d["query"])
        assert torch.equal(got, query)
        for name in ("key", "value"):
            assert torch.equal(_bits(d[name + "_cache"].contiguous()).cpu(),
                               _bits(after[name + "_cache"]))
            if pages is E4M3:
                assert torch.equal(d[name + "_scale"].cpu(), after[name + "_scale"])
        assert not both[0].any()
        for shift in (1, 4):                  # pieces of one element, of 8 bytes
            d = _to(dev, args)
            for name in ("query", "key", "value", "key_cache", "value_cache"):
                x = _bits(d[name])
                room = torch.zeros(x.numel() + shift, dtype=x.dtype, device=dev)
                room[shift:] = x.flatten()
                d[name] = room[shift:].view(d[name].dtype).view(x.shape)
            assert torch.equal(append_tokens(**d), query)
            for name in ("key_cache", "value_cache"):
                assert torch.equal(_bits(d[name]).cpu(), _bits(after[name]))


def test_far_pages(cuda_device):
    """A cache whose last page starts past 2^31 elements."""
    pages = (1 << 31) // (16 * 8 * 128) + 2
    if torch.cuda.mem_get_info()[0] < 2 * pages * 16 * 8 * 128 + (1 << 30):
        pytest.skip("needs 5 GB")
    args = _case(16, new=[20, 1], past=[3, 14], heads=8, kv_heads=8, width=128, pages=E4M3)
    pool = args["key_cache"].shape[0]
    d = _to(cuda_device, args)
    from graph_rewrite_system_b200.token_cache import append_tokens

    for name in ("key", "value"):
        big = torch.zeros(pages, 16, 8, 128, dtype=torch.uint8, device=cuda_device)
        big[-pool:] = _bits(d[name + "_cache"])
        d[name + "_cache"] = big.view(E4M3)
        scale = torch.zeros(pages, 8, device=cuda_device)
        scale[-pool:] = d[name + "_scale"]
        d[name + "_scale"] = scale
    d["block_table"] += pages - pool
    query = append_tokens(**d)
    after = {n: d[n][-pool:].cpu() if "cache" not in n else _bits(d[n])[-pool:].cpu().view(E4M3)
             for n in ("key_cache", "value_cache", "key_scale", "value_scale")}
    _check(after, query, args)


@pytest.mark.parametrize("pages", [BF16, E4M3])
def test_captured_and_on_another_stream(cuda_device, pages):
    """Two captured graphs and an eager call on a side stream, each into caches of
    its own, with inputs that change between replays."""
    from graph_rewrite_system_b200.token_cache import append_tokens

    dev = cuda_device
    size = dict(new=[5, 30, 1], past=[3, 16, 0], pages=pages, fork=True)
    first, second = _case(17, **size), _case(18, **size)
    names = ("key_cache", "value_cache", "key_scale", "value_scale")
    d = [_to(dev, first) for _ in range(3)]
    append_tokens(**_to(dev, first))
    graphs, outs = [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(append_tokens(**d[i]))
        graphs.append(g)
    for args in (second, first):
        for x in d:
            for n, t in args.items():
                if isinstance(t, torch.Tensor):
                    x[n].copy_(t)
        streams = [torch.cuda.Stream() for _ in range(3)]
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        with torch.cuda.stream(streams[2]):
            other = append_tokens(**d[2])
        for s in streams:
            torch.cuda.current_stream().wait_stream(s)
        assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], other)
        after = [{n: x[n].cpu() for n in names if n in x} for x in d]
        for x in after[1:]:
            assert all(torch.equal(_bits(x[n]), _bits(after[0][n])) for n in x)
        _check(after[0], outs[0], args)


def test_wide_batch(cuda_device):
    """More sequences than a round of the search among the offsets has probes,
    most of them empty."""
    g = torch.Generator().manual_seed(20)
    new = (torch.randint(0, 40, (1500,), generator=g) * (torch.rand(1500, generator=g) < 0.1)).tolist()
    past = torch.randint(0, 30, (1500,), generator=g).tolist()
    args = _case(19, new=new, past=past, heads=1, kv_heads=1, width=16, page=4, pages=E4M3)
    _check(*_call(cuda_device, args), args)
