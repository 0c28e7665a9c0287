"""Decode attention behind a shared prefix vs the fp64 oracle."""
from __future__ import annotations

import pytest
import torch

from oracle import grouped_attention as oracle

pytestmark = pytest.mark.gpu

BF16, FP32 = torch.bfloat16, torch.float32


def _case(seed, *, batch, heads, kv_heads, width, prefix, max_len, page=16, dtype=BF16,
          current=True, lengths=None):
    g = torch.Generator().manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g).to(dtype)
    args = dict(query=rand(batch, heads, width), prefix_key=rand(prefix, kv_heads, width),
                prefix_value=rand(prefix, kv_heads, width))
    if max_len:
        columns = -(-max_len // page)
        pages = max(3, batch * columns // 2)
        args.update(key_cache=rand(pages, page, kv_heads, width),
                    value_cache=rand(pages, page, kv_heads, width),
                    block_table=torch.randint(0, pages, (batch, columns), generator=g,
                                              dtype=torch.int32))
        if lengths is None:
            lengths = torch.randint(0, max_len + 1, (batch,), generator=g, dtype=torch.int32)
            lengths[0] = 0
            lengths[-1] = max_len
        args["lengths"] = lengths
    if current:
        args.update(current_key=rand(batch, kv_heads, width),
                    current_value=rand(batch, kv_heads, width),
                    current_valid=torch.rand(batch, generator=g) > 0.3)
    return args


def _call(dev, args, **kw):
    from graph_rewrite_system_b200.prefix_attention import shared_prefix_attention

    return shared_prefix_attention(**{n: t.to(dev) for n, t in args.items()}, **kw)


def _check(got, args, scale=None):
    out, spread, reach = oracle.shared_prefix_attention(**args, scale=scale)
    keys = args["prefix_key"].shape[0] + 1
    if "lengths" in args:
        keys += int(args["lengths"].max().clamp(min=0))
    bound = oracle.attention_bound(out, spread, reach, got.dtype, got.shape[2], keys)
    worst = ((got.double().cpu() - out).abs() / bound).max()
    assert torch.isfinite(got).all()
    assert float(worst) <= 1.0, f"error {float(worst):.3f} of the bound"


def _clean(dev):
    from graph_rewrite_system_b200.paged_attention import check_decode_status

    check_decode_status(dev)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("batch,prefix,max_len", [
    (1, 0, 1), (1, 1, 0), (1, 129, 20), (5, 0, 40), (3, 0, 0), (9, 127, 1), (33, 128, 64),
    (64, 700, 0), (40, 381, 65), (7, 5000, 300), (2, 33, 1000), (9, 256, 30), (9, 257, 30),
    (1, 640, 5), (130, 384, 17), (33, 1025, 0), (2500, 64, 3), (600, 255, 9)])
def test_sizes(cuda_device, batch, prefix, max_len, dtype):
    args = _case(batch + prefix, batch=batch, heads=8, kv_heads=2, width=64, prefix=prefix,
                 max_len=max_len, dtype=dtype)
    _check(_call(cuda_device, args), args)
    _clean(cuda_device)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("heads,kv_heads", [(8, 8), (8, 1), (3, 1), (10, 2), (14, 2), (32, 2),
                                            (40, 1), (130, 1)])
@pytest.mark.parametrize("prefix", [200, 410])
def test_head_groups(cuda_device, heads, kv_heads, dtype, prefix):
    """A prefix that the pages' kernel reads itself, and a sliced one."""
    args = _case(heads, batch=19, heads=heads, kv_heads=kv_heads, width=32, prefix=prefix,
                 max_len=40, page=8, dtype=dtype)
    _check(_call(cuda_device, args), args)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("width", [1, 8, 16, 24, 33, 40, 64, 80, 96, 128, 160, 256])
@pytest.mark.parametrize("prefix", [150, 390])
def test_widths(cuda_device, width, dtype, prefix):
    args = _case(width, batch=11, heads=4, kv_heads=2, width=width, prefix=prefix, max_len=50,
                 dtype=dtype)
    _check(_call(cuda_device, args), args)


@pytest.mark.parametrize("page", [1, 3, 8, 16, 32, 100])
def test_pages(cuda_device, page):
    # pages that end inside a tile of keys, beams that share pages
    args = _case(page, batch=13, heads=8, kv_heads=2, width=64, prefix=100, max_len=137, page=page)
    _check(_call(cuda_device, args), args)
    _clean(cuda_device)


@pytest.mark.parametrize("batch,group,prefix", [(70, 4, 900), (300, 1, 640), (200, 3, 2100),
                                                (520, 2, 260)])
def test_wide_batches(cuda_device, batch, group, prefix):
    """More rows than one tile, with and without several prefix slices."""
    args = _case(batch, batch=batch, heads=2 * group, kv_heads=2, width=128, prefix=prefix,
                 max_len=33)
    _check(_call(cuda_device, args), args)


@pytest.mark.parametrize("width", [30, 32, 64, 100, 128, 256])
@pytest.mark.parametrize("group,prefix", [(2, 300), (3, 0), (5, 40), (9, 500)])
def test_fp32_groups_in_wide_batches(cuda_device, group, prefix, width):
    """More heads than SMs: a CTA takes four heads of a group, or what is left."""
    args = _case(group + width, batch=80, heads=2 * group, kv_heads=2, width=width,
                 prefix=prefix, max_len=45, dtype=FP32)
    _check(_call(cuda_device, args), args)


def test_empty_rows_are_zero(cuda_device):
    args = _case(1, batch=6, heads=4, kv_heads=2, width=64, prefix=0, max_len=20,
                 lengths=torch.tensor([0, 3, 0, 20, 0, 1], dtype=torch.int32))
    args["current_valid"] = torch.tensor([0, 0, 1, 1, 0, 0], dtype=torch.bool)
    got = _call(cuda_device, args)
    assert not got[0].any() and not got[4].any() and got[2].any()
    _check(got, args)


def test_large_scores_and_scale(cuda_device):
    args = _case(2, batch=20, heads=8, kv_heads=2, width=64, prefix=600, max_len=70)
    args["query"] = args["query"] * 9
    _check(_call(cuda_device, args), args)
    _check(_call(cuda_device, args, scale=-0.02), args, scale=-0.02)


def test_bad_pages_and_lengths(cuda_device):
    """Pages outside the cache are skipped, lengths beyond the table cut; both
    are reported and leave the other beams exact."""
    args = _case(3, batch=8, heads=8, kv_heads=2, width=64, prefix=64, max_len=48,
                 lengths=torch.full((8,), 48, dtype=torch.int32))
    args["block_table"][2, 1] = 1 << 30
    args["block_table"][3, 0] = -1
    for code, lengths in ((-2, None), (-7, torch.tensor([48, -3, 10, 48, 48, 49, 1 << 30, 2],
                                                        dtype=torch.int32))):
        if lengths is not None:
            args["lengths"] = lengths
            args["block_table"].clamp_(0, args["key_cache"].shape[0] - 1)
        status = torch.zeros(1, dtype=torch.int32, device=cuda_device)
        got = _call(cuda_device, args, status=status)
        assert int(status.item()) == code
        _check(got, args)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("prefix", [0, 40, 500])
def test_no_pages(cuda_device, prefix, dtype):
    """A cache without pages, and a table without columns: tokens that the
    lengths claim are reported and skipped."""
    args = _case(9, batch=4, heads=4, kv_heads=2, width=64, prefix=prefix, max_len=0, dtype=dtype)
    for pages, columns, lengths, code in ((0, 2, [0, 0, 0, 0], 0), (0, 2, [0, 3, 0, 32], -2),
                                          (0, 2, [0, 33, 0, 0], None), (5, 0, [0, 0, 0, 0], 0),
                                          (5, 0, [0, 0, 1, 0], -7), (0, 0, [0, -1, 0, 0], -7)):
        status = torch.zeros(1, dtype=torch.int32, device=cuda_device)
        more = dict(args, key_cache=torch.zeros(pages, 16, 2, 64, dtype=dtype),
                    value_cache=torch.zeros(pages, 16, 2, 64, dtype=dtype),
                    block_table=torch.zeros(4, columns, dtype=torch.int32),
                    lengths=torch.tensor(lengths, dtype=torch.int32))
        got = _call(cuda_device, more, status=status)
        _check(got, args)
        # either report of a beam with both faults
        assert int(status.item()) in ((code,) if code is not None else (-2, -7))


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("prefix", [100, 500])
def test_bad_values_reach_only_their_beam(cuda_device, dtype, prefix):
    """NaN in unused cache rows, in another beam's pages and query."""
    args = _case(4, batch=6, heads=8, kv_heads=2, width=64, prefix=prefix, max_len=40, dtype=dtype,
                 lengths=torch.tensor([0, 17, 40, 33, 5, 31], dtype=torch.int32))
    args["block_table"] = torch.arange(18, dtype=torch.int32).view(6, 3)
    clean = {n: t.clone() for n, t in args.items()}
    for name in ("key_cache", "value_cache"):
        cache = torch.full((20,) + tuple(args[name].shape[1:]), float("nan"), dtype=dtype)
        full = torch.zeros_like(cache)
        for b, n in enumerate(args["lengths"].tolist()):
            for t in range(n):
                row = torch.randn(cache.shape[2:], generator=torch.Generator().manual_seed(
                    97 * b + t + len(name))).to(dtype)
                cache[3 * b + t // 16, t % 16] = full[3 * b + t // 16, t % 16] = row
        args[name], clean[name] = cache, full
    args["value_cache"][3 * 2, 0] = float("nan")
    args["query"][4] = float("nan")
    got = _call(cuda_device, args)
    assert torch.isnan(got[2]).all() and torch.isnan(got[4]).all()
    keep = [0, 1, 3, 5]
    out, spread, reach = oracle.shared_prefix_attention(**clean)
    bound = oracle.attention_bound(out, spread, reach, dtype, 64, prefix + 41)
    assert float(((got.double().cpu() - out).abs() / bound)[keep].max()) <= 1.0


@pytest.mark.parametrize("prefix", [90, 700])
def test_layouts(cuda_device, prefix):
    """A layer of a PagedKVCache, one projection's slices, unaligned rows, one
    K/V head broadcast to two."""
    from graph_rewrite_system_b200.prefix_attention import shared_prefix_attention

    dev = cuda_device
    args = _case(5, batch=10, heads=8, kv_heads=2, width=64, prefix=prefix, max_len=30)
    got = _call(dev, args)
    d = {n: t.to(dev) for n, t in args.items()}
    qkv = torch.cat([d["query"], d["current_key"], d["current_value"]], 1)
    d["query"], d["current_key"], d["current_value"] = qkv.split([8, 2, 2], 1)
    stacked = torch.stack([torch.zeros_like(d["key_cache"]), d["key_cache"]])
    d["key_cache"] = stacked[1]
    table = torch.full((10, 5), 1 << 20, dtype=torch.int32, device=dev)
    table[:, :2] = d["block_table"]
    d["block_table"] = table[:, :2]
    pk = torch.cat([d["prefix_key"], d["prefix_value"]], 1)
    d["prefix_key"], d["prefix_value"] = pk.split([2, 2], 1)
    assert torch.equal(shared_prefix_attention(**d), got)
    for name in ("prefix_key", "prefix_value", "key_cache", "value_cache", "query"):
        room = torch.zeros(args[name].numel() + 1, dtype=BF16, device=dev)
        room[1:] = args[name].to(dev).reshape(-1)
        d[name] = room[1:].view(args[name].shape)
    _check(shared_prefix_attention(**d), args)
    for name in ("prefix_key", "prefix_value", "key_cache", "value_cache"):
        args[name] = args[name][..., :1, :].expand(*args[name].shape)
        d[name] = args[name][..., :1, :].to(dev).expand(*args[name].shape)
    _check(shared_prefix_attention(**d), args)


def test_far_pages(cuda_device):
    """A cache whose last page starts past 2^31 elements."""
    pages = (1 << 31) // (16 * 8 * 128) + 2
    if torch.cuda.mem_get_info()[0] < 2 * pages * 16 * 8 * 128 * 2 + (1 << 30):
        pytest.skip("needs 10 GB")
    from graph_rewrite_system_b200.prefix_attention import shared_prefix_attention

    args = _case(6, batch=3, heads=8, kv_heads=8, width=128, prefix=10, max_len=32)
    d = {n: t.to(cuda_device) for n, t in args.items()}
    for name in ("key_cache", "value_cache"):
        big = torch.empty(pages, 16, 8, 128, dtype=BF16, device=cuda_device)
        big[-3:] = d[name][:3]
        d[name] = big
    args["block_table"] %= 3
    d["block_table"] = (args["block_table"] + pages - 3).to(cuda_device)
    _check(shared_prefix_attention(**d), args)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("prefix", [250, 2100])
def test_far_prefix(cuda_device, prefix, dtype):
    """Prefix rows, and with the short prefix the beams' too, whose last start
    past 2^31 elements, all in one buffer."""
    from graph_rewrite_system_b200.prefix_attention import shared_prefix_attention

    step = (1 << 31) // (prefix - 2) // 64 * 64 + 128
    if torch.cuda.mem_get_info()[0] < prefix * step * dtype.itemsize + (1 << 30):
        pytest.skip("needs 10 GB")
    batch = min(prefix, 250)
    args = _case(7, batch=batch, heads=4, kv_heads=1, width=64, prefix=prefix, max_len=20,
                 dtype=dtype)
    buffer = torch.empty(prefix, step // 64, 64, dtype=dtype, device=cuda_device)
    assert buffer[-1].data_ptr() - buffer.data_ptr() > (1 << 31) * dtype.itemsize
    d, at = {n: t.to(cuda_device) for n, t in args.items()}, 0
    for name in ("query", "prefix_key", "prefix_value", "current_key", "current_value"):
        part = buffer[:args[name].shape[0], at:at + args[name].shape[1]]
        d[name] = part.copy_(args[name])
        at += args[name].shape[1]
    out = buffer[:batch, at:at + 4]
    _check(shared_prefix_attention(**d, out=out), args)


def test_captured_and_on_another_stream(cuda_device):
    from graph_rewrite_system_b200.prefix_attention import shared_prefix_attention

    dev = cuda_device
    size = dict(batch=24, heads=8, kv_heads=2, width=64, prefix=1500, max_len=50)
    first, second = _case(7, **size), _case(8, **size)
    d = {n: t.to(dev) for n, t in first.items()}
    eager = shared_prefix_attention(**d)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(shared_prefix_attention(**d))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for args in (second, first):
        for n, t in args.items():
            d[n].copy_(t)
        for s, g in zip(streams, graphs):     # both replays at once
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                g.replay()
                other = shared_prefix_attention(**d)
        for s in streams:
            torch.cuda.current_stream().wait_stream(s)
        assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], other)
        _check(outs[0], args)
    assert torch.equal(outs[0], eager)


def test_equals_paged_attention(cuda_device):
    """The framework's own shared-prefix decode at the layout both take."""
    from graph_rewrite_system_b200.paged_attention import paged_attention

    args = _case(9, batch=40, heads=8, kv_heads=8, width=32, prefix=381, max_len=64)
    d = {n: t.to(cuda_device) for n, t in args.items()}
    got = _call(cuda_device, args)
    q = d.pop("query")
    exp = paged_attention(q.unsqueeze(2), d["key_cache"], d["value_cache"], d["block_table"],
                          d["lengths"], current_key=d["current_key"],
                          current_value=d["current_value"], current_valid=d["current_valid"],
                          shared_key=d["prefix_key"], shared_value=d["prefix_value"]).squeeze(2)
    torch.testing.assert_close(got.float(), exp.float(), rtol=2e-2, atol=2e-2)


def test_two_calls_at_once(cuda_device):
    """Calls on two streams, each sliced with a workspace of its own."""
    from graph_rewrite_system_b200.prefix_attention import shared_prefix_attention

    cases = [_case(10 + i, batch=30, heads=8, kv_heads=2, width=64, prefix=3000 + 700 * i,
                   max_len=60) for i in range(2)]
    d = [{n: t.to(cuda_device) for n, t in c.items()} for c in cases]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(10):
        for s, x, o in zip(streams, d, outs):
            with torch.cuda.stream(s):
                o.append(shared_prefix_attention(**x))
    torch.cuda.synchronize()
    for c, o in zip(cases, outs):
        _check(o[0], c)
        assert all(torch.equal(y, o[0]) for y in o)
