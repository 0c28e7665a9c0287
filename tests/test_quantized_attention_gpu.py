"""Attention over 8-bit pages vs the fp64 oracle."""
from __future__ import annotations

import pytest
import torch

from oracle import token_cache as oracle

pytestmark = pytest.mark.gpu

BF16, FP32, E4M3 = torch.bfloat16, torch.float32, torch.float8_e4m3fn
CACHES = ("key_cache", "value_cache")


def _case(seed, *, batch, heads, kv_heads, width, longest, page=16, dtype=BF16, lengths=None,
          powers=(-9, -5)):
    g = torch.Generator().manual_seed(seed)
    columns = max(1, -(-longest // page))
    pages = max(3, batch * columns // 2)
    args = dict(query=torch.randn(batch, heads, width, generator=g).to(dtype))
    for name in ("key", "value"):
        x = torch.randn(pages, page, kv_heads, width, generator=g) * 60
        args[name + "_cache"] = x.clamp(-448, 448).to(E4M3)
        args[name + "_scale"] = torch.exp2(torch.randint(
            *powers, (pages, kv_heads), generator=g).float())
    args["block_table"] = torch.randint(0, pages, (batch, columns), generator=g, dtype=torch.int32)
    if lengths is None:
        lengths = torch.randint(0, longest + 1, (batch,), generator=g, dtype=torch.int32)
        lengths[0] = longest
    args["lengths"] = lengths
    return args


def _to(dev, args):
    return {n: t.to(dev) for n, t in args.items()}


def _call(dev, args, **kw):
    from graph_rewrite_system_b200.quantized_attention import quantized_attention

    return quantized_attention(**_to(dev, args), **kw)


def _check(got, args, scale=None, rows=None, generic=False):
    results = oracle.quantized_attention(**args, scale=scale)
    keys = max(1, int(args["lengths"].max()))
    bound = oracle.quantized_bound(results, args["query"].dtype, got.shape[2],
                                   min(keys, args["block_table"].shape[1] * args["key_cache"].shape[1]),
                                   args["value_scale"] if generic else None)
    off = (got.double().cpu() - results[0]).abs() / bound
    if rows is not None:
        off, got = off[rows], got[rows]
    assert torch.isfinite(got).all()
    assert float(off.max()) <= 1.0, f"error {float(off.max()):.3f} of the bound"


def _clean(dev):
    from graph_rewrite_system_b200.paged_attention import check_decode_status

    check_decode_status(dev)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("batch,longest", [
    (1, 1), (1, 2), (3, 15), (2, 16), (2, 17), (5, 64), (5, 65), (7, 129), (2, 1000), (1, 5000),
    (40, 300), (600, 33), (1100, 3)])
def test_sizes(cuda_device, batch, longest, dtype):
    args = _case(batch + longest, batch=batch, heads=8, kv_heads=2, width=64, longest=longest,
                 dtype=dtype)
    _check(_call(cuda_device, args), args)
    _clean(cuda_device)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (8, 8), (8, 1), (3, 1), (9, 1), (14, 2),
                                            (32, 2), (17, 1), (40, 1), (130, 1)])
@pytest.mark.parametrize("longest", [40, 700])
def test_head_groups(cuda_device, heads, kv_heads, dtype, longest):
    args = _case(heads, batch=5, heads=heads, kv_heads=kv_heads, width=32, longest=longest,
                 page=8, dtype=dtype)
    _check(_call(cuda_device, args), args)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("width", [1, 7, 8, 16, 24, 32, 33, 40, 56, 64, 72, 80, 96, 100, 112, 128,
                                   136, 160, 200, 256])
@pytest.mark.parametrize("heads", [4, 24])
def test_widths(cuda_device, width, dtype, heads):
    args = _case(width, batch=5, heads=heads, kv_heads=2, width=width, longest=90, dtype=dtype)
    _check(_call(cuda_device, args), args)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("page", [1, 2, 3, 7, 8, 16, 24, 32, 100, 1000])
def test_pages(cuda_device, page, dtype):
    """Pages that end inside a tile of tokens, sequences that share pages."""
    args = _case(page, batch=6, heads=4, kv_heads=2, width=64, longest=137, page=page, dtype=dtype)
    _check(_call(cuda_device, args), args)
    _clean(cuda_device)


# tiles enough for ranges of tiles over all sequences, whatever their lengths
STREAMS = [(40, 8, 8, 32, 3000), (30, 32, 8, 128, 1500), (1, 16, 8, 64, 40000),
           (1000, 8, 8, 32, 70), (1024, 8, 4, 64, 90), (1025, 4, 4, 64, 90),
           (12, 48, 4, 128, 3100), (9, 40, 4, 64, 4000), (9, 80, 4, 32, 5000),
           (14, 4, 4, 256, 2600), (9, 8, 8, 40, 3800), (9, 4, 4, 136, 6000)]


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("batch,heads,kv_heads,width,longest", STREAMS)
def test_many_tiles(cuda_device, batch, heads, kv_heads, width, longest, dtype):
    """Ragged sequences, empty ones and ones of a token among them, first and last."""
    g = torch.Generator().manual_seed(longest)
    lengths = torch.randint(0, longest + 1, (batch,), generator=g, dtype=torch.int32)
    lengths[torch.rand(batch, generator=g) < 0.2] = 0
    lengths[batch // 2] = longest
    if batch > 4:
        lengths[[1, batch - 2]] = 1
        lengths[[0, batch - 1]] = 0
    args = _case(batch, batch=batch, heads=heads, kv_heads=kv_heads, width=width, longest=longest,
                 page=8 if width == 64 else 24, lengths=lengths, dtype=dtype)
    got = _call(cuda_device, args)
    assert not got[(lengths == 0).to(cuda_device)].any()
    _check(got, args)
    _clean(cuda_device)


@pytest.mark.parametrize("lengths", [[0] * 30, [0] * 29 + [1], [1] + [0] * 29, [2000] * 30,
                                     [16] * 30, [17] * 30, [2000] + [0] * 28 + [2000]])
def test_lengths_that_leave_tables_empty(cuda_device, lengths):
    """Wide tables whose sequences fill them or do not."""
    args = _case(len(lengths), batch=30, heads=8, kv_heads=8, width=64, longest=2000,
                 lengths=torch.tensor(lengths, dtype=torch.int32))
    _check(_call(cuda_device, args), args)


def test_bad_pages_and_lengths_of_many_tiles(cuda_device):
    args = _case(9, batch=20, heads=8, kv_heads=8, width=64, longest=2000,
                 lengths=torch.full((20,), 2000, dtype=torch.int32))
    args["block_table"][2, 1] = 1 << 30
    args["block_table"][3, 100:] = -1
    for code, change in ((-2, None), (-7, {0: -5, 7: 2001, 19: 1 << 30})):
        if change:
            args["block_table"].clamp_(0, args["key_cache"].shape[0] - 1)
            for b, n in change.items():
                args["lengths"][b] = n
        status = torch.zeros(1, dtype=torch.int32, device=cuda_device)
        got = _call(cuda_device, args, status=status)
        assert int(status.item()) == code
        _check(got, args)
    more = dict(args, lengths=torch.ones(20, dtype=torch.int32))
    for name in ("key", "value"):
        more[name + "_cache"] = args[name + "_cache"][:0]
        more[name + "_scale"] = args[name + "_scale"][:0]
    status = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    assert not _call(cuda_device, more, status=status).any() and int(status.item()) == -2


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_empty_rows_are_zero(cuda_device, dtype):
    lengths = torch.tensor([0, 3, 0, 20, 0, 900], dtype=torch.int32)
    args = _case(1, batch=6, heads=4, kv_heads=2, width=64, longest=900, lengths=lengths,
                 dtype=dtype)
    got = _call(cuda_device, args)
    assert not got[[0, 2, 4]].any()
    _check(got, args)
    args["lengths"] = torch.zeros(6, dtype=torch.int32)
    assert not _call(cuda_device, args).any()
    assert _call(cuda_device, dict(args, query=args["query"][:0], lengths=lengths[:0],
                                   block_table=args["block_table"][:0])).shape == (0, 4, 64)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("factor", [1e-30, 1e-6, 30.0, 1e4])
def test_sizes_of_queries(cuda_device, factor, dtype):
    """Queries far from one, in heads of different sizes, scores to 1e5."""
    args = _case(2, batch=4, heads=8, kv_heads=2, width=64, longest=300, dtype=dtype)
    spread = torch.exp2(torch.arange(8.0) - 4)[:, None]
    args["query"] = (args["query"].float() * factor * spread).to(dtype)
    _check(_call(cuda_device, args), args)


@pytest.mark.parametrize("scale", [0.0, -0.03, 2.0, 1e-20])
def test_scale(cuda_device, scale):
    args = _case(3, batch=4, heads=4, kv_heads=2, width=32, longest=200, dtype=FP32)
    _check(_call(cuda_device, args, scale=scale), args, scale=scale)


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_value_scales_far_apart(cuda_device, dtype):
    """Pages of values 2^60 apart: the weights keep their digits for the small
    pages, where those carry the row, and rows of zeros count in the sum."""
    args = _case(4, batch=6, heads=4, kv_heads=2, width=32, longest=256, dtype=dtype)
    g = torch.Generator().manual_seed(5)
    args["value_scale"] = torch.exp2(torch.randint(-60, 1, args["value_scale"].shape,
                                                   generator=g).float())
    args["value_scale"][0], args["value_cache"][0] = 2.0 ** -118, torch.zeros(()).to(E4M3)
    _check(_call(cuda_device, args), args)
    # the largest page last, its tokens far below the others' scores
    args["lengths"][:] = 256
    args["value_scale"][:] = 2.0 ** -40
    args["block_table"][:, 15] = 1
    args["block_table"][:, :15] = 2
    args["value_scale"][1] = 1.0
    args["key_cache"][1] = (args["key_cache"][1].float() * 0).to(E4M3)
    args["query"] = (args["query"].float().abs() * 3).to(dtype)
    args["key_cache"][2] = args["key_cache"][2].float().abs().to(E4M3)
    _check(_call(cuda_device, args), args)


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_any_positive_scales(cuda_device, dtype):
    args = _case(6, batch=5, heads=4, kv_heads=2, width=64, longest=300, dtype=dtype)
    g = torch.Generator().manual_seed(7)
    for name in ("key_scale", "value_scale"):
        args[name] = 0.002 + torch.rand(args[name].shape, generator=g) / 50
    _check(_call(cuda_device, args), args, generic=True)


def test_every_code(cuda_device):
    """All finite codes, subnormal ones among them, as values and as keys."""
    codes = torch.arange(256, dtype=torch.uint8)
    codes[[127, 255]] = 0
    args = _case(8, batch=1, heads=1, kv_heads=1, width=256, longest=16, dtype=FP32, powers=(0, 1))
    args["block_table"] = torch.tensor([[0]], dtype=torch.int32)
    args["lengths"] = torch.tensor([1], dtype=torch.int32)
    args["value_cache"][0, 0, 0] = codes.view(E4M3)
    got = _call(cuda_device, args)
    # one key: its weight and the sum round alike, 2^-22 for the two parts
    exp = codes.view(E4M3).double()
    assert bool(((got[0, 0].double().cpu() - exp).abs() <= 2.0 ** -21 * exp.abs()).all())
    args["lengths"] = torch.tensor([16], dtype=torch.int32)
    args["key_cache"][0, :, 0] = codes.view(E4M3)
    args["query"] = args["query"] / 100
    _check(_call(cuda_device, args), args)


@pytest.mark.parametrize("width", [64, 33])
def test_bad_pages_and_lengths(cuda_device, width):
    args = _case(9, batch=8, heads=4, kv_heads=2, width=width, longest=48,
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


@pytest.mark.parametrize("width", [64, 33])
def test_no_pages(cuda_device, width):
    args = _case(10, batch=4, heads=4, kv_heads=2, width=width, longest=30)
    for pages, columns, lengths, code in ((0, 2, [0, 0, 0, 0], 0), (0, 2, [0, 3, 0, 32], -2),
                                          (5, 0, [0, 0, 0, 0], 0), (5, 0, [0, 0, 1, 0], -7)):
        more = dict(args, block_table=torch.zeros(4, columns, dtype=torch.int32),
                    lengths=torch.tensor(lengths, dtype=torch.int32))
        for name in ("key", "value"):
            more[name + "_cache"] = args[name + "_cache"][:pages]
            more[name + "_scale"] = args[name + "_scale"][:pages]
        status = torch.zeros(1, dtype=torch.int32, device=cuda_device)
        got = _call(cuda_device, more, status=status)
        assert int(status.item()) == code and not got.any()


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("width", [64, 33])
def test_bad_values_reach_only_their_sequence(cuda_device, dtype, width):
    """NaN behind a sequence's last token, in pages of no sequence and their
    scales, in another sequence's values and query."""
    args = _case(11, batch=6, heads=8, kv_heads=2, width=width, longest=48, dtype=dtype,
                 lengths=torch.tensor([0, 17, 40, 33, 5, 31], dtype=torch.int32))
    args["block_table"] = torch.arange(18, dtype=torch.int32).view(6, 3)
    for name in ("key", "value"):
        g = torch.Generator().manual_seed(len(name))
        args[name + "_cache"] = (torch.randn(20, 16, 2, width, generator=g) * 60).clamp(
            -448, 448).to(E4M3)
        args[name + "_scale"] = torch.full((20, 2), 2.0 ** -7)
    clean = {n: t.clone() for n, t in args.items()}
    nan = torch.tensor(127, dtype=torch.uint8)
    for name in CACHES:
        bits = args[name].view(torch.uint8)
        for b, n in enumerate(args["lengths"].tolist()):
            for t in range(n, 48):
                bits[3 * b + t // 16, t % 16] = nan
        bits[18:] = nan
    for name in ("key_scale", "value_scale"):
        args[name][18:] = float("nan")
        args[name][17] = float("nan")          # a page behind sequence 5's last token
    args["value_cache"].view(torch.uint8)[6, 0] = nan
    args["query"][4] = float("nan")
    got = _call(cuda_device, args)
    assert torch.isnan(got[2]).all() and torch.isnan(got[4]).all()
    _check(got, clean, rows=[0, 1, 3, 5])
    _clean(cuda_device)


def test_layouts(cuda_device):
    """A layer of stacked arenas, a slice of a projection, wider tables, K and V
    in one buffer, rows off 16 and off 8 bytes, a head expanded to two."""
    from graph_rewrite_system_b200.quantized_attention import quantized_attention

    dev = cuda_device
    args = _case(12, batch=10, heads=8, kv_heads=2, width=64, longest=400)
    got = _call(dev, args)
    _check(got, args)
    d = _to(dev, args)
    pool = d["key_cache"].shape[0]
    both = torch.zeros(2, pool, 16, 2, 2, 64, dtype=torch.uint8, device=dev)
    for i, name in enumerate(CACHES):
        both[1, :, :, i] = d[name].view(torch.uint8)
    d["key_cache"], d["value_cache"] = (both.view(E4M3)[1, :, :, i] for i in range(2))
    scales = torch.zeros(pool, 4, device=dev)
    scales[:, :2], scales[:, 2:] = d["key_scale"], d["value_scale"]
    d["key_scale"], d["value_scale"] = scales[:, :2], scales[:, 2:]
    d["query"] = torch.cat([d["query"], d["query"]], 1)[:, :8]
    table = torch.full((10, d["block_table"].shape[1] + 3), 1 << 20, dtype=torch.int32, device=dev)
    table[:, :-3] = d["block_table"]
    d["block_table"] = table[:, :-3]
    out = torch.zeros(8, 10, 64, dtype=BF16, device=dev).transpose(0, 1)
    assert quantized_attention(**d, out=out) is out and torch.equal(out, got)
    for shift in (1, 8):
        d = _to(dev, args)
        for name in CACHES:
            room = torch.zeros(d[name].numel() + shift, dtype=torch.uint8, device=dev)
            room[shift:] = d[name].view(torch.uint8).flatten()
            d[name] = room[shift:].view(E4M3).view(args[name].shape)
        room = torch.zeros(d["query"].numel() + 1, dtype=BF16, device=dev)
        room[1:] = d["query"].flatten()
        d["query"] = room[1:].view(args["query"].shape)
        _check(quantized_attention(**d), args)
    for name in CACHES:
        one = args[name].view(torch.uint8)[:, :, :1]
        args[name] = one.expand(-1, -1, 2, -1).view(E4M3)
        d[name] = one.to(dev).expand(-1, -1, 2, -1).view(E4M3)
    _check(quantized_attention(**d), args)


def test_new_tokens_of_one_sequence(cuda_device):
    """Several queries of a sequence: an expanded table, lengths one after another."""
    args = _case(13, batch=1, heads=4, kv_heads=2, width=64, longest=80)
    more = dict(args, query=torch.randn(9, 4, 64).to(BF16),
                block_table=args["block_table"].expand(9, -1),
                lengths=torch.arange(70, 79, dtype=torch.int32))
    _check(_call(cuda_device, more), more)


def test_far_pages(cuda_device):
    """A cache whose last page starts past 2^32 bytes."""
    pages = (1 << 32) // (16 * 8 * 128) + 2
    if torch.cuda.mem_get_info()[0] < 2 * pages * 16 * 8 * 128 + (1 << 30):
        pytest.skip("needs 9 GB")
    from graph_rewrite_system_b200.quantized_attention import quantized_attention

    args = _case(14, batch=3, heads=8, kv_heads=8, width=128, longest=70)
    d = _to(cuda_device, args)
    pool = args["key_cache"].shape[0]
    for name in ("key", "value"):
        big = torch.zeros(pages, 16, 8, 128, dtype=torch.uint8, device=cuda_device)
        big[-pool:] = d[name + "_cache"].view(torch.uint8)
        d[name + "_cache"] = big.view(E4M3)
        scale = torch.zeros(pages, 8, device=cuda_device)
        scale[-pool:] = d[name + "_scale"]
        d[name + "_scale"] = scale
    d["block_table"] += pages - pool
    _check(quantized_attention(**d), args)


@pytest.mark.parametrize("many", [False, True])
def test_captured_and_two_calls_at_once(cuda_device, many):
    """Two captured graphs replayed together and an eager call, sliced, each with
    a workspace of its own; results do not depend on the run."""
    from graph_rewrite_system_b200.quantized_attention import quantized_attention

    dev = cuda_device
    size = dict(batch=3, heads=8, kv_heads=2, width=64, longest=2500)
    if many:
        size = dict(batch=20, heads=8, kv_heads=8, width=64, longest=2500)
    first, second = _case(15, **size), _case(16, **size)
    d = _to(dev, first)
    eager = quantized_attention(**d)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(quantized_attention(**d))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for args in (second, first):
        for n, t in args.items():
            d[n].copy_(t)
        for s, g in zip(streams, graphs):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                g.replay()
                other = quantized_attention(**d)
        for s in streams:
            torch.cuda.current_stream().wait_stream(s)
        assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], other)
        _check(outs[0], args)
    assert torch.equal(outs[0], eager)


def test_empty_rows_past_31_bits(cuda_device):
    """A row without keys that has 2^31 elements is zeroed, between two that have keys
    (ranges of tiles; every head's output is the value of its only key)."""
    from graph_rewrite_system_b200.quantized_attention import quantized_attention

    heads, width = 1 << 24, 128
    if torch.cuda.mem_get_info()[0] < 5 * 2 * heads * width + 4 * heads * (width + 1) * 4:
        pytest.skip("needs 60 GB")
    dev = cuda_device
    query = torch.ones(1, 1, 1, dtype=BF16, device=dev).expand(2, heads, width).contiguous()
    codes = torch.ones(2, 3, 8, 1, width, device=dev).to(E4M3)
    scales = torch.ones(2, 3, 1, device=dev)
    for lengths in ([0, 1], [1, 0], [0, 0]):
        out = torch.full_like(query, 5.0)
        got = quantized_attention(
            query, codes[0], codes[1], scales[0], scales[1],
            torch.zeros(2, 200, dtype=torch.int32, device=dev),
            torch.tensor(lengths, dtype=torch.int32, device=dev), out=out)
        for row, length in zip(got, lengths):
            assert bool((row == float(length)).all())
        del out, got
    del query
    torch.cuda.empty_cache()
