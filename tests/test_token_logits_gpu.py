"""Logit adjustment vs the fp64 oracle."""
from __future__ import annotations

import pytest
import torch

from oracle import grouped_attention as oracle

pytestmark = pytest.mark.gpu

BF16, FP32 = torch.bfloat16, torch.float32


def _case(seed, rows, vocab, history, dtype, *, bias="none", mask="none", ids=torch.int32):
    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn(rows, vocab, generator=g) * 4).to(dtype)
    kw = {}
    if history:
        kw["tokens"] = (vocab * torch.rand(rows, history, generator=g) ** 3).to(ids)
        kw["lengths"] = torch.randint(0, history + 1, (rows,), generator=g, dtype=torch.int32)
        kw["lengths"][0] = history
        kw["prompt_lengths"] = kw["lengths"] // 2
        kw["repetition"] = 1 + torch.rand(rows, generator=g)
        kw["presence"] = torch.randn(rows, generator=g)
        kw["frequency"] = torch.randn(rows, generator=g)
    if bias != "none":
        kw["bias"] = torch.randn(*((vocab,) if bias == "shared" else (rows, vocab)), generator=g)
    if mask != "none":
        words = -(-vocab // 32)
        shape = (words,) if mask == "shared" else (rows, words)
        kw["allowed"] = torch.randint(-2 ** 31, 2 ** 31, shape, generator=g).to(torch.int32)
        if mask == "row":
            kw["allowed"][-1] = 0
    return logits, kw


def _call(dev, logits, kw, **more):
    from graph_rewrite_system_b200.token_logits import adjust_logits

    kw = {n: v.to(dev) if isinstance(v, torch.Tensor) else v for n, v in kw.items()}
    return adjust_logits(logits.to(dev), **kw, **more)


def _check(got, logits, kw):
    """fp32 arithmetic: a quotient or product, two products and sums and a
    bias, each rounded relative to the terms; then the output's rounding."""
    exp = oracle.adjust_logits(logits, **kw)
    got = got.double().cpu()
    fill = ~torch.isfinite(exp) | ~torch.isfinite(got)
    assert torch.equal(torch.nan_to_num(got[fill], nan=7e77), torch.nan_to_num(exp[fill], nan=7e77))
    size = logits.double().abs() * 2
    if "tokens" in kw:
        count = kw["tokens"].shape[1]
        knob = lambda n: (kw[n].double().abs()[:, None] if isinstance(kw.get(n), torch.Tensor)
                          else abs(kw.get(n, 0.0)))
        size = size + knob("frequency") * count + knob("presence")
    if "bias" in kw:
        size = size + kw["bias"].double().abs()
    half = 2.0 ** -8 if logits.dtype == BF16 else 2.0 ** -24
    bound = 6 * 2.0 ** -24 * size + half * exp.abs() * 1.01
    assert ((got - exp).abs() <= bound)[~fill].all()


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("rows,vocab,history", [(1, 1, 1), (3, 31, 5), (2, 4096, 100),
                                                (2, 4097, 700), (5, 12345, 40), (4, 33, 0),
                                                (1, 40001, 2000), (70, 257, 9)])
@pytest.mark.parametrize("bias,mask", [("none", "none"), ("shared", "row"), ("row", "shared")])
def test_sizes(cuda_device, rows, vocab, history, dtype, bias, mask):
    logits, kw = _case(rows + vocab, rows, vocab, history, dtype, bias=bias, mask=mask)
    _check(_call(cuda_device, logits, kw), logits, kw)


@pytest.mark.parametrize("ids", [torch.int32, torch.int64])
def test_token_ids_outside_the_vocabulary_pad(cuda_device, ids):
    logits, kw = _case(1, 4, 300, 60, FP32, ids=ids)
    kw["tokens"][:, ::3] = -1
    kw["tokens"][:, 1::7] = 300
    kw["tokens"][2, 5] = 2 ** 31 - 1
    if ids == torch.int64:
        kw["tokens"][1, 7] = 2 ** 32 + 5
        kw["tokens"][1, 8] = -2 ** 63
    _check(_call(cuda_device, logits, kw), logits, kw)


def test_lengths_outside_the_history_are_cut(cuda_device):
    logits, kw = _case(2, 4, 300, 60, FP32)
    kw["lengths"] = torch.tensor([-5, 61, 2 ** 31 - 1, 0], dtype=torch.int32)
    kw["prompt_lengths"] = torch.tensor([3, -4, 2 ** 31 - 1, 9], dtype=torch.int32)
    _check(_call(cuda_device, logits, kw), logits, kw)


@pytest.mark.parametrize("knobs", [dict(), dict(repetition=1.3), dict(presence=0.7),
                                   dict(frequency=-0.4), dict(repetition=0.5, frequency=2.0)])
def test_scalar_penalties(cuda_device, knobs):
    logits, kw = _case(3, 3, 500, 90, FP32)
    kw = {"tokens": kw["tokens"], **knobs}
    kw["tokens"][0] = 17                        # one token 90 times
    _check(_call(cuda_device, logits, kw), logits, kw)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("fill", [-float("inf"), "lowest", -1e4])
def test_odd_values(cuda_device, dtype, fill):
    """Infinite, NaN and lowest logits, masked and not; an all-masked row."""
    logits, kw = _case(4, 3, 200, 30, dtype, mask="row", bias="shared")
    low = torch.finfo(dtype).min
    logits[:, ::5], logits[:, 1::5] = float("nan"), float("inf")
    logits[:, 2::5], logits[:, 3::10] = -float("inf"), low
    kw["bias"][::4] = 0
    kw["bias"][7] = -float("inf")
    kw["fill"] = low if fill == "lowest" else fill
    got = _call(cuda_device, logits, kw)
    exp = oracle.adjust_logits(logits, **kw)
    got, fine = got.double().cpu(), torch.isfinite(exp) & (exp.abs() < 3e38)
    # past the largest number both are infinite after rounding
    assert torch.equal(torch.isnan(got), torch.isnan(exp))
    assert torch.equal(torch.isposinf(got), torch.isposinf(exp.to(dtype)))
    assert torch.equal(torch.isneginf(got), torch.isneginf(exp.to(dtype)))
    assert ((got - exp).abs()[fine] <= 2.0 ** -7 * (1 + exp.abs())[fine]).all()
    assert (got[-1] == torch.tensor(kw["fill"], dtype=dtype).double()).all()


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_in_place_and_strided(cuda_device, dtype):
    from graph_rewrite_system_b200.token_logits import adjust_logits

    logits, kw = _case(5, 6, 1003, 64, dtype, mask="row", bias="row")
    got = _call(cuda_device, logits, kw)
    d = {n: v.to(cuda_device) for n, v in kw.items()}
    for pad, shift in ((0, 0), (5, 0), (5, 3), (1021, 1)):
        room = torch.full((6, 1003 + pad + shift), 9.0, dtype=dtype, device=cuda_device)
        rows = room[:, shift:shift + 1003]
        rows.copy_(logits)
        into = torch.full((6, 1003 + 8), 9.0, dtype=dtype, device=cuda_device)
        assert torch.equal(adjust_logits(rows, **d, out=into[:, 2:1005]), got)
        assert (into[:, :2] == 9).all() and (into[:, 1005:] == 9).all()
        assert adjust_logits(rows, **d, out=rows) is rows
        assert torch.equal(rows, got)
        assert (room[:, :shift] == 9).all() and (room[:, shift + 1003:] == 9).all()
    wide = torch.zeros(6, 70, dtype=torch.int32, device=cuda_device)
    wide[:, 3:67] = d["tokens"]
    d["tokens"] = wide[:, 3:67]
    d["allowed"] = torch.cat([d["allowed"], d["allowed"]], 1)[:, :32]
    assert torch.equal(adjust_logits(logits.to(cuda_device), **d), got)


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_far_and_shared_rows(cuda_device, dtype):
    """Rows that start past 2^31 elements, adjusted in place; and one row of
    logits, history and mask that every row shares by a stride of zero."""
    from graph_rewrite_system_b200.token_logits import adjust_logits

    logits, kw = _case(8, 3, 5003, 30, dtype, mask="row", bias="row")
    d = {n: v.to(cuda_device) for n, v in kw.items()}
    step = (1 << 30) + 16
    if torch.cuda.mem_get_info()[0] < 3 * step * dtype.itemsize + (1 << 30):
        pytest.skip("needs 14 GB")
    rows = torch.empty(3, step, dtype=dtype, device=cuda_device)[:, 5:5008]
    assert rows[2].data_ptr() - rows.data_ptr() > (1 << 31) * dtype.itemsize
    rows.copy_(logits)
    _check(adjust_logits(rows, **d, out=rows), logits, kw)
    one = {n: v[1:2].expand(3, -1) if n in ("tokens", "allowed") else v for n, v in kw.items()}
    d = {n: kw[n][1:2].to(cuda_device).expand(3, -1) if n in ("tokens", "allowed") else v
         for n, v in d.items()}
    got = adjust_logits(logits[:1].to(cuda_device).expand(3, -1), **d)
    _check(got, logits[:1].expand(3, -1), one)


def test_captured(cuda_device):
    from graph_rewrite_system_b200.token_logits import adjust_logits

    logits, kw = _case(6, 8, 2000, 50, FP32, mask="row")
    x = logits.to(cuda_device)
    d = {n: v.to(cuda_device) for n, v in kw.items()}
    adjust_logits(x, **d)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(adjust_logits(x, **d))
        graphs.append(g)
    logits, kw = _case(7, 8, 2000, 50, FP32, mask="row")
    x.copy_(logits)
    for n, v in kw.items():
        d[n].copy_(v)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s, g in zip(streams, graphs):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            g.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], outs[1])
    _check(outs[0], logits, kw)


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_histories_past_the_packed_counters(cuda_device, dtype):
    """2^14 tokens and more count in whole words; one token fills them all."""
    for history in (16383, 16384, 40000):
        logits, kw = _case(9, 2, 30001, history, dtype)
        kw["tokens"][1] = 5
        kw["lengths"][:] = history
        kw["prompt_lengths"][:] = 0
        _check(_call(cuda_device, logits, kw), logits, kw)


def test_many_rows(cuda_device):
    logits, kw = _case(8, 70000, 3, 2, FP32)
    got = _call(cuda_device, logits, kw)
    pick = torch.randperm(70000, generator=torch.Generator().manual_seed(1))[:300]
    _check(got[pick.to(got.device)], logits[pick], {n: v[pick] for n, v in kw.items()})
