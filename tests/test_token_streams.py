"""The token operators under ``pinned_stream()``: on the CPU with fakes of torch's
stream calls, and on the GPU with a TokenKVCache."""
from __future__ import annotations

import pytest
import torch

from test_pinned_stream import fakes                      # noqa: F401

BF16, E4M3 = torch.bfloat16, torch.float8_e4m3fn


def _calls():
    from graph_rewrite_system_b200 import quantized_attention, rotary, token_cache

    z = lambda *s, dtype=BF16: torch.zeros(*s, dtype=dtype)
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)
    f = torch.ones(16, dtype=torch.float64)
    pages = dict(key_cache=z(5, 8, 2, 32, dtype=E4M3), value_cache=z(5, 8, 2, 32, dtype=E4M3),
                 key_scale=torch.ones(5, 2), value_scale=torch.ones(5, 2))
    return [
        (rotary, "grs_rotate_positions", rotary.rotate_positions,
         dict(query=z(3, 4, 32), key=z(3, 2, 32), positions=i(3), frequencies=f)),
        (token_cache, "grs_append_tokens", token_cache.append_tokens,
         dict(key=z(3, 2, 32), value=z(3, 2, 32), block_table=i(3, 2), lengths=i(3),
              query=z(3, 4, 32), frequencies=f, status=i(1), **pages)),
        (quantized_attention, "grs_quantized_attention", quantized_attention.quantized_attention,
         dict(query=z(3, 4, 32), block_table=i(3, 200), lengths=i(3), status=i(1), **pages)),
    ]


@pytest.mark.parametrize("which", [0, 1, 2])
def test_memory_comes_from_the_stream_of_the_launch(fakes, monkeypatch, which):   # noqa: F811
    from graph_rewrite_system_b200 import _lib
    from test_pinned_stream import _Stream

    module, name, call, args = _calls()[which]
    at, launched = [], []
    empty_like, new_empty = torch.empty_like, torch.Tensor.new_empty
    monkeypatch.setattr(torch, "empty_like", lambda *a, **k: (
        at.append(fakes["stream"].cuda_stream), empty_like(*a, **k))[1])
    monkeypatch.setattr(torch.Tensor, "new_empty", lambda *a, **k: (
        at.append(fakes["stream"].cuda_stream), new_empty(*a, **k))[1])
    monkeypatch.setattr(module, "_entry",
                        lambda t: launched.append(_lib.words_of(name).unpack(t)[-1]) or 0)
    with _lib.pinned_stream():
        fakes["stream"] = _Stream(12)
        call(**args)
        assert fakes["stream"].cuda_stream == 12
    assert launched == [11] and set(at) == {11}
    at.clear(), launched.clear()
    call(**args)
    assert launched == [12] and set(at) == {12}


def test_new_outputs_are_contiguous(fakes, monkeypatch):   # noqa: F811
    """Whatever the order of the inputs' dimensions."""
    for module, name, call, args in _calls():
        monkeypatch.setattr(module, "_entry", lambda t: 0)
        for q in (args["query"].transpose(0, 1).contiguous().transpose(0, 1),
                  torch.zeros(3, 9, 32, dtype=BF16)[:, :4],
                  torch.zeros(3, 1, 32, dtype=BF16).expand(3, 4, 32)):
            got = call(**{**args, "query": q})
            assert (got[0] if isinstance(got, tuple) else got).is_contiguous()


@pytest.mark.gpu
def test_a_cache_on_the_pinned_stream(cuda_device):
    """Fork, append, attention and release go to the pinned stream while another one
    is current and busy with memory that it has given back."""
    from graph_rewrite_system_b200 import _lib
    from graph_rewrite_system_b200.rotary import rotary_frequencies
    from graph_rewrite_system_b200.token_cache import TokenKVCache

    dev = cuda_device
    f = rotary_frequencies(64, device=dev)
    g = torch.Generator().manual_seed(3)
    qkv = torch.randn(10, 40, 12, 64, generator=g).to(BF16).to(dev)

    side = torch.cuda.Stream()

    def decode(call):
        cache = TokenKVCache(layers=1, capacity=300, page_size=4, heads=2, head_width=64,
                             device=dev, dtype=E4M3)
        table = call(lambda: cache.alloc_pages(40)).view(40, 1)
        lengths = torch.zeros(40, dtype=torch.int32, device=dev)
        outs = []
        for step in range(10):
            q, k, v = qkv[step].split([8, 2, 2], 1)
            held = lengths if step else lengths + 1       # the first pages hold no tokens
            children = call(lambda: cache.fork_device(table, lengths))
            call(lambda: cache.release_device(table, held))
            q = call(lambda: cache.append(0, k, v, children, lengths, source_table=table,
                                          query=q, frequencies=f))
            with_new = lengths + 1
            outs.append(call(lambda: cache.attend(0, q, children, with_new)))
            table, lengths = children, with_new
        call(cache.check_status)
        return outs

    expected = [o.clone() for o in decode(lambda fn: fn())]
    torch.cuda.synchronize()

    def elsewhere(fn):
        """The call under another current stream, which writes memory that it has freed."""
        with torch.cuda.stream(side):
            for _ in range(3):
                torch.zeros(1 << 20, device=dev).fill_(float("nan"))
            return fn()

    mine = torch.cuda.Stream()
    with torch.cuda.stream(mine), _lib.pinned_stream():
        got = [o.clone() for o in decode(elsewhere)]
    torch.cuda.synchronize()
    for a, b in zip(got, expected):
        assert torch.equal(a, b)
