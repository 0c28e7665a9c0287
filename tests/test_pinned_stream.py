"""``pinned_stream()`` and the operators that allocate: on the CPU with fakes of
torch's stream calls, and on the GPU."""
from __future__ import annotations

import threading

import pytest
import torch


class _Stream:
    def __init__(self, handle, device_index=-1):
        self.cuda_stream = handle
        self.device_index = device_index


@pytest.fixture
def fakes(monkeypatch):
    """Streams that are numbers: `now` holds the current one of the device that
    CPU tensors report (-1); torch.cuda.stream makes another current."""
    now = {"stream": _Stream(11)}

    class Use:
        def __init__(self, stream):
            self.stream = stream

        def __enter__(self):
            self.before, now["stream"] = now["stream"], self.stream

        def __exit__(self, *exc):
            now["stream"] = self.before

    from graph_rewrite_system_b200 import _lib

    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: now["stream"])
    monkeypatch.setattr(torch.cuda, "stream", Use)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream",
                        lambda i: now["stream"].cuda_stream if i == -1 else 100 + i, raising=False)
    monkeypatch.setattr(_lib, "current_device", lambda: -1)
    monkeypatch.setattr(_lib, "require_cuda", lambda *t: None)
    return now


def test_the_pin_is_its_devices(fakes):
    from graph_rewrite_system_b200 import _lib

    with _lib.pinned_stream():
        fakes["stream"] = _Stream(12)
        assert _lib.current_stream() == 11
        assert _lib.stream_on(-1) == 11
        assert _lib.stream_on(3) == 103      # another device's launches stay on it
    assert _lib.stream_on(-1) == 12


def test_the_pin_is_its_threads(fakes):
    from graph_rewrite_system_b200 import _lib

    seen = []
    with _lib.pinned_stream():
        fakes["stream"] = _Stream(12)
        thread = threading.Thread(target=lambda: seen.append(_lib.stream_on(-1)))
        thread.start()
        thread.join()
        assert _lib.stream_on(-1) == 11
    assert seen == [12]


def _calls():
    from graph_rewrite_system_b200 import prefix_attention, prompt_attention, token_logits

    z = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)
    status = torch.zeros(1, dtype=torch.int32)
    return [
        (prompt_attention, prompt_attention.prompt_attention,
         dict(query=z(6, 4, 32), key=z(6, 2, 32), value=z(6, 2, 32),
              offsets=torch.tensor([0, 6], dtype=torch.int32), status=status)),
        (prefix_attention, prefix_attention.shared_prefix_attention,
         dict(query=z(3, 4, 32), prefix_key=z(900, 2, 32), prefix_value=z(900, 2, 32),
              status=status)),
        (token_logits, token_logits.adjust_logits, dict(logits=z(3, 70))),
    ]


@pytest.mark.parametrize("which", [0, 1, 2])
def test_memory_comes_from_the_stream_of_the_launch(fakes, monkeypatch, which):
    """Under a pin of another stream than torch's current one, the output and the
    workspace are allocated with the pinned stream current: what the allocator
    hands out for the current one may still be in use there."""
    from graph_rewrite_system_b200 import _lib

    module, call, args = _calls()[which]
    at, launched = [], []
    empty_like, new_empty = torch.empty_like, torch.Tensor.new_empty
    monkeypatch.setattr(torch, "empty_like", lambda *a, **k: (
        at.append(fakes["stream"].cuda_stream), empty_like(*a, **k))[1])
    monkeypatch.setattr(torch.Tensor, "new_empty", lambda *a, **k: (
        at.append(fakes["stream"].cuda_stream), new_empty(*a, **k))[1])
    name = {0: "grs_prompt_attention", 1: "grs_shared_prefix_attention",
            2: "grs_adjust_logits"}[which]
    monkeypatch.setattr(module, "_entry",
                        lambda t: launched.append(_lib.words_of(name).unpack(t)[-1]) or 0)
    with _lib.pinned_stream():
        fakes["stream"] = _Stream(12)
        call(**args)
        assert fakes["stream"].cuda_stream == 12
    assert launched == [11] and set(at) == {11}
    at.clear(), launched.clear()
    call(**args)                              # and without a pin from the current one
    assert launched == [12] and set(at) == {12}


@pytest.mark.gpu
@pytest.mark.parametrize("which", [0, 1, 2])
def test_calls_under_another_stream_than_the_pinned(cuda_device, which):
    """The current stream still writes memory that it has given back while the
    call runs on the pinned one; the call's output and workspace are not that."""
    from graph_rewrite_system_b200 import _lib

    _, call, args = _calls()[which]
    g = torch.Generator().manual_seed(which)
    args = {n: torch.randn(t.shape, generator=g).to(t.dtype) if t.is_floating_point() else t
            for n, t in args.items()}
    args = {n: t.to(cuda_device) for n, t in args.items()}
    expected = call(**args)
    pinned, other = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(pinned):           # what is loaded and allocated first waits
        call(**args)
    with torch.cuda.stream(pinned), _lib.pinned_stream():
        with torch.cuda.stream(other):
            sizes = [1 << n for n in range(9, 22)]
            blocks = [torch.empty(n, dtype=torch.uint8, device=cuda_device) for n in sizes * 4]
            for block in blocks:
                block.fill_(1)
            torch.cuda.synchronize()
            torch.cuda._sleep(400_000_000)    # some 0.2 s
            for block in blocks:
                block.fill_(255)
            del blocks, block
            got = call(**args)
        assert not other.query()              # the fills are still to come
    torch.cuda.synchronize()
    assert torch.equal(got, expected)
