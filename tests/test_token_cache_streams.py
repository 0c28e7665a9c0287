"""Where a TokenKVCache makes its memory and launches its kernels, on the CPU: torch's
stream and device calls are fakes that record the current device and stream."""
from __future__ import annotations

import pytest
import torch

BF16, E4M3 = torch.bfloat16, torch.float8_e4m3fn


class _Stream:
    def __init__(self, handle, device_index):
        self.cuda_stream, self.device_index = handle, device_index


class _Machine:
    """Two devices; `seen` holds (what, current device, its stream) of every torch call
    that touches memory, (name, device, launch's stream) of every launch."""

    def __init__(self):
        self.device, self.streams, self.seen = 0, {0: 50, 1: 60}, []

    def note(self, what):
        self.seen.append((what, self.device, self.streams[self.device]))

    def __getattr__(self, name):
        def launch(*args):
            self.seen.append((name, self.device, args[-1]))
            return 0
        if not name.startswith("grs_"):
            raise AttributeError(name)
        return launch


@pytest.fixture
def machine(monkeypatch):
    from graph_rewrite_system_b200 import _lib

    m = _Machine()

    class Use:
        def __init__(self, index, handle=None):
            self.index, self.handle = index, handle

        def __enter__(self):
            self.before = m.device, dict(m.streams)
            m.device = self.index
            if self.handle is not None:
                m.streams[self.index] = self.handle

        def __exit__(self, *exc):
            m.device, m.streams = self.before

    monkeypatch.setattr(torch.cuda, "device", lambda i: Use(i))
    monkeypatch.setattr(torch.cuda, "stream", lambda s: Use(s.device_index, s.cuda_stream))
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: _Stream(
        m.streams[m.device if device is None else device.index],
        m.device if device is None else device.index))
    monkeypatch.setattr(torch.cuda, "current_device", lambda: m.device)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda i: m.streams[i],
                        raising=False)
    monkeypatch.setattr(_lib, "current_device", lambda: m.device)
    monkeypatch.setattr(_lib, "lib", lambda: m)
    for name in ("empty", "zeros", "ones"):
        def make(*size, _real=getattr(torch, name), _name=name, **kw):
            assert kw.pop("device").index == 1
            m.note(_name)
            return _real(*size, **kw)
        monkeypatch.setattr(torch, name, make)
    for name in ("empty_like", "ones_like"):
        def like(t, _real=getattr(torch, name), _name=name, **kw):
            m.note(_name)
            return _real(t, **kw)
        monkeypatch.setattr(torch, name, like)
    for name in ("zero_", "tolist", "item", "amin", "to", "__rsub__"):
        def method(t, *args, _real=getattr(torch.Tensor, name), _name=name, **kw):
            m.note(_name)
            args = tuple(torch.device("cpu") if isinstance(a, torch.device) else a for a in args)
            return _real(t, *args, **kw)
        monkeypatch.setattr(torch.Tensor, name, method)
    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: 1)
    return m


def _everything(machine, dtype, elsewhere):
    """All of a cache's own calls, each with `elsewhere()` made current before it."""
    from graph_rewrite_system_b200.paged_cache import PrefixHandle
    from graph_rewrite_system_b200.token_cache import TokenKVCache

    elsewhere()
    cache = TokenKVCache(layers=2, capacity=8, page_size=4, heads=2, head_width=8,
                         device=torch.device("cuda", 1), dtype=dtype)
    rows, lengths = torch.arange(4, dtype=torch.int32).view(2, 2), torch.arange(
        2, dtype=torch.int32)
    cache._free_count[0] = 3
    for call in (cache.reset, lambda: cache.alloc_pages(3), lambda: cache.fork_device(rows, lengths),
                 lambda: cache.release_device(rows.long(), lengths.long()),
                 lambda: cache.release(PrefixHandle((1, 2), 7)),
                 lambda: cache.block_table([PrefixHandle((1, 2), 7)]), cache.check_status,
                 cache.status_tensor, cache.allocated_pages_tensor, lambda: cache.refcounts,
                 lambda: cache.free, lambda: cache.allocated_pages):
        before = len(machine.seen)
        elsewhere()
        call()
        assert len(machine.seen) > before
    return cache


@pytest.mark.parametrize("dtype", [BF16, E4M3])
def test_on_another_device_than_the_current(machine, dtype):
    def elsewhere():
        machine.device = 0

    _everything(machine, dtype, elsewhere)
    assert {"grs_cache_init", "grs_cache_fork", "grs_cache_alloc", "grs_cache_release"} <= {
        s[0] for s in machine.seen}
    assert {s[1:] for s in machine.seen} == {(1, 60)}, machine.seen


@pytest.mark.parametrize("device", [0, 1])
@pytest.mark.parametrize("dtype", [BF16, E4M3])
def test_under_another_stream_than_the_pinned(machine, dtype, device):
    from graph_rewrite_system_b200 import _lib

    def elsewhere():
        machine.device, machine.streams = device, {0: 50, 1: 60}

    machine.device, machine.streams = 1, {0: 50, 1: 77}
    with _lib.pinned_stream():
        _everything(machine, dtype, elsewhere)
    assert {s[1:] for s in machine.seen} == {(1, 77)}, machine.seen
