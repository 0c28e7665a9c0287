"""Sizes past what the kernels' 32-bit indexes hold are refused, on the CPU: the
wrappers' checks (nothing is launched before them) and the C ABI's (which return
before any CUDA call)."""
from __future__ import annotations

import pytest
import torch


@pytest.fixture
def lifted(monkeypatch):
    from graph_rewrite_system_b200 import _lib

    def nothing(*a):
        raise AssertionError("a launch was reached")

    monkeypatch.setattr(_lib, "require_cuda", lambda *t: None)
    monkeypatch.setattr(_lib, "current_device", lambda: -1)
    monkeypatch.setattr(_lib, "lib", nothing)
    monkeypatch.setattr(_lib, "stream_on", nothing)


def _z(*shape):
    return torch.zeros(*shape, dtype=torch.bfloat16)


STATUS = torch.zeros(1, dtype=torch.int32)


def test_sequences(lifted):
    """The search among the offsets adds two places: they stay below 2^30."""
    from graph_rewrite_system_b200.prompt_attention import prompt_attention

    offsets = torch.empty((1 << 30) + 1, dtype=torch.int32, device="meta")
    with pytest.raises(ValueError, match="2\\^30"):
        prompt_attention(_z(6, 4, 32), _z(6, 2, 32), _z(6, 2, 32), offsets, status=STATUS)


def test_heads(lifted):
    from graph_rewrite_system_b200.prefix_attention import shared_prefix_attention
    from graph_rewrite_system_b200.prompt_attention import prompt_attention

    query = _z(1, 1, 1).expand(1, 1 << 30, 1)
    with pytest.raises(ValueError, match="2\\^30"):
        prompt_attention(query, _z(1, 1, 1), _z(1, 1, 1), torch.zeros(2, dtype=torch.int32),
                         status=STATUS)
    with pytest.raises(ValueError, match="2\\^30"):
        shared_prefix_attention(query, _z(9, 1, 1), _z(9, 1, 1), status=STATUS)


def test_c_abi():
    from graph_rewrite_system_b200 import _lib

    lib, far = _lib.lib(), 1 << 30
    prompt = dict(dtype=0, q=256, q_st=1, q_sh=1, k=256, k_st=1, k_sh=1, v=256, v_st=1, v_sh=1,
                  offsets=256, sequences=1, out=256, o_st=1, o_sh=1, tokens=1, heads=4, kv=2,
                  width=32, scale=1.0, clear=0, status=None, stream=None)
    prefix = dict(dtype=0, q=256, q_sb=1, q_sh=1, pk=256, pk_st=1, pk_sh=1, pv=256, pv_st=1,
                  pv_sh=1, n=300, kc=256, vc=256, kc_sp=1, kc_st=1, kc_sh=1, bt=256, bt_s=1,
                  blocks=1, lengths=256, pages=1, page=16, ck=None, cv=None, ck_sb=0, ck_sh=0,
                  valid=None, out=256, o_sb=1, o_sh=1, batch=2, heads=4, kv=2, width=32, scale=1.0,
                  work=None, bytes=0, status=None, stream=None)
    for change in (dict(sequences=far), dict(sequences=2 ** 31 - 1), dict(tokens=far),
                   dict(heads=far, kv=1)):
        assert lib.grs_prompt_attention(*{**prompt, **change}.values()) == -4, change
    for change in (dict(batch=far), dict(n=far), dict(heads=far, kv=1)):
        assert lib.grs_shared_prefix_attention(*{**prefix, **change}.values()) == -4, change


@pytest.mark.parametrize("scale", [2.4e38, -3.4e38, 1e39, -1e300])
def test_scales_beyond_fp32(lifted, scale):
    """The kernels hold scale * log2(e) in fp32: infinite, it made every row NaN."""
    from graph_rewrite_system_b200.prefix_attention import shared_prefix_attention
    from graph_rewrite_system_b200.prompt_attention import prompt_attention

    with pytest.raises(ValueError, match="scale"):
        prompt_attention(_z(6, 4, 32), _z(6, 2, 32), _z(6, 2, 32),
                         torch.tensor([0, 6], dtype=torch.int32), scale=scale, status=STATUS)
    with pytest.raises(ValueError, match="scale"):
        shared_prefix_attention(_z(6, 4, 32), _z(9, 2, 32), _z(9, 2, 32), scale=scale,
                                status=STATUS)


def test_c_abi_scales():
    from graph_rewrite_system_b200 import _lib

    for scale in (2.4e38, -3.4e38):
        assert _lib.lib().grs_prompt_attention(
            0, 256, 1, 1, 256, 1, 1, 256, 1, 1, 256, 1, 256, 1, 1, 1, 4, 2, 32, scale, 0, None,
            None) == -4
        assert _lib.lib().grs_shared_prefix_attention(
            0, 256, 1, 1, 256, 1, 1, 256, 1, 1, 300, None, None, 0, 0, 0, None, 0, 0, None, 0, 0,
            None, None, 0, 0, None, 256, 1, 1, 2, 4, 2, 32, scale, None, 0, None, None) == -4


def test_out_is_not_the_bias(lifted):
    """A bias row that every row of logits adds would be overwritten by the first."""
    from graph_rewrite_system_b200.token_logits import adjust_logits

    logits = torch.zeros(3, 70)
    room = torch.zeros(3, 70)
    for bias in (room, room[0], room[:1]):
        with pytest.raises(ValueError, match="bias"):
            adjust_logits(logits, bias=bias, out=room)
