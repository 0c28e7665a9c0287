"""Refusals of the rotary positions, the append and the attention over 8-bit
pages, on the CPU: the argument checks (with the CUDA check lifted, nothing is
launched before them) and the C ABI's own (which return before any CUDA call)."""
from __future__ import annotations

import pytest
import torch

BF16, FP32, E4M3 = torch.bfloat16, torch.float32, torch.float8_e4m3fn


@pytest.fixture
def lifted(monkeypatch):
    from graph_rewrite_system_b200 import _lib

    def nothing(*a):
        raise AssertionError("a launch was reached")

    monkeypatch.setattr(_lib, "require_cuda", lambda *t: None)
    monkeypatch.setattr(_lib, "current_device", lambda: -1)
    monkeypatch.setattr(_lib, "lib", nothing)
    monkeypatch.setattr(_lib, "stream_on", nothing)


def _z(*shape, dtype=BF16):
    return torch.zeros(*shape, dtype=dtype)


def _i(*shape, dtype=torch.int32):
    return torch.zeros(*shape, dtype=dtype)


def _f(n):
    return torch.ones(n, dtype=torch.float64)


ROTATE = dict(query=_z(6, 4, 32), key=_z(6, 2, 32), positions=_i(6), frequencies=_f(16))


@pytest.mark.parametrize("change", [
    dict(query=_z(6, 4, 32, dtype=torch.float16), key=None), dict(query=_z(6, 4, 1, 32)),
    dict(query=_z(6, 4, 32, dtype=FP32)), dict(query=_z(6, 0, 32)), dict(key=_z(6, 0, 32)),
    dict(key=_z(5, 2, 32)), dict(key=_z(6, 2, 16)), dict(query=_z(6, 4, 64)[:, :, ::2]),
    dict(key=_z(6, 32, 2).transpose(1, 2)), dict(query=_z(6, 4, 300), key=_z(6, 2, 300)),
    dict(positions=_i(5)), dict(positions=_i(6, dtype=torch.int16)), dict(positions=_i(6, 1)),
    dict(positions=_i(12)[::2]), dict(frequencies=_f(17)), dict(frequencies=_f(0)),
    dict(frequencies=torch.ones(16)), dict(frequencies=_f(32)[::2]), dict(magnitude=float("nan")),
    dict(magnitude=float("inf")), dict(magnitude=1e39), dict(query_out=_z(6, 4, 31)),
    dict(query_out=_z(6, 4, 32, dtype=FP32)), dict(query_out=_z(6, 1, 32).expand(6, 4, 32)),
    dict(query_out=ROTATE["key"].expand(6, 2, 32).repeat(1, 2, 1)[:, :3]),
    dict(key_out=ROTATE["query"][:, :2]), dict(key=None, key_out=_z(6, 2, 32)),
    dict(query=_z(1, 4, 32).expand(1 << 30, 4, 32), key=None),
])
def test_rotate_refusals(lifted, change):
    from graph_rewrite_system_b200.rotary import rotate_positions

    with pytest.raises(ValueError):
        rotate_positions(**{**ROTATE, **change})


def test_rotated_in_place_with_other_strides(lifted):
    from graph_rewrite_system_b200.rotary import rotate_positions

    q = _z(4, 4, 32)
    with pytest.raises(ValueError, match="itself"):
        rotate_positions(q, None, _i(4), _f(16), query_out=q.transpose(0, 1))
    key = _z(6, 4, 32)
    with pytest.raises(ValueError, match="another"):
        rotate_positions(_z(6, 4, 32), key, _i(6), _f(16), query_out=key)


@pytest.mark.parametrize("args,kw", [
    ((0,), {}), ((7,), {}), ((8,), dict(base=0.0)), ((8,), dict(stretch=-1.0)),
    ((8,), dict(base=float("inf"))), ((8,), dict(stretch=2.0, trained=0)),
    ((8,), dict(stretch=2.0, trained=100, keep=(4.0, 4.0)))])
def test_frequency_refusals(args, kw):
    from graph_rewrite_system_b200.rotary import rotary_frequencies

    with pytest.raises(ValueError):
        rotary_frequencies(*args, device="cpu", **kw)


APPEND = dict(key=_z(3, 2, 32), value=_z(3, 2, 32), key_cache=_z(5, 8, 2, 32, dtype=E4M3),
              value_cache=_z(5, 8, 2, 32, dtype=E4M3), block_table=_i(3, 2), lengths=_i(3),
              key_scale=torch.ones(5, 2), value_scale=torch.ones(5, 2), query=_z(3, 4, 32),
              frequencies=_f(16))
PLAIN = dict(key_cache=_z(5, 8, 2, 32), value_cache=_z(5, 8, 2, 32), key_scale=None,
             value_scale=None)


@pytest.mark.parametrize("change", [
    dict(key=_z(3, 2, 32, dtype=torch.float16)), dict(key=_z(3, 64)), dict(value=_z(3, 1, 32)),
    dict(value=_z(3, 2, 32, dtype=FP32)), dict(key=_z(3, 4, 32), value=_z(3, 4, 32)),
    dict(key=_z(3, 0, 32), value=_z(3, 0, 32)), dict(key=_z(3, 2, 64)[:, :, ::2]),
    dict(key_scale=None), dict(value_scale=None), dict(key_scale=torch.ones(4, 2)),
    dict(key_scale=torch.ones(5, 2, dtype=torch.float64)), dict(key_scale=torch.ones(2, 5).T),
    dict(key_scale=torch.ones(1, 2).expand(5, 2), value_scale=torch.ones(1, 2).expand(5, 2)),
    dict(key_scale=torch.ones(5, 3)[:, :2]), dict(value_scale=APPEND["key_scale"]),
    dict(key_cache=_z(5, 8, 2, 32)), dict(value_cache=_z(5, 8, 2, 32)),
    dict(**{**PLAIN, "key_scale": torch.ones(5, 2)}),
    dict(**{**PLAIN, "key_cache": _z(5, 8, 2, 32, dtype=FP32)}),
    dict(**{**PLAIN, "value_cache": PLAIN["key_cache"]}),
    dict(**{**PLAIN, "key_cache": _z(1, 8, 2, 32).expand(5, 8, 2, 32),
            "value_cache": _z(1, 8, 2, 32).expand(5, 8, 2, 32)}),
    dict(value_cache=_z(5, 2, 8, 32, dtype=E4M3).transpose(1, 2)),
    dict(key_cache=_z(5, 0, 2, 32, dtype=E4M3), value_cache=_z(5, 0, 2, 32, dtype=E4M3)),
    dict(block_table=_i(3, 2, dtype=torch.int64)), dict(block_table=_i(4, 2)),
    dict(block_table=_i(2, 3).T), dict(block_table=_i(3, 1).expand(3, 1 << 27)),
    dict(lengths=_i(2)), dict(lengths=_i(3, dtype=torch.int64)), dict(lengths=_i(6)[::2]),
    dict(offsets=_i(3)), dict(offsets=_i(4, dtype=torch.int64)), dict(offsets=_i(8)[::2]),
    dict(key=_z(4, 2, 32), value=_z(4, 2, 32), query=None), dict(source_table=_i(2, 3).T),
    dict(source_table=_i(2, 2)), dict(frequencies=None), dict(frequencies=_f(17)),
    dict(frequencies=None, query=None, positions=_i(3)), dict(positions=_i(4)),
    dict(magnitude=float("nan")), dict(query=_z(3, 3, 32)), dict(query=_z(2, 4, 32)),
    dict(query=_z(3, 0, 32)), dict(query=_z(3, 4, 32, dtype=FP32)), dict(query=_z(3, 128)),
    dict(query=None, query_out=_z(3, 4, 32)), dict(query_out=_z(3, 4, 33)),
    dict(query=_z(3, 2, 32), query_out=APPEND["key"]),
    dict(status=torch.zeros(1, dtype=torch.int64)),
])
def test_append_refusals(lifted, change):
    from graph_rewrite_system_b200.token_cache import append_tokens

    with pytest.raises(ValueError):
        append_tokens(**{**APPEND, "status": _i(1), **change})


ATTEND = dict(query=_z(3, 4, 32), key_cache=_z(5, 8, 2, 32, dtype=E4M3),
              value_cache=_z(5, 8, 2, 32, dtype=E4M3), key_scale=torch.ones(5, 2),
              value_scale=torch.ones(5, 2), block_table=_i(3, 2), lengths=_i(3))


@pytest.mark.parametrize("change", [
    dict(query=_z(3, 4, 32, dtype=torch.float16)), dict(query=_z(3, 5, 32)),
    dict(query=_z(3, 128)), dict(query=_z(3, 4, 64)[:, :, ::2]), dict(query=_z(3, 4, 31)),
    dict(key_cache=_z(5, 8, 2, 32)), dict(value_cache=_z(5, 8, 2, 32, dtype=torch.float8_e5m2)),
    dict(value_cache=_z(4, 8, 2, 32, dtype=E4M3)), dict(key_cache=_z(5, 8, 64, dtype=E4M3)),
    dict(value_cache=_z(5, 2, 8, 32, dtype=E4M3).transpose(1, 2)),
    dict(key_scale=torch.ones(5, 1)), dict(value_scale=torch.ones(5, 2, dtype=BF16)),
    dict(key_scale=torch.ones(2, 5).T), dict(value_scale=torch.ones(5, 4)[:, :2]),
    dict(block_table=_i(3, 2, dtype=torch.int64)), dict(block_table=_i(2, 2)),
    dict(block_table=_i(2, 3).T), dict(block_table=_i(3, 1).expand(3, 1 << 27)),
    dict(lengths=_i(4)), dict(lengths=_i(3, dtype=torch.int64)), dict(scale=float("nan")),
    dict(scale=float("inf")), dict(scale=3e38), dict(out=_z(3, 4, 33)), dict(out=ATTEND["query"]),
    dict(out=_z(3, 1, 32).expand(3, 4, 32)), dict(status=torch.zeros(2, dtype=torch.int32)),
    dict(query=_z(1, 4, 32).expand(1 << 30, 4, 32)),
])
def test_attention_refusals(lifted, change):
    from graph_rewrite_system_b200.quantized_attention import quantized_attention

    with pytest.raises(ValueError):
        quantized_attention(**{**ATTEND, "status": _i(1), **change})


def test_nothing_to_do_launches_nothing(lifted):
    from graph_rewrite_system_b200.quantized_attention import quantized_attention
    from graph_rewrite_system_b200.rotary import rotate_positions
    from graph_rewrite_system_b200.token_cache import append_tokens

    got = rotate_positions(_z(0, 4, 32), _z(0, 2, 32), _i(0), _f(16))
    assert got[0].shape == (0, 4, 32) and got[1].shape == (0, 2, 32)
    none = dict(key=_z(0, 2, 32), value=_z(0, 2, 32), query=_z(0, 4, 32), offsets=_i(4))
    assert append_tokens(**{**APPEND, **none}).shape == (0, 4, 32)
    none = dict(query=_z(0, 4, 32), block_table=_i(0, 2), lengths=_i(0))
    assert quantized_attention(**{**ATTEND, **none}).shape == (0, 4, 32)


def test_cpu_tensors_raise():
    from graph_rewrite_system_b200.quantized_attention import quantized_attention
    from graph_rewrite_system_b200.rotary import rotate_positions
    from graph_rewrite_system_b200.token_cache import TokenKVCache, append_tokens

    for call, args in ((rotate_positions, ROTATE), (append_tokens, APPEND),
                       (quantized_attention, ATTEND)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call(**args)
    size = dict(layers=1, capacity=4, page_size=4, heads=2, head_width=8)
    with pytest.raises(RuntimeError, match="CUDA"):
        TokenKVCache(device="cpu", dtype=BF16, **size)
    with pytest.raises(ValueError, match="arenas"):
        TokenKVCache(device="cuda", dtype=torch.float16, **size)
    with pytest.raises(ValueError, match="positive"):
        TokenKVCache(device="cuda", dtype=BF16, **{**size, "heads": 0})


def test_c_abi_refusals():
    from graph_rewrite_system_b200 import _lib

    lib, shape, far = _lib.lib(), -4, 1 << 30
    rotate = dict(dtype=0, q=256, q_st=1, q_sh=1, k=256, k_st=1, k_sh=1, pos=256, wide=0, freq=256,
                  pairs=16, inter=0, mag=1.0, qo=256, qo_st=1, qo_sh=1, ko=256, ko_st=1, ko_sh=1,
                  tokens=1, heads=4, kv=2, width=32, stream=None)
    for change in (dict(dtype=2), dict(tokens=-1), dict(tokens=far), dict(heads=0),
                   dict(heads=far), dict(kv=-1), dict(width=0), dict(width=257), dict(pairs=17),
                   dict(pairs=0), dict(q=None), dict(qo=None), dict(pos=None), dict(freq=None),
                   dict(k=None), dict(ko=None), dict(mag=float("inf"))):
        assert lib.grs_rotate_positions(*{**rotate, **change}.values()) == shape, change
    assert lib.grs_rotate_positions(*{**rotate, "tokens": 0}.values()) == 0
    append = dict(dtype=0, cache=2, q=256, q_st=1, q_sh=1, qo=256, qo_st=1, qo_sh=1, clear=0,
                  k=256, k_st=1, k_sh=1, v=256, v_st=1, v_sh=1, kc=256, vc=256, c_sp=1, c_st=1,
                  c_sh=1, ks=256, vs=256, s_sp=1, bt=256, bt_s=1, src=None, src_s=0,
                  src_blocks=0, blocks=2,
                  lengths=256, offsets=None, pos=None, wide=0, freq=256, pairs=16, inter=0,
                  mag=1.0, tokens=1, seqs=1, heads=4, kv=2, width=32, pages=5, page=16,
                  status=None, stream=None)
    for change in (dict(dtype=2), dict(cache=1), dict(cache=7), dict(tokens=-1), dict(tokens=far),
                   dict(seqs=-1), dict(seqs=2), dict(seqs=far), dict(kv=0), dict(heads=3),
                   dict(heads=0), dict(width=0), dict(width=257), dict(pairs=17), dict(pairs=-1),
                   dict(page=0), dict(page=far), dict(blocks=far), dict(blocks=-1), dict(pages=-1),
                   dict(src_blocks=-1), dict(k=None), dict(v=None), dict(kc=None), dict(vc=None), dict(ks=None),
                   dict(vs=None), dict(bt=None), dict(lengths=None), dict(freq=None),
                   dict(qo=None), dict(mag=float("nan"))):
        assert lib.grs_append_tokens(*{**append, **change}.values()) == shape, change
    assert lib.grs_append_tokens(*{**append, "tokens": 0, "seqs": 0}.values()) == 0
    attend = dict(dtype=0, q=256, q_sb=1, q_sh=1, kc=256, vc=256, c_sp=1, c_st=1, c_sh=1, ks=256,
                  vs=256, s_sp=1, bt=256, bt_s=1, blocks=100, lengths=256, pages=5, page=16,
                  out=256, o_sb=1, o_sh=1, batch=1, heads=4, kv=2, width=32, scale=1.0, work=256,
                  bytes=1 << 30, status=None, stream=None)
    for change in (dict(dtype=2), dict(batch=-1), dict(batch=far), dict(heads=3), dict(heads=0),
                   dict(heads=far, kv=1), dict(kv=0), dict(width=0), dict(width=257),
                   dict(scale=float("inf")), dict(scale=2.4e38), dict(blocks=-1),
                   dict(blocks=far), dict(page=0), dict(pages=-1), dict(q=None), dict(out=None),
                   dict(lengths=None), dict(bt=None), dict(kc=None), dict(vc=None), dict(ks=None),
                   dict(vs=None)):
        assert lib.grs_quantized_attention(*{**attend, **change}.values()) == shape, change
    for change in (dict(work=None), dict(bytes=8), dict(work=260)):
        assert lib.grs_quantized_attention(*{**attend, **change}.values()) == -8, change
    assert lib.grs_quantized_attention(*{**attend, "batch": 0}.values()) == 0
    assert lib.grs_quantized_attention_workspace_bytes(1, 4, 2, 32, 16) == 0
    fork = dict(refs=256, free=256, count=256, capacity=4, table=256, stride=1, cols=1, lengths=256,
                n=1, page=4, child=256, c_stride=2, c_lengths=256, c_cols=2, status=None,
                stream=None)
    for change in (dict(n=-1), dict(capacity=0), dict(page=0), dict(c_cols=0)):
        assert lib.grs_cache_fork(*{**fork, **change}.values()) == shape, change
    assert lib.grs_cache_fork(*{**fork, "n": 0}.values()) == 0
    for name, args, change in (("rotate_positions", rotate, dict(tokens=0)),
                               ("rotate_positions", rotate, dict(mag=float("inf"))),
                               ("append_tokens", append, dict(mag=float("nan"))),
                               ("append_tokens", append, dict(kc=None)),
                               ("quantized_attention", attend, dict(work=None)),
                               ("quantized_attention", attend, dict(scale=float("nan")))):
        values = [v or 0 for v in {**args, **change}.values()]
        table = _lib.words_of(f"grs_{name}").pack(*values)
        expected = getattr(lib, f"grs_{name}")(*{**args, **change}.values())
        assert getattr(lib, f"grs_{name}_words")(table) == expected, (name, change)
        assert getattr(lib, f"grs_{name}_words")(None) == shape


def test_guarded_append_refusals(lifted):
    from graph_rewrite_system_b200.token_cache import append_tokens

    for status in (_i(3), _i(2, 1), _i(4)[::2], _i(2, dtype=torch.int64)):
        with pytest.raises(ValueError, match="status"):
            append_tokens(**{**APPEND, "status": status})


def test_c_abi_refusals_of_guards_and_forks_without_status():
    from graph_rewrite_system_b200 import _lib

    values = dict(dtype=0, cache=2, q=256, q_st=1, q_sh=1, qo=256, qo_st=1, qo_sh=1, flags=2,
                  k=256, k_st=1, k_sh=1, v=256, v_st=1, v_sh=1, kc=256, vc=256, c_sp=1, c_st=1,
                  c_sh=1, ks=256, vs=256, s_sp=1, bt=256, bt_s=1, src=None, src_s=0, src_blocks=0,
                  blocks=2, lengths=256, offsets=None, pos=None, wide=0, freq=256, pairs=16,
                  inter=0, mag=1.0, tokens=1, seqs=1, heads=4, kv=2, width=32, pages=5, page=16,
                  status=None, stream=None).values()
    assert _lib.lib().grs_append_tokens(*values) == -4
    fork = dict(refs=256, free=256, count=256, capacity=4, table=256, stride=1, cols=1, lengths=256,
                n=1, page=4, child=256, c_stride=2, c_lengths=256, c_cols=2, status=None,
                stream=None)
    for change in (dict(), dict(cols=-1, status=256)):
        assert _lib.lib().grs_cache_fork(*{**fork, **change}.values()) == -4, change


def test_pages_whose_rows_pass_31_bits(lifted):
    """Kept rows are counted in pieces, up to an element each, in 32 bits."""
    from graph_rewrite_system_b200.token_cache import append_tokens

    huge = lambda: _z(1, 1, 1, 256).expand(2, 1 << 23, 1, 256)
    args = dict(key=_z(3, 1, 256), value=_z(3, 1, 256), key_cache=huge(), value_cache=huge(),
                block_table=_i(3, 2), lengths=_i(3), status=_i(1))
    with pytest.raises(ValueError, match="2\\^31 elements"):
        append_tokens(**args, source_table=_i(3, 2))
    with pytest.raises(ValueError, match="overlap"):       # and without a source the next check
        append_tokens(**args)


def test_c_abi_refuses_pages_whose_rows_pass_31_bits():
    from graph_rewrite_system_b200 import _lib

    values = dict(dtype=0, cache=0, q=None, q_st=1, q_sh=1, qo=None, qo_st=1, qo_sh=1, flags=0,
                  k=256, k_st=1, k_sh=1, v=256, v_st=1, v_sh=1, kc=256, vc=256, c_sp=1, c_st=1,
                  c_sh=1, ks=None, vs=None, s_sp=0, bt=256, bt_s=1, src=256, src_s=1, src_blocks=2,
                  blocks=2, lengths=256, offsets=None, pos=None, wide=0, freq=None, pairs=0,
                  inter=0, mag=1.0, tokens=1, seqs=1, heads=0, kv=1, width=256, pages=2,
                  page=1 << 23, status=None, stream=None).values()
    assert _lib.lib().grs_append_tokens(*values) == -4
