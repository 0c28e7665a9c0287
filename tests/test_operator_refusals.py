"""Refusals of the prompt, shared-prefix and logit operators, on the CPU: the
argument checks (with the CUDA check lifted, nothing is launched before them)
and the C ABI's own (which return before any CUDA call)."""
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


def _z(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype)


def _offsets(*values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype)


PROMPT = dict(query=_z(6, 4, 32), key=_z(6, 2, 32), value=_z(6, 2, 32), offsets=_offsets(0, 6))


@pytest.mark.parametrize("change", [
    dict(query=_z(6, 4, 32, dtype=torch.float16)), dict(query=_z(6, 4, 32, dtype=torch.float32)),
    dict(query=_z(1, 4, 32).expand(1 << 30, 4, 32), key=_z(1, 2, 32).expand(1 << 30, 2, 32),
         value=_z(1, 2, 32).expand(1 << 30, 2, 32)),
    dict(query=_z(6, 3, 32)), dict(query=_z(6, 4, 1, 32)), dict(query=_z(6, 4, 300),
                                                                key=_z(6, 2, 300),
                                                                value=_z(6, 2, 300)),
    dict(key=_z(5, 2, 32)), dict(value=_z(6, 1, 32)), dict(key=_z(6, 0, 32), value=_z(6, 0, 32)),
    dict(query=_z(6, 4, 64)[:, :, ::2]), dict(value=_z(6, 32, 2).transpose(1, 2)),
    dict(offsets=_offsets(0, 6, dtype=torch.int64)), dict(offsets=_offsets()),
    dict(offsets=_offsets(0, 1, 6)[::2]), dict(offsets=_offsets(0, 6)[None]),
    dict(out=_z(6, 4, 31)), dict(out=_z(6, 4, 32, dtype=torch.float32)),
    dict(out=_z(1, 4, 32).expand(6, 4, 32)), dict(out=PROMPT["query"]),
    dict(status=torch.zeros(1, dtype=torch.int64)), dict(scale=float("nan")),
    dict(scale=float("inf")),
])
def test_prompt_refusals(lifted, change):
    from graph_rewrite_system_b200.prompt_attention import prompt_attention

    args = {**PROMPT, **change}
    rest = {n: args.pop(n) for n in ("out", "status", "scale") if n in args}
    rest.setdefault("status", torch.zeros(1, dtype=torch.int32))
    with pytest.raises(ValueError):
        prompt_attention(**args, **rest)


def test_prompt_without_tokens_launches_nothing(lifted):
    from graph_rewrite_system_b200.prompt_attention import prompt_attention

    out = prompt_attention(_z(0, 4, 32), _z(0, 2, 32), _z(0, 2, 32), _offsets(0))
    assert out.shape == (0, 4, 32)


PREFIX = dict(query=_z(3, 4, 32), prefix_key=_z(9, 2, 32), prefix_value=_z(9, 2, 32),
              key_cache=_z(5, 8, 2, 32), value_cache=_z(5, 8, 2, 32),
              block_table=torch.zeros(3, 2, dtype=torch.int32),
              lengths=torch.zeros(3, dtype=torch.int32), current_key=_z(3, 2, 32),
              current_value=_z(3, 2, 32), current_valid=torch.ones(3, dtype=torch.bool))


@pytest.mark.parametrize("change", [
    dict(query=_z(3, 4, 32, dtype=torch.float16)), dict(query=_z(3, 5, 32)),
    dict(query=_z(3, 4, 1, 32)), dict(prefix_key=_z(9, 2, 64)), dict(prefix_value=_z(8, 2, 32)),
    dict(prefix_key=_z(2, 9, 32)), dict(key_cache=None), dict(lengths=None),
    dict(block_table=None), dict(key_cache=_z(5, 8, 4, 32)), dict(value_cache=_z(4, 8, 2, 32)),
    dict(value_cache=_z(5, 2, 8, 32).transpose(1, 2)),
    dict(key_cache=_z(5, 8, 2, 32, dtype=torch.float32)),
    dict(block_table=torch.zeros(3, 2, dtype=torch.int64)),
    dict(block_table=torch.zeros(4, 2, dtype=torch.int32)),
    dict(block_table=torch.zeros(2, 3, dtype=torch.int32).T),
    dict(lengths=torch.zeros(3, dtype=torch.int64)), dict(lengths=torch.zeros(2, dtype=torch.int32)),
    dict(current_value=None), dict(current_key=None), dict(current_key=_z(3, 4, 32)),
    dict(current_key=_z(2, 3, 32).transpose(0, 1)),
    dict(current_key=None, current_value=None),
    dict(current_valid=torch.ones(3)), dict(current_valid=torch.ones(2, dtype=torch.bool)),
    dict(scale=float("nan")), dict(out=_z(3, 4, 33)), dict(out=PREFIX["query"]), dict(out=_z(3, 1, 32).expand(3, 4, 32)),
    dict(block_table=torch.zeros(3, 1, dtype=torch.int32).expand(3, 1 << 27)),
    dict(prefix_key=_z(1, 2, 32).expand(1 << 30, 2, 32),
         prefix_value=_z(1, 2, 32).expand(1 << 30, 2, 32)),
])
def test_prefix_refusals(lifted, change):
    from graph_rewrite_system_b200.prefix_attention import shared_prefix_attention

    with pytest.raises(ValueError):
        shared_prefix_attention(**{**PREFIX, "status": torch.zeros(1, dtype=torch.int32), **change})


LOGITS = dict(logits=torch.zeros(3, 70), tokens=torch.zeros(3, 5, dtype=torch.int32))


@pytest.mark.parametrize("change", [
    dict(logits=torch.zeros(3, 70, dtype=torch.float16)), dict(logits=torch.zeros(70)),
    dict(logits=torch.zeros(70, 3).T), dict(tokens=torch.zeros(3, 5)),
    dict(tokens=torch.zeros(3, 1, dtype=torch.int32).expand(3, 1 << 30)),
    dict(tokens=torch.zeros(2, 5, dtype=torch.int32)),
    dict(tokens=torch.zeros(5, 3, dtype=torch.int32).T),
    dict(lengths=torch.zeros(3, dtype=torch.int64)),
    dict(prompt_lengths=torch.zeros(2, dtype=torch.int32)),
    dict(tokens=None, lengths=torch.zeros(3, dtype=torch.int32)),
    dict(repetition=0.0), dict(repetition=-1.0), dict(repetition=float("nan")),
    dict(repetition=torch.ones(2)), dict(presence=torch.ones(3, dtype=torch.float64)),
    dict(frequency=torch.ones(3, 1)), dict(bias=torch.zeros(69)), dict(bias=torch.zeros(2, 70)),
    dict(bias=torch.zeros(70, dtype=torch.bfloat16)), dict(bias=torch.zeros(70, 3).T),
    dict(allowed=torch.zeros(2, dtype=torch.int32)), dict(allowed=torch.zeros(3, dtype=torch.int64)),
    dict(allowed=torch.zeros(2, 3, dtype=torch.int32)),
    dict(out=torch.zeros(3, 71)), dict(out=torch.zeros(1, 70).expand(3, 70)),
    dict(out=torch.zeros(3, 70, dtype=torch.bfloat16)),
])
def test_logits_refusals(lifted, change):
    from graph_rewrite_system_b200.token_logits import adjust_logits

    with pytest.raises(ValueError):
        adjust_logits(**{**LOGITS, **change})


def test_cpu_tensors_raise():
    from graph_rewrite_system_b200.prefix_attention import shared_prefix_attention
    from graph_rewrite_system_b200.prompt_attention import prompt_attention
    from graph_rewrite_system_b200.token_logits import adjust_logits

    for call, args in ((prompt_attention, PROMPT), (shared_prefix_attention, PREFIX),
                       (adjust_logits, LOGITS)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call(**args)


def test_c_abi_refusals():
    from graph_rewrite_system_b200 import _lib

    lib = _lib.lib()
    shape, work = -4, -8
    prompt = dict(dtype=0, q=256, q_st=1, q_sh=1, k=256, k_st=1, k_sh=1, v=256, v_st=1, v_sh=1,
                  offsets=256, sequences=1, out=256, o_st=1, o_sh=1, tokens=1, heads=4, kv=2,
                  width=32, scale=1.0, clear=0, status=None, stream=None)
    for change in (dict(dtype=7), dict(heads=3), dict(kv=0), dict(heads=0), dict(width=0),
                   dict(width=257), dict(tokens=-1), dict(sequences=-1), dict(q=None),
                   dict(offsets=None), dict(out=None), dict(scale=float("inf"))):
        assert lib.grs_prompt_attention(*{**prompt, **change}.values()) == shape, change
    assert lib.grs_prompt_attention(*{**prompt, "tokens": 0}.values()) == 0
    prefix = dict(dtype=0, q=256, q_sb=1, q_sh=1, pk=256, pk_st=1, pk_sh=1, pv=256, pv_st=1,
                  pv_sh=1, n=300, kc=256, vc=256, kc_sp=1, kc_st=1, kc_sh=1, bt=256, bt_s=1,
                  blocks=1, lengths=256, pages=1, page=16, ck=None, cv=None, ck_sb=0, ck_sh=0,
                  valid=None, out=256, o_sb=1, o_sh=1, batch=2, heads=4, kv=2, width=32, scale=1.0,
                  work=256, bytes=1 << 30, status=None, stream=None)
    for change in (dict(dtype=7), dict(heads=3), dict(kv=0), dict(width=257), dict(batch=-1),
                   dict(n=-1), dict(pk=None), dict(kc=None), dict(bt=None), dict(lengths=None),
                   dict(page=0), dict(blocks=1 << 30), dict(ck=256), dict(q=None), dict(out=None)):
        assert lib.grs_shared_prefix_attention(*{**prefix, **change}.values()) == shape, change
    for change in (dict(work=None), dict(bytes=8), dict(work=260)):
        assert lib.grs_shared_prefix_attention(*{**prefix, **change}.values()) == work, change
    assert lib.grs_shared_prefix_attention(*{**prefix, "batch": 0}.values()) == 0
    # short prefixes are read by the pages' kernel and need no workspace
    assert lib.grs_shared_prefix_workspace_bytes(2, 4, 2, 32, 0, 32) == 0
    assert lib.grs_shared_prefix_workspace_bytes(2, 4, 2, 32, 5, 16) == 0
    assert lib.grs_shared_prefix_workspace_bytes(2, 4, 2, 32, 300, 16) > 0
    logits = dict(dtype=1, x=256, x_sb=9, out=256, o_sb=9, rows=1, vocab=9, tokens=256, i64=0,
                  t_sb=3, history=3, lengths=None, prompts=None, rep=None, pres=None, freq=None,
                  r=1.0, p=0.0, f=0.0, bias=None, b_sb=0, allowed=None, a_sb=0, fill=0.0,
                  stream=None)
    for change in (dict(dtype=7), dict(rows=-1), dict(vocab=-1), dict(history=-1),
                   dict(history=1 << 30), dict(tokens=None), dict(x=None), dict(out=None)):
        assert lib.grs_adjust_logits(*{**logits, **change}.values()) == shape, change
    assert lib.grs_adjust_logits(*{**logits, "rows": 0}.values()) == 0
    # the table forms: the same answers, floats and null pointers included
    for name, args, change in (("prompt_attention", prompt, dict(tokens=0)),
                               ("prompt_attention", prompt, dict(scale=float("inf"))),
                               ("shared_prefix_attention", prefix, dict(work=None)),
                               ("shared_prefix_attention", prefix, dict(scale=float("nan"))),
                               ("adjust_logits", logits, dict(rows=0)),
                               ("adjust_logits", logits, dict(out=None))):
        values = [v or 0 for v in {**args, **change}.values()]
        table = _lib.words_of(f"grs_{name}").pack(*values)
        expected = getattr(lib, f"grs_{name}")(*{**args, **change}.values())
        assert getattr(lib, f"grs_{name}_words")(table) == expected, (name, change)
        assert getattr(lib, f"grs_{name}_words")(None) == shape
