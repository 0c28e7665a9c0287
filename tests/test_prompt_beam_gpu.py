"""The prompt, shared-prefix and logit operators together: a beam search of a
small token model behind one prompt, on the framework's paged cache, against
the whole sequences recomputed in fp64."""
from __future__ import annotations

import pytest
import torch

from oracle import grouped_attention as oracle

pytestmark = pytest.mark.gpu

LAYERS, WIDTH, HEADS, KV_HEADS, D, VOCAB, BEAMS = 2, 64, 4, 2, 32, 101, 5


def _weights(seed):
    g = torch.Generator().manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g)
    return dict(embed=rand(VOCAB, WIDTH), place=0.3 * rand(400, WIDTH),
                qkv=rand(LAYERS, WIDTH, (HEADS + 2 * KV_HEADS) * D) / WIDTH ** 0.5,
                out=rand(LAYERS, HEADS * D, WIDTH) / (HEADS * D) ** 0.5,
                head=rand(WIDTH, VOCAB) / WIDTH ** 0.5)


def _whole(w, tokens):
    """Logits of the last token, every layer recomputed in fp64."""
    w = {n: t.double() for n, t in w.items()}
    x = w["embed"][tokens] + w["place"][:len(tokens)]
    for layer in range(LAYERS):
        qkv = (x @ w["qkv"][layer]).view(len(tokens), -1, D)
        q, k, v = qkv.split([HEADS, KV_HEADS, KV_HEADS], 1)
        o, _, _ = oracle.prompt_attention(q, k, v, [0, len(tokens)])
        x = x + o.flatten(1) @ w["out"][layer]
    return x[-1] @ w["head"]


def test_beam_search_behind_a_prompt(cuda_device):
    from graph_rewrite_system_b200.paged_cache import PagedKVCache
    from graph_rewrite_system_b200.prefix_attention import shared_prefix_attention
    from graph_rewrite_system_b200.prompt_attention import prompt_attention
    from graph_rewrite_system_b200.token_logits import adjust_logits

    dev = cuda_device
    host = _weights(3)
    w = {n: t.to(dev) for n, t in host.items()}
    prompt = torch.randint(0, VOCAB, (70,), generator=torch.Generator().manual_seed(4)).tolist()
    # the prompt, packed with another one that nothing else uses
    packed = prompt + [7] * 9
    offsets = torch.tensor([0, len(prompt), len(packed)], dtype=torch.int32, device=dev)
    place = torch.tensor(list(range(len(prompt))) + list(range(9)), device=dev)
    x = w["embed"][torch.tensor(packed, device=dev)] + w["place"][place]
    prefix = []
    for layer in range(LAYERS):
        qkv = (x @ w["qkv"][layer]).view(len(packed), -1, D)
        q, k, v = qkv.split([HEADS, KV_HEADS, KV_HEADS], 1)
        prefix.append((k[:len(prompt)], v[:len(prompt)]))
        x = x + prompt_attention(q, k, v, offsets).flatten(1) @ w["out"][layer]
    logits = (x[len(prompt) - 1] @ w["head"])[None]

    # fp32 sums of at most 128 + 80 terms, twice per layer, each relative to
    # absolute sums a few times the result: 2 layers * 2 * 208 * 2^-24 * 8 < 5e-4
    # of the logits' size
    def close(got, exp):
        assert float((got.double().cpu() - exp).abs().max()) <= 5e-4 * float(exp.abs().max())

    close(logits[0], _whole(host, prompt))
    knobs = dict(repetition=1.2, presence=0.1, frequency=0.2)
    # a grammar: even tokens, and never token 4
    allowed = torch.zeros((VOCAB + 31) // 32, dtype=torch.int64)
    for t in range(0, VOCAB, 2):
        if t != 4:
            allowed[t // 32] |= 1 << (t % 32)
    allowed = allowed.to(torch.int32)
    cache = PagedKVCache(layers=LAYERS, capacity=400, page_size=4, heads=KV_HEADS, head_width=D,
                         model_width=WIDTH, device=dev, dtype=torch.float32)
    history = [list(prompt)]
    handles = [cache.empty_handle()]
    scores = torch.zeros(1, device=dev)
    for step in range(9):
        rows = len(history)
        tokens = torch.tensor(history, dtype=torch.int32, device=dev)
        prompts = torch.full((rows,), len(prompt), dtype=torch.int32, device=dev)
        adjusted = adjust_logits(logits, tokens=tokens, prompt_lengths=prompts,
                                 allowed=allowed.to(dev), **knobs)
        exp = oracle.adjust_logits(logits.cpu(), tokens=tokens.cpu(), prompt_lengths=prompts.cpu(),
                                   allowed=allowed, **knobs)
        assert torch.equal(torch.isfinite(adjusted).cpu(), torch.isfinite(exp))
        fine = torch.isfinite(exp)
        assert torch.allclose(adjusted.double().cpu()[fine], exp[fine], rtol=1e-6, atol=1e-5)
        ranked = scores[:, None] + torch.log_softmax(adjusted, -1)
        scores, pick = ranked.flatten().topk(BEAMS)
        parents, chosen = (pick // VOCAB).tolist(), (pick % VOCAB).tolist()
        assert all(t % 2 == 0 and t != 4 for t in chosen)
        history = [history[p] + [t] for p, t in zip(parents, chosen)]
        handles = [handles[p] for p in parents]
        # the chosen tokens through the model: prefix, pages, the token itself
        table, lengths = cache.block_table(handles)
        x = w["embed"][pick % VOCAB] + w["place"][len(history[0]) - 1]
        keys, values = [], []
        for layer in range(LAYERS):
            qkv = (x @ w["qkv"][layer]).view(BEAMS, -1, D)
            q, k, v = qkv.split([HEADS, KV_HEADS, KV_HEADS], 1)
            o = shared_prefix_attention(q, *prefix[layer], cache.keys[layer], cache.values[layer],
                                        table, lengths, current_key=k, current_value=v)
            keys.append(k)
            values.append(v)
            x = x + o.flatten(1) @ w["out"][layer]
        logits = x @ w["head"]
        handles = cache.append_batch(handles, torch.stack(keys), torch.stack(values), x)
        for b in range(BEAMS):
            close(logits[b], _whole(host, history[b]))
    assert len({tuple(h) for h in history}) == BEAMS
