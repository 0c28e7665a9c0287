"""The rotary, append and attention operators together: prompts and forked beams of a
small token model on a TokenKVCache of each type, against whole sequences in fp64 and,
for 8-bit pages, against what the pages hold."""
from __future__ import annotations

import pytest
import torch

from oracle import grouped_attention as grouped
from oracle import token_cache as oracle

pytestmark = pytest.mark.gpu

BF16, FP32, E4M3 = torch.bfloat16, torch.float32, torch.float8_e4m3fn
LAYERS, WIDTH, HEADS, KV_HEADS, D, VOCAB, PAGE = 2, 64, 4, 2, 32, 61, 4


def _weights(seed):
    g = torch.Generator().manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g)
    return dict(embed=rand(VOCAB, WIDTH),
                qkv=rand(LAYERS, WIDTH, (HEADS + 2 * KV_HEADS) * D) / WIDTH ** 0.5,
                out=rand(LAYERS, HEADS * D, WIDTH) / (HEADS * D) ** 0.5)


def _whole(w, tokens, frequencies):
    """The last token's state and every layer's turned keys and values, in fp64."""
    w = {n: t.double() for n, t in w.items()}
    x, cache = w["embed"][tokens], []
    places = torch.arange(len(tokens))
    for layer in range(LAYERS):
        qkv = (x @ w["qkv"][layer]).view(len(tokens), -1, D)
        q, k, v = qkv.split([HEADS, KV_HEADS, KV_HEADS], 1)
        q, _ = oracle.turn(q, places, frequencies, False)
        k, _ = oracle.turn(k, places, frequencies, False)
        cache.append((k, v))
        o, _, _ = grouped.prompt_attention(q, k, v, [0, len(tokens)])
        x = x + o.flatten(1) @ w["out"][layer]
    return x[-1], cache


@pytest.mark.parametrize("dtype", [FP32, E4M3])
def test_prompts_and_beams(cuda_device, dtype):
    from graph_rewrite_system_b200.prompt_attention import prompt_attention
    from graph_rewrite_system_b200.rotary import rotary_frequencies, rotate_positions
    from graph_rewrite_system_b200.token_cache import TokenKVCache

    dev = cuda_device
    host = _weights(5)
    w = {n: t.to(dev) for n, t in host.items()}
    f = rotary_frequencies(D, device=dev)
    cache = TokenKVCache(layers=LAYERS, capacity=300, page_size=PAGE, heads=KV_HEADS,
                         head_width=D, device=dev, dtype=dtype)
    g = torch.Generator().manual_seed(6)
    prompts = [torch.randint(0, VOCAB, (n,), generator=g).tolist() for n in (18, 7)]
    lengths = torch.tensor([len(p) for p in prompts], dtype=torch.int32, device=dev)
    table = torch.zeros(2, 5, dtype=torch.int32, device=dev)
    for b, p in enumerate(prompts):
        need = -(-len(p) // PAGE)
        table[b, :need] = cache.alloc_pages(need)
    # the prompts, packed: into the pages, and through their own attention
    packed = torch.tensor(prompts[0] + prompts[1], device=dev)
    offsets = torch.tensor([0, 18, 25], dtype=torch.int32, device=dev)
    places = torch.cat([torch.arange(18), torch.arange(7)]).to(dev)
    empty = torch.zeros(2, dtype=torch.int32, device=dev)
    x = w["embed"][packed]
    for layer in range(LAYERS):
        q, k, v = (x @ w["qkv"][layer]).view(25, -1, D).split([HEADS, KV_HEADS, KV_HEADS], 1)
        turned = cache.append(layer, k, v, table, empty, offsets=offsets, query=q, frequencies=f)
        q, k = rotate_positions(q, k, places, f)
        assert torch.equal(turned, q)
        x = x + prompt_attention(q, k, v, offsets).flatten(1) @ w["out"][layer]
    cache.check_status()
    history = [list(p) for p in prompts]

    def read(layer, rows, n):
        """Keys and values that a row's pages hold, as fp64."""
        slot, row = rows[torch.arange(n) // PAGE].long(), torch.arange(n) % PAGE
        out = []
        for arena, scales in ((cache.keys, cache.key_scales), (cache.values, cache.value_scales)):
            held = arena[layer].cpu().double()[slot, row]
            if scales is not None:
                held = held * scales[layer].cpu().double()[slot][..., None]
            out.append(held)
        return out

    def check(states, table, lengths):
        """fp32: sums of at most 128 + 128 terms a layer, each relative to absolute sums
        a few times the result: 2 layers * 256 * 2^-24 * 16 < 5e-4 of the size.  8 bits:
        each value within half a step of what was written, 2^-4 of it, and where it
        has sunk below the scale's normal numbers, at most twice half of 2^-9."""
        for b, tokens in enumerate(history):
            exp, caches = _whole(host, tokens, f.cpu())
            n = int(lengths[b])
            assert n == len(tokens)
            if dtype is FP32:
                off = (states[b].double().cpu() - exp).abs().max()
                assert float(off) <= 5e-4 * float(exp.abs().max())
            for layer, (k, v) in enumerate(caches[:1 if dtype is E4M3 else LAYERS]):
                # (deeper layers' keys hang on what the first one's pages hold)
                for held, true in zip(read(layer, table[b].cpu(), n), (k, v)):
                    if dtype is FP32:
                        assert float((held - true).abs().max()) <= 5e-4 * float(true.abs().max())
                        continue
                    near = 2.0 ** -4 * true.abs() * 1.01 + 2.0 ** -9 * float(
                        torch.maximum(cache.key_scales[layer].max(),
                                      cache.value_scales[layer].max())) + 1e-5
                    assert bool(((held - true).abs() <= near).all())

    check(x[offsets[1:].long() - 1], table, lengths)
    children = [[0, 0, 1], [0, 0, 1, 2, 2], [4, 3, 3, 0, 1], [0, 1, 2, 3, 4], [0, 0, 0, 0, 0]]
    for step, parents in enumerate(children * 2):
        if step == 5:
            parents = [0, 1, 2]
        if step > 5:
            parents = [p % len(history) for p in parents]
        pick = torch.tensor(parents, device=dev)
        chosen = torch.randint(0, VOCAB, (len(parents),), generator=g).tolist()
        parent_table, parent_lengths = table[pick], lengths[pick]
        grown = cache.fork_device(parent_table, parent_lengths)
        cache.release_device(table, lengths)              # shared pages live on
        now = parent_lengths + 1
        x = w["embed"][torch.tensor(chosen, device=dev)]
        for layer in range(LAYERS):
            qkv = (x @ w["qkv"][layer]).view(len(parents), -1, D)
            q, k, v = qkv.split([HEADS, KV_HEADS, KV_HEADS], 1)
            q = cache.append(layer, k, v, grown, parent_lengths, source_table=parent_table,
                             query=q, frequencies=f)
            context = cache.attend(layer, q, grown, now)
            if dtype is E4M3:
                results = oracle.quantized_attention(
                    q.cpu(), cache.keys[layer].cpu(), cache.values[layer].cpu(),
                    cache.key_scales[layer].cpu(), cache.value_scales[layer].cpu(), grown.cpu(),
                    now.cpu())
                bound = oracle.quantized_bound(results, FP32, D, int(now.max()))
                assert bool(((context.double().cpu() - results[0]).abs() <= bound).all())
            x = x + context.flatten(1) @ w["out"][layer]
        cache.check_status()
        history = [history[p] + [t] for p, t in zip(parents, chosen)]
        table, lengths = grown, now
        check(x, table, lengths)
        # pages in use: those that the beams' tables name
        used = {int(table[b, c]) for b in range(len(parents))
                for c in range(-(-int(lengths[b]) // PAGE))}
        assert cache.allocated_pages == len(used)
    cache.release_device(table, lengths)
    cache.check_status()
    assert cache.allocated_pages == 0


def test_fork_errors(cuda_device):
    """Parents whose tables do not hold their lengths, and an exhausted pool."""
    from graph_rewrite_system_b200.token_cache import TokenKVCache

    size = dict(layers=1, page_size=4, heads=1, head_width=8, device=cuda_device, dtype=BF16)
    cache = TokenKVCache(capacity=6, **size)
    table = cache.alloc_pages(2).view(1, 2).expand(2, 2).contiguous()
    for bad in (-1, 9, 1 << 30):
        lengths = torch.tensor([bad, 5], dtype=torch.int32, device=cuda_device)
        child = cache.fork_device(table, lengths)
        assert child.shape == (2, 3) and not child[0].any()
        with pytest.raises(RuntimeError, match="length"):
            cache.check_status()
        cache.reset()
        table = cache.alloc_pages(2).view(1, 2).expand(2, 2).contiguous()
    lengths = torch.full((2,), 8, dtype=torch.int32, device=cuda_device)
    for _ in range(2):
        cache.fork_device(table, lengths)
    cache.check_status()
    cache.fork_device(table, lengths)
    with pytest.raises(RuntimeError, match="exhausted"):
        cache.check_status()
    with pytest.raises(ValueError, match="parent_table"):
        cache.fork_device(table.long(), lengths)


@pytest.mark.parametrize("dtype", [BF16, E4M3])
def test_step_in_a_graph(cuda_device, dtype):
    """Append and attention of one step captured once and replayed as the sequences
    grow, on the tensors that hold the step's inputs."""
    from graph_rewrite_system_b200.rotary import rotary_frequencies
    from graph_rewrite_system_b200.token_cache import TokenKVCache

    dev = cuda_device
    f = rotary_frequencies(64, device=dev)
    make = lambda: TokenKVCache(layers=1, capacity=40, page_size=8, heads=2, head_width=64,
                                device=dev, dtype=dtype)
    caches = make(), make()
    table = torch.arange(36, dtype=torch.int32, device=dev).view(6, 6)
    lengths = torch.tensor([0, 3, 7, 8, 15, 20], dtype=torch.int32, device=dev)
    g = torch.Generator().manual_seed(7)
    qkv = torch.zeros(6, 12, 64, dtype=BF16, device=dev)
    q, k, v = qkv.split([8, 2, 2], 1)
    for c in caches:
        c.keys.copy_(torch.zeros(()).to(dtype)), c.values.copy_(torch.zeros(()).to(dtype))

    def step(cache):
        turned = cache.append(0, k, v, table, lengths, query=q, frequencies=f)
        return cache.attend(0, turned, table, lengths + 1)

    step(make())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(caches[0])
        lengths += 1
    start = torch.tensor([0, 3, 7, 8, 15, 20], dtype=torch.int32, device=dev)
    rows = [torch.randn(6, 12, 64, generator=g).to(BF16) for _ in range(12)]
    seen = []
    lengths.copy_(start)
    for r in rows:
        qkv.copy_(r)
        graph.replay()
        seen.append(out.clone())
    lengths.copy_(start)
    for r, exp in zip(rows, seen):
        qkv.copy_(r)
        assert torch.equal(step(caches[1]), exp)
        lengths += 1
    for a, b in zip((caches[0].keys, caches[0].values), (caches[1].keys, caches[1].values)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
