"""Cases of the operators that keep a token model's keys and values.

Three operators of one decode step: ``rotate_positions`` (rotary positions of
queries and keys), ``append_tokens`` (new keys, rotated on the way, and values
into the pages of a paged cache, held as they are or in 8 bits with a scale for
each page and head) and ``quantized_attention`` (one query per sequence against
such 8-bit pages).

``run`` computes a case with elementary torch operations, or, where ``own`` is
true, through the framework's entry points; ``exact`` computes the same outputs
from the definitions in 64 bits.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
E4M3 = torch.float8_e4m3fn
LARGEST = 448.0          # of e4m3
CHUNK = 1 << 27          # gathered cache elements the plain attention holds at once


def listed():
    return [
        # one token of one sequence at this framework's own head layout (8 heads of 32)
        dict(name="rotate_one_token", op="rotate", dtype="bf16", heads=8, kv_heads=8, width=32,
             rotated=32, interleaved=False, tokens=1, far=900, stretch=1.0, magnitude=1.0),
        # a long packed prompt with grouped heads
        dict(name="rotate_prompt", op="rotate", dtype="bf16", heads=32, kv_heads=8, width=128,
             rotated=128, interleaved=False, tokens=16384, far=16384, stretch=1.0, magnitude=1.0),
        # half of each fp32 head, pairs side by side, far positions of a stretched context
        dict(name="rotate_partial_fp32", op="rotate", dtype="fp32", heads=8, kv_heads=8, width=64,
             rotated=32, interleaved=True, tokens=2003, far=1000000, stretch=8.0, magnitude=1.2),
        # a handful of sequences decoding into bf16 pages: the smallest call
        dict(name="append_few", op="append", dtype="bf16", pages="same", heads=8, kv_heads=2,
             width=64, rotated=64, interleaved=False, sequences=5, longest=1, least=1, past=129,
             page=16, fan=0, tail=0, spread=1, stretch=1.0, magnitude=1.0),
        # this framework's beam of 1000, four children of a parent, each with a copy of the
        # parent's last page in 8 bits
        dict(name="append_beam_e4m3", op="append", dtype="bf16", pages="e4m3", heads=32,
             kv_heads=8, width=128, rotated=128, interleaved=False, sequences=1000, longest=1,
             least=1, past=400, page=16, fan=4, tail=0, spread=2, stretch=1.0, magnitude=1.0),
        # a serving batch of ragged prompts into 8-bit pages, some behind cached turns, padded
        dict(name="append_prompts_e4m3", op="append", dtype="bf16", pages="e4m3", heads=32,
             kv_heads=8, width=128, rotated=128, interleaved=True, sequences=16, longest=1500,
             least=90, past=100, page=16, fan=0, tail=61, spread=3, stretch=8.0, magnitude=1.1),
        # one long document into bf16 pages
        dict(name="append_document", op="append", dtype="bf16", pages="same", heads=32,
             kv_heads=8, width=128, rotated=128, interleaved=False, sequences=1, longest=16384,
             least=16384, past=0, page=32, fan=0, tail=0, spread=4, stretch=1.0, magnitude=1.0),
        # a few samples of a short prompt: the smallest read of 8-bit pages
        dict(name="attend_few", op="attend", dtype="bf16", heads=8, kv_heads=2, width=64,
             sequences=5, longest=129, least=1, page=16, fan=1, spread=5),
        # a batch of requests of ragged lengths
        dict(name="attend_batch", op="attend", dtype="bf16", heads=32, kv_heads=8, width=128,
             sequences=64, longest=4099, least=300, page=16, fan=1, spread=6),
        # a wide batch over long contexts
        dict(name="attend_wide", op="attend", dtype="bf16", heads=32, kv_heads=8, width=128,
             sequences=512, longest=4096, least=2048, page=32, fan=1, spread=7),
        # two very long documents
        dict(name="attend_long", op="attend", dtype="bf16", heads=32, kv_heads=8, width=128,
             sequences=2, longest=131000, least=100000, page=64, fan=1, spread=8),
        # fp32 queries at this framework's own head layout
        dict(name="attend_fp32", op="attend", dtype="fp32", heads=8, kv_heads=8, width=32,
             sequences=200, longest=1001, least=0, page=16, fan=4, spread=9),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["rotate", "append", "attend"])
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    group = rng.choice([1, 1, 2, 3, 4, 5, 7, 8, 16])
    width = rng.choice([32, 64, 128, 32, 64, 128, 40, 80, 96, 256])
    case = dict(op=op, dtype=rng.choice(["bf16", "bf16", "bf16", "fp32"]),
                heads=kv_heads * group, kv_heads=kv_heads, width=width)
    if op == "attend":
        longest = _log_int(rng, 1, 131072)
        sequences = _log_int(rng, 1, 1000)
        while sequences * longest * kv_heads * width > 400 * 4096 * 8 * 128:
            sequences = max(1, sequences // 2)
            longest = longest if sequences > 1 else longest // 2
        return dict(case, sequences=sequences, longest=longest,
                    least=rng.choice([0, 1, longest // 2, longest]),
                    page=rng.choice([8, 16, 16, 32, 64]), fan=rng.choice([1, 1, 4]),
                    spread=rng.randrange(1 << 30))
    scaled = rng.random() < 0.4
    case.update(rotated=rng.choice([width, width, width // 2, width // 4 * 2]),
                interleaved=rng.random() < 0.5, stretch=8.0 if scaled else 1.0,
                magnitude=1.2 if scaled else 1.0)
    most = 16384 * 48 * 128 // ((kv_heads * group + 2 * kv_heads) * width)
    most = min(16384, most) // (2 if case["dtype"] == "fp32" else 1)
    if op == "rotate":
        return dict(case, tokens=_log_int(rng, 1, most), far=_log_int(rng, 100, 2000000))
    case.update(pages=rng.choice(["same", "e4m3", "e4m3"]), page=rng.choice([8, 16, 16, 32, 64]),
                past=rng.choice([0, _log_int(rng, 1, 2000), _log_int(rng, 1, 2000)]),
                spread=rng.randrange(1 << 30))
    if rng.random() < 0.5:
        sequences = min(_log_int(rng, 1, 1000), most)
        # every sequence has a page or two of its own
        while sequences * case["page"] * kv_heads * width > 8 * 16384 * 8 * 128:
            sequences = max(1, sequences // 2)
        return dict(case, sequences=sequences, longest=1, least=1, fan=rng.choice([0, 1, 4]),
                    tail=0)
    sequences = _log_int(rng, 1, 300)
    longest = _log_int(rng, 1, most)
    while sequences * longest > most:
        sequences = max(1, sequences // 2)
    while sequences * case["page"] * kv_heads * width > 8 * 16384 * 8 * 128:
        sequences = max(1, sequences // 2)
    return dict(case, sequences=sequences, longest=longest,
                least=rng.choice([0, 1, longest // 2, longest]), fan=0,
                tail=rng.choice([0, 0, rng.randrange(1, 100)]))


def _ragged(rng, count, low, high):
    """Lengths between low and high; the longest one is there."""
    out = [rng.randint(low, high) for _ in range(count)]
    out[rng.randrange(count)] = high
    return out


def _new_and_past(case):
    """New and cached tokens of each sequence of an append; the `fan` children of
    one parent have one past."""
    rng, n = random.Random(case["spread"]), case["sequences"]
    new = _ragged(rng, n, case["least"], case["longest"])
    parents = _ragged(rng, -(-n // max(1, case["fan"])), 0, case["past"])
    return new, [parents[i // max(1, case["fan"])] for i in range(n)]


def _attended(case):
    """Lengths and tables: sequences of one family (`fan` of them) share the full
    pages that all of them have, each owns the rest."""
    rng, page = random.Random(case["spread"]), case["page"]
    lengths = _ragged(rng, case["sequences"], case["least"], case["longest"])
    rows, used, tokens = [], 0, 0
    for first in range(0, len(lengths), case["fan"]):
        family = lengths[first:first + case["fan"]]
        common = min(family) // page if len(family) > 1 else 0
        shared = list(range(used, used + common))
        used += common
        tokens += common * page
        for length in family:
            more = -(-length // page) - common
            rows.append(shared + list(range(used, used + more)))
            used += more
            tokens += length - common * page
    return lengths, rows, used, tokens


def work(case):
    e = DTYPES[case["dtype"]].itemsize
    heads, kv_heads, width = case["heads"], case["kv_heads"], case["width"]
    if case["op"] == "rotate":
        n = case["tokens"]
        return dict(bytes=2.0 * n * (heads + kv_heads) * width * e + 8.0 * n,
                    flops=3.0 * n * (heads + kv_heads) * case["rotated"])
    if case["op"] == "append":
        new, past = _new_and_past(case)
        n, p = sum(new), 1 if case["pages"] == "e4m3" else e
        copied = sum(t % case["page"] for t in past) if case["fan"] else 0
        row = 2 * kv_heads * width
        return dict(bytes=float(n * (2 * heads * width * e + row * (e + p)) + 2 * copied * row * p),
                    flops=float(3 * n * (heads + kv_heads) * case["rotated"] + 1))
    lengths, _, pages, tokens = _attended(case)
    pairs = sum(lengths)
    return dict(bytes=float(2 * tokens * kv_heads * width + 8 * pages * kv_heads
                            + 2 * case["sequences"] * heads * width * e),
                flops=4.0 * pairs * heads * width + 1.0)


def _frequencies(case):
    """Inverse frequencies of the pairs, fp64; those that turn less than four
    times within a context of 4096 are stretched, those of less than one fully."""
    half = case["rotated"] // 2
    f = 10000.0 ** (-torch.arange(half, dtype=torch.float64, device="cuda") / max(1, half))
    if case["stretch"] != 1.0:
        keep = ((4096 * f / (2 * math.pi) - 1.0) / 3.0).clamp(0.0, 1.0)
        f = f * (keep + (1.0 - keep) / case["stretch"])
    return f


def _pages(gen, shape, dtype, e4m3):
    """A pool of pages [pages, page, heads, width] and their scales (8 bits: powers
    of two, the heads' and pages' values of different sizes), or None."""
    if not e4m3:
        return torch.randn(shape, device="cuda", generator=gen).to(dtype), None
    pool = torch.empty(shape, device="cuda", dtype=E4M3)
    scale = torch.empty(shape[0], shape[2], device="cuda")
    step = max(1, (1 << 28) // max(1, shape[1] * shape[2] * shape[3]))
    for a in range(0, shape[0], step):
        x = torch.randn((min(step, shape[0] - a), *shape[1:]), device="cuda", generator=gen)
        size = torch.randint(-1, 2, (x.shape[0], shape[2]), device="cuda", generator=gen)
        x *= torch.exp2(size.float())[:, None, :, None]
        part, exponent = torch.frexp(x.abs().amax((1, 3)))
        s = torch.exp2((exponent - 9 + (part > 0.875)).float())
        pool[a:a + step] = (x / s[:, None, :, None]).to(E4M3)
        scale[a:a + step] = s
    return pool, scale


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    heads, kv_heads, width = case["heads"], case["kv_heads"], case["width"]
    state = dict(case=case)

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=gen).to(dtype)

    if case["op"] == "rotate":
        # one projection's output holds the three, as a model's does
        qkv = normal(case["tokens"], heads + 2 * kv_heads, width)
        state["query"], state["key"], _ = qkv.split([heads, kv_heads, kv_heads], 1)
        state["frequencies"] = _frequencies(case)
        state["positions"] = torch.randint(0, case["far"] + 1, (case["tokens"],), device="cuda",
                                           generator=gen, dtype=torch.int32)
        return state
    page = case["page"]
    if case["op"] == "append":
        new, past = _new_and_past(case)
        tokens = sum(new) + case["tail"]
        qkv = normal(tokens, heads + 2 * kv_heads, width)
        state["query"], state["key"], state["value"] = qkv.split([heads, kv_heads, kv_heads], 1)
        bounds = [0]
        for n in new:
            bounds.append(bounds[-1] + n)
        state["offsets"] = None
        if not case["longest"] == case["least"] == 1:
            state["offsets"] = torch.tensor(bounds, device="cuda", dtype=torch.int32)
            qkv[bounds[-1]:] = float("nan")              # rows behind the last sequence
        state["frequencies"] = _frequencies(case)
        # the full pages behind are those of a prompt that all share; a last page that is not
        # full is the sequence's own, or, with children, its parent's
        used = max(p // page for p in past)
        rows, sources, tails = [], [], {}
        columns = max(1, max(-(-(p + n) // page) for p, n in zip(past, new)))
        for i, (p, n) in enumerate(zip(past, new)):
            full, last = p // page, -(-(p + n) // page)
            row = list(range(full)) + list(range(used, used + last - full))
            used += last - full
            source = list(row)
            if case["fan"] and p % page:
                parent = i // case["fan"]
                if parent not in tails:
                    tails[parent] = used
                    used += 1
                source[full] = tails[parent]
            rows.append(row + [0] * (columns - len(row)))
            sources.append(source + [0] * (columns - len(source)))
        place = torch.randperm(used + 2, device="cuda", generator=gen, dtype=torch.int32)
        state["block_table"] = place[torch.tensor(rows).cuda()].contiguous()
        state["source_table"] = None
        if case["fan"]:
            state["source_table"] = place[torch.tensor(sources).cuda()].contiguous()
        state["lengths"] = torch.tensor(past, device="cuda", dtype=torch.int32)
        shape = (used + 2, page, kv_heads, width)
        for name in ("key", "value"):
            state[name + "_cache"], state[name + "_scale"] = _pages(
                gen, shape, dtype, case["pages"] == "e4m3")
        return state
    lengths, rows, used, _ = _attended(case)
    columns = max(1, -(-case["longest"] // page))
    place = torch.randperm(used + 2, device="cuda", generator=gen, dtype=torch.int32)
    flat = torch.tensor([r + [0] * (columns - len(r)) for r in rows], dtype=torch.int64)
    state["block_table"] = place[flat.cuda()].contiguous()
    state["lengths"] = torch.tensor(lengths, device="cuda", dtype=torch.int32)
    state["query"] = normal(case["sequences"], heads, width)
    for name in ("key", "value"):
        state[name + "_cache"], state[name + "_scale"] = _pages(
            gen, (used + 2, page, kv_heads, width), dtype, True)
    return state


# ---- the plain forms ---------------------------------------------------------

def _turned(x, positions, state):
    """x [tokens, heads, width] turned by its positions, fp32."""
    case = state["case"]
    n = case["rotated"]
    angle = positions.double()[:, None] * state["frequencies"]
    c = (torch.cos(angle) * case["magnitude"]).float()[:, None]
    s = (torch.sin(angle) * case["magnitude"]).float()[:, None]
    x = x.float()
    r = x[..., :n]
    if case["interleaved"]:
        a, b = r[..., 0::2], r[..., 1::2]
        turned = torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2)
    else:
        a, b = r[..., :n // 2], r[..., n // 2:]
        turned = torch.cat([a * c - b * s, a * s + b * c], -1)
    return torch.cat([turned, x[..., n:]], -1)


def _plain_rotate(state):
    dtype = DTYPES[state["case"]["dtype"]]
    return [_turned(state[n], state["positions"], state).to(dtype) for n in ("query", "key")]


def _held(x):
    """Values held in 8 bits; what is not finite is NaN."""
    x = torch.where(torch.isfinite(x), x, torch.full_like(x, float("nan")))
    return x.clamp(-LARGEST, LARGEST).to(E4M3)


def _plain_append(state):
    case, page, dtype = state["case"], state["case"]["page"], DTYPES[state["case"]["dtype"]]
    lengths, table, offsets = state["lengths"].long(), state["block_table"].long(), state["offsets"]
    if offsets is None:
        offsets = torch.arange(case["sequences"] + 1, device="cuda")
    total = state["key"].shape[0] - case["tail"]
    token = torch.arange(total, device="cuda")
    offsets = offsets.long()
    sequence = torch.searchsorted(offsets, token, right=True) - 1
    position = lengths[sequence] + token - offsets[sequence]
    query = torch.zeros(state["query"].shape, device="cuda", dtype=dtype)
    query[:total] = _turned(state["query"][:total], position, state).to(dtype)
    fresh = {"key": _turned(state["key"][:total], position, state),
             "value": state["value"][:total].float()}
    slot, row = table[sequence, position // page], position % page
    # the rows that are kept of a last page that is not full
    source = table if state["source_table"] is None else state["source_table"].long()
    column = (lengths // page).clamp(max=table.shape[1] - 1)[:, None]
    kept = lengths % page * (offsets[1:] > offsets[:-1])
    tail, origin = table.gather(1, column)[:, 0], source.gather(1, column)[:, 0]
    keep = torch.arange(page, device="cuda") < kept[:, None]
    out = [query]
    for name in ("key", "value"):
        cache, scale = state[name + "_cache"], state[name + "_scale"]
        if scale is None:
            cache[tail] = torch.where(keep[..., None, None], cache[origin], cache[tail])
            cache[slot, row] = fresh[name].to(dtype)
            out.append(cache)
            continue
        # a rotation lengthens a value by at most the square root of 2
        most = 1.0 if name == "value" else max(1.0, 1.41421366 * case["magnitude"])
        top = state[name][:total].float().abs().amax(-1) * most
        need = torch.zeros_like(scale).index_reduce_(0, slot, top, "amax")
        part, exponent = torch.frexp(need)
        need = torch.exp2((exponent - 9 + (part > 0.875)).float().clamp(-118, 119))
        old = scale[origin] * (kept > 0)[:, None]
        before = torch.zeros_like(scale).index_reduce_(0, tail, old, "amax")
        touched = torch.zeros(scale.shape[0], 1, device="cuda", dtype=torch.bool)
        touched[slot] = True
        scale.copy_(torch.where(touched, torch.maximum(need, before), scale))
        ratio = old / scale[tail]
        moved = _held(cache[origin].float() * ratio[:, None, :, None])
        bits = cache.view(torch.uint8)
        bits[tail] = torch.where(keep[..., None, None], moved.view(torch.uint8), bits[tail])
        bits[slot, row] = _held(fresh[name] / scale[slot][..., None]).view(torch.uint8)
        out += [cache, scale]
    return out


def _plain_attend(state):
    case = state["case"]
    n, kv_heads, width = case["sequences"], case["kv_heads"], case["width"]
    group, page = case["heads"] // kv_heads, case["page"]
    columns = state["block_table"].shape[1]
    out = torch.empty(state["query"].shape, device="cuda", dtype=DTYPES[case["dtype"]])
    at = torch.arange(columns * page, device="cuda")
    step = max(1, CHUNK // (columns * page * kv_heads * max(width, group)))
    for a in range(0, n, step):
        b = min(n, a + step)
        slot = state["block_table"][a:b].long()
        q = state["query"][a:b].float().view(b - a, kv_heads, group, width)
        rows = []
        for name in ("key", "value"):
            x = state[name + "_cache"].view(torch.uint8)[slot].view(E4M3).float()
            x = x * state[name + "_scale"][slot][:, :, None, :, None]
            rows.append(x.flatten(1, 2).transpose(1, 2))           # [b, Hkv, T, D]
        scores = torch.matmul(q, rows[0].transpose(2, 3)) / math.sqrt(width)
        seen = at < state["lengths"][a:b, None]
        scores = scores.masked_fill(~seen[:, None, None], float("-inf"))
        top = scores.amax(-1, keepdim=True)
        weight = torch.exp(scores - torch.where(top == float("-inf"), 0.0, top))
        total = weight.sum(-1, keepdim=True)
        weight = weight / torch.where(total > 0, total, 1.0)
        # what is stale behind a sequence's last row may be anything
        values = rows[1].masked_fill(~seen[:, None, :, None], 0.0)
        out[a:b] = torch.matmul(weight, values).flatten(1, 2)
    return out


def run(state):
    op = state["case"]["op"]
    if not own:
        return {"rotate": _plain_rotate, "append": _plain_append, "attend": _plain_attend}[op](state)
    case = state["case"]
    if op == "rotate":
        from graph_rewrite_system_b200.rotary import rotate_positions

        return list(rotate_positions(
            state["query"], state["key"], state["positions"], state["frequencies"],
            interleaved=case["interleaved"], magnitude=case["magnitude"]))
    if op == "append":
        from graph_rewrite_system_b200.token_cache import append_tokens

        query = append_tokens(
            state["key"], state["value"], state["key_cache"], state["value_cache"],
            state["block_table"], state["lengths"], key_scale=state["key_scale"],
            value_scale=state["value_scale"], offsets=state["offsets"],
            source_table=state["source_table"], frequencies=state["frequencies"],
            interleaved=case["interleaved"], magnitude=case["magnitude"], query=state["query"])
        if state["key_scale"] is None:
            return [query, state["key_cache"], state["value_cache"]]
        return [query, state["key_cache"], state["key_scale"], state["value_cache"],
                state["value_scale"]]
    from graph_rewrite_system_b200.quantized_attention import quantized_attention

    return quantized_attention(
        state["query"], state["key_cache"], state["value_cache"], state["key_scale"],
        state["value_scale"], state["block_table"], state["lengths"])


# ---- the definitions in 64 bits ----------------------------------------------

def _as_complex(x, positions, frequencies, case):
    """A rotation of pairs is a product of complex numbers."""
    n = case["rotated"]
    x = x.double()
    pairs = x[..., :n].unflatten(-1, (n // 2, 2) if case["interleaved"] else (2, n // 2))
    first, second = pairs.unbind(-1 if case["interleaved"] else -2)
    angle = positions.double()[:, None, None] * frequencies
    z = torch.complex(first, second) * torch.polar(torch.full_like(angle, case["magnitude"]), angle)
    pairs = torch.stack([z.real, z.imag], -1 if case["interleaved"] else -2)
    return torch.cat([pairs.flatten(-2), x[..., n:]], -1)


def _exact_append(case, s):
    """Page by page, as a list of sequences with their rows; the codes before
    they are rounded."""
    new, past = _new_and_past(case)
    page = case["page"]
    query = torch.zeros(s["query"].shape, device="cuda", dtype=torch.float64)
    pools = {n: s[n + "_cache"].double() for n in ("key", "value")}
    first = 0
    ends = {}
    for b, (n, p) in enumerate(zip(new, past)):
        at = torch.arange(p, p + n, device="cuda")
        rows = slice(first, first + n)
        first += n
        query[rows] = _as_complex(s["query"][rows], at, s["frequencies"], case)
        held = {"key": _as_complex(s["key"][rows], at, s["frequencies"], case),
                "value": s["value"][rows].double()}
        table = s["block_table"][b].tolist()
        source = table if s["source_table"] is None else s["source_table"][b].tolist()
        for column in range(p // page, -(-(p + n) // page) if n else 0):
            low, high = max(p, column * page), min(p + n, (column + 1) * page)
            kept = low - column * page
            to, origin = table[column], source[column]
            for name in ("key", "value"):
                pool, scale = pools[name], s[name + "_scale"]
                fresh = held[name][low - p:high - p]
                before = s[name + "_cache"][origin, :kept].double()
                if scale is None:
                    pool[to, :kept] = before
                    pool[to, kept:kept + high - low] = fresh
                    continue
                most = 1.0 if name == "value" else max(1.0, 1.41421366 * case["magnitude"])
                top = s[name][rows][low - p:high - p].float().abs().amax((0, 2)) * most
                power = torch.ceil(torch.log2(top.double() / LARGEST)).clamp(-118, 119)
                grown = torch.exp2(power)
                if kept:
                    grown = torch.maximum(grown, scale[origin].double())
                    pool[to, :kept] = before * (scale[origin].double() / grown)[:, None]
                pool[to, kept:kept + high - low] = fresh / grown[:, None]
                ends[name, to] = grown
    out = [query]
    for name in ("key", "value"):
        out.append(pools[name])
        if s[name + "_scale"] is not None:
            scale = s[name + "_scale"].double()
            for (which, slot), grown in ends.items():
                if which == name:
                    scale[slot] = grown
            out.append(scale)
    return out


def _exact_attend(case, s):
    group, page = case["heads"] // case["kv_heads"], case["page"]
    lengths, _, _, _ = _attended(case)
    result = torch.zeros(s["query"].shape, device="cuda", dtype=torch.float64)
    for b, length in enumerate(lengths):
        if not length:
            continue
        blocks = s["block_table"][b, :-(-length // page)].long()
        k, v = ((s[n + "_cache"].view(torch.uint8)[blocks].view(E4M3).double()
                 * s[n + "_scale"][blocks].double()[:, None, :, None]).flatten(0, 1)[:length]
                for n in ("key", "value"))
        q = s["query"][b].double().view(case["kv_heads"], group, case["width"])
        logit = torch.einsum("hgd,thd->hgt", q, k) / math.sqrt(case["width"])
        weight = (logit - torch.logsumexp(logit, 2, keepdim=True)).exp()
        result[b] = torch.einsum("hgt,thd->hgd", weight, v).flatten(0, 1)
    return result


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotate":
        return [_as_complex(s[n], s["positions"], s["frequencies"], case) for n in ("query", "key")]
    return (_exact_append if case["op"] == "append" else _exact_attend)(case, s)
