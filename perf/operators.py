"""Cases of the operators that serve a prompt and its beams.

Three operators of one decode: ``prompt_attention`` (causal attention over
packed prompts with grouped heads), ``shared_prefix_attention`` (one query per
beam against a long prefix that all beams share and the beam's own pages) and
``adjust_logits`` (repeated-token penalties, biases and grammar masks).

``run`` computes a case with elementary torch operations in fp32, or, where
``own`` is true, through the framework's entry points; ``exact`` computes the
same outputs from the definitions in 64 bits.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
CHUNK = 1 << 28          # score elements the plain forms hold at once


def listed():
    return [
        # one short prompt at this framework's own head layout (8 heads of 32): the smallest call
        dict(name="prompt_one_short", op="prompt", dtype="bf16", heads=8, kv_heads=8, width=32,
             sequences=1, longest=37, least=37, spread=1, tail=0),
        # a serving batch of mixed prompts in one packed buffer, padded behind the last one
        dict(name="prompt_mixed", op="prompt", dtype="bf16", heads=32, kv_heads=8, width=128,
             sequences=16, longest=1500, least=90, spread=2, tail=61),
        # hundreds of very short prompts (classification, tool calls), some of them empty
        dict(name="prompt_many_short", op="prompt", dtype="bf16", heads=16, kv_heads=4, width=64,
             sequences=500, longest=64, least=0, spread=3, tail=0),
        # one long document
        dict(name="prompt_long", op="prompt", dtype="bf16", heads=32, kv_heads=8, width=128,
             sequences=1, longest=16384, least=16384, spread=4, tail=0),
        # the fp32 configuration of this framework's model, four ragged prompts
        dict(name="prompt_fp32", op="prompt", dtype="fp32", heads=8, kv_heads=8, width=32,
             sequences=4, longest=1001, least=100, spread=5, tail=3),
        # a handful of samples of a short prompt: the smallest decode call
        dict(name="prefix_few_beams", op="prefix", dtype="bf16", heads=8, kv_heads=2, width=64,
             beams=5, prefix=129, longest=20, least=0, spread=6, page=16, fan=1, current=True),
        # a batch of requests behind one system prompt
        dict(name="prefix_batch", op="prefix", dtype="bf16", heads=32, kv_heads=8, width=128,
             beams=64, prefix=4099, longest=256, least=0, spread=7, page=16, fan=1, current=True),
        # the widest beam over a long document, beams of one parent sharing their full pages
        dict(name="prefix_wide_beam", op="prefix", dtype="bf16", heads=32, kv_heads=8, width=128,
             beams=512, prefix=16384, longest=128, least=33, spread=8, page=16, fan=4,
             current=True),
        # the fp32 configuration of this framework's model over its 381-key prefix
        dict(name="prefix_fp32", op="prefix", dtype="fp32", heads=8, kv_heads=8, width=32,
             beams=64, prefix=381, longest=64, least=0, spread=9, page=16, fan=1, current=True),
        # one sampled sequence, fp32 logits, every feature on: the smallest step
        dict(name="logits_one_row", op="logits", dtype="fp32", rows=1, vocab=32000, history=300,
             bias="shared", mask=True, permitted=0.5),
        # this framework's beam of 1000 over an odd vocabulary (rows of every alignment)
        dict(name="logits_beam", op="logits", dtype="bf16", rows=1000, vocab=32003, history=64,
             bias="none", mask=True, permitted=0.9),
        # a large batch over a large vocabulary with long histories and a bias per row
        dict(name="logits_large", op="logits", dtype="fp32", rows=256, vocab=150000, history=4096,
             bias="row", mask=False, permitted=1.0),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["prompt", "prefix", "logits"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
    if op == "logits":
        rows = _log_int(rng, 1, 1000)
        vocab = min(_log_int(rng, 90, 150000), 256 * 150000 // rows)
        return dict(op=op, dtype=dtype, rows=rows, vocab=vocab,
                    history=rng.choice([0, _log_int(rng, 1, 4096)]),
                    bias=rng.choice(["none", "shared", "row"]), mask=rng.random() < 0.6,
                    permitted=rng.choice([0.002, 0.5, 0.95]))
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    group = rng.choice([1, 1, 2, 3, 4, 5, 7, 8])
    width = rng.choice([32, 64, 128, 32, 64, 128, 40, 80, 96])
    head = dict(op=op, dtype=dtype, heads=kv_heads * group, kv_heads=kv_heads, width=width)
    if op == "prompt":
        sequences = _log_int(rng, 1, 500)
        most = 16384 if dtype == "bf16" else 2048
        longest = _log_int(rng, 1, most)
        while sequences * longest > 2 * most:
            sequences = max(1, sequences // 2)
        return dict(head, sequences=sequences, longest=longest,
                    least=rng.choice([0, 1, longest // 2, longest]), spread=rng.randrange(1 << 30),
                    tail=rng.choice([0, 0, rng.randrange(1, 200)]))
    beams = _log_int(rng, 1, 1000)
    prefix = rng.choice([0, _log_int(rng, 1, 32768), _log_int(rng, 1, 32768)])
    longest = rng.choice([0, _log_int(rng, 1, 512), _log_int(rng, 1, 512)])
    heads = kv_heads * group
    if not prefix:
        longest = max(longest, 1)
    if dtype == "fp32":
        prefix = min(prefix, 4096)
    while beams * heads * width * (prefix + longest) > 512 * 32 * 128 * 16384:
        beams = max(1, beams // 2)
    return dict(head, beams=beams, prefix=prefix, longest=longest,
                least=rng.choice([0, longest // 2, longest]), spread=rng.randrange(1 << 30),
                page=rng.choice([8, 16, 16, 32, 64]), fan=rng.choice([1, 1, 4]),
                current=rng.random() < 0.7)


def _lengths(case, count):
    """Ragged lengths between least and longest; the longest one is there."""
    rng = random.Random(case["spread"])
    out = [rng.randint(case["least"], case["longest"]) for _ in range(count)]
    out[rng.randrange(count)] = case["longest"]
    return out


def _tables(case, lengths):
    """Pages of each beam: beams of one parent (`fan` of them) share the full
    pages that all of them have, each owns the rest.  Returns the rows of page
    numbers and the count of distinct pages."""
    page, fan = case["page"], case["fan"]
    rows, used = [], 0
    for first in range(0, len(lengths), fan):
        group = lengths[first:first + fan]
        common = min(group) // page if len(group) > 1 else 0
        shared = list(range(used, used + common))
        used += common
        for length in group:
            more = -(-length // page) - common
            rows.append(shared + list(range(used, used + more)))
            used += more
    return rows, used


def work(case):
    if case["op"] == "logits":
        e = DTYPES[case["dtype"]].itemsize
        n = case["rows"] * case["vocab"]
        share = case["permitted"] if case["mask"] else 1.0
        words = case["rows"] * (-(-case["vocab"] // 32)) if case["mask"] else 0
        bias = {"none": 0, "shared": case["vocab"], "row": n}[case["bias"]]
        # a masked logit is written without being read
        read = n * share * e + 4 * (words + bias) + 4 * case["rows"] * case["history"]
        return dict(bytes=read + n * e, flops=4.0 * n)
    e = DTYPES[case["dtype"]].itemsize
    heads, kv_heads, width = case["heads"], case["kv_heads"], case["width"]
    if case["op"] == "prompt":
        lengths = _lengths(case, case["sequences"])
        tokens = sum(lengths)
        pairs = sum(n * (n + 1) // 2 for n in lengths)
        return dict(bytes=2.0 * tokens * (heads + kv_heads) * width * e,
                    flops=4.0 * pairs * heads * width)
    lengths = _lengths(case, case["beams"])
    _, pages = _tables(case, lengths)
    current = case["beams"] if case["current"] else 0
    rows = case["prefix"] + min(pages * case["page"], sum(lengths)) + current
    pairs = case["beams"] * case["prefix"] + sum(lengths) + current
    return dict(bytes=2.0 * (rows * kv_heads + case["beams"] * heads) * width * e,
                flops=4.0 * pairs * heads * width + 1.0)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, device="cuda", generator=gen).mul_(scale).to(dtype)

    state = dict(case=case)
    if case["op"] == "logits":
        rows, vocab, history = case["rows"], case["vocab"], case["history"]
        state["logits"] = normal(rows, vocab, scale=4.0)
        # histories repeat few tokens often, as text does
        u = torch.rand(rows, history, device="cuda", generator=gen)
        state["tokens"] = (vocab * u.pow(4)).to(torch.int32).clamp_(max=vocab - 1)
        state["lengths"] = torch.randint(0, history + 1, (rows,), device="cuda", generator=gen,
                                         dtype=torch.int32)
        state["lengths"][0] = history
        state["prompt_lengths"] = state["lengths"] // 3
        knob = torch.rand(3, rows, device="cuda", generator=gen)
        state["repetition"] = 1.0 + 0.3 * knob[0]
        state["presence"] = knob[1] - 0.3
        state["frequency"] = 0.5 * knob[2]
        state["bias"] = None
        if case["bias"] != "none":
            shape = (vocab,) if case["bias"] == "shared" else (rows, vocab)
            state["bias"] = torch.randn(*shape, device="cuda", generator=gen)
        state["allowed"] = None
        if case["mask"]:
            words = -(-vocab // 32)
            bits = torch.rand(rows, words, 32, device="cuda", generator=gen) < case["permitted"]
            # a grammar that is at its end leaves nothing in its last row
            bits[-1] &= rows == 1
            weight = 1 << torch.arange(32, device="cuda", dtype=torch.int64)
            state["allowed"] = (bits * weight).sum(-1).to(torch.int32)
        return state
    heads, kv_heads, width = case["heads"], case["kv_heads"], case["width"]
    state["scale"] = 1.0 / math.sqrt(width)
    if case["op"] == "prompt":
        lengths = _lengths(case, case["sequences"])
        tokens = sum(lengths) + case["tail"]
        state["bounds"] = [0]
        for n in lengths:
            state["bounds"].append(state["bounds"][-1] + n)
        state["offsets"] = torch.tensor(state["bounds"], device="cuda", dtype=torch.int32)
        # one projection's output holds the three, as a model's does
        qkv = normal(tokens, heads + 2 * kv_heads, width)
        qkv[state["bounds"][-1]:] = float("nan")         # rows behind the last prompt
        state["query"], state["key"], state["value"] = qkv.split([heads, kv_heads, kv_heads], 1)
        return state
    beams, page = case["beams"], case["page"]
    lengths = _lengths(case, beams)
    rows, pages = _tables(case, lengths)
    columns = max(1, -(-case["longest"] // page))
    place = torch.randperm(pages + 3, device="cuda", generator=gen, dtype=torch.int32)
    flat = torch.tensor([r + [0] * (columns - len(r)) for r in rows], dtype=torch.int64)
    state["block_table"] = place[flat.cuda()].contiguous()
    state["lengths"] = torch.tensor(lengths, device="cuda", dtype=torch.int32)
    state["query"] = normal(beams, heads, width)
    state["prefix_key"] = normal(case["prefix"], kv_heads, width)
    state["prefix_value"] = normal(case["prefix"], kv_heads, width)
    state["key_cache"] = normal(pages + 3, page, kv_heads, width)
    state["value_cache"] = normal(pages + 3, page, kv_heads, width)
    state["current"] = {}
    if case["current"]:
        state["current"] = dict(
            current_key=normal(beams, kv_heads, width),
            current_value=normal(beams, kv_heads, width),
            current_valid=torch.rand(beams, device="cuda", generator=gen) < 0.97)
    return state


# ---- the plain forms ---------------------------------------------------------

def _softmax(scores):
    """Softmax over the last dimension; a row of -inf gives zeros."""
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == float("-inf"), torch.zeros_like(top), top)
    weight = torch.exp(scores - top)
    total = weight.sum(-1, keepdim=True)
    return weight / torch.where(total > 0, total, torch.ones_like(total))


def _plain_prompt(state):
    case = state["case"]
    group = case["heads"] // case["kv_heads"]
    out = torch.zeros(state["query"].shape, device="cuda", dtype=DTYPES[case["dtype"]])
    for first, last in zip(state["bounds"], state["bounds"][1:]):
        if first == last:
            continue
        q = state["query"][first:last].float().transpose(0, 1)
        k = state["key"][first:last].float().permute(1, 2, 0).repeat_interleave(group, 0)
        v = state["value"][first:last].float().transpose(0, 1).repeat_interleave(group, 0)
        n = last - first
        step = max(1, CHUNK // (case["heads"] * n))
        for a in range(0, n, step):
            b = min(n, a + step)
            scores = torch.matmul(q[:, a:b], k[:, :, :b]) * state["scale"]
            seen = torch.arange(b, device="cuda") <= torch.arange(a, b, device="cuda")[:, None]
            scores = scores.masked_fill(~seen, float("-inf"))
            out[first + a:first + b] = torch.matmul(_softmax(scores), v[:, :b]).transpose(0, 1)
    return out


def _plain_prefix(state):
    case = state["case"]
    beams, kv_heads, width = case["beams"], case["kv_heads"], case["width"]
    group, page, longest = case["heads"] // kv_heads, case["page"], case["longest"]
    out = torch.empty(state["query"].shape, device="cuda", dtype=DTYPES[case["dtype"]])
    prefix_key = state["prefix_key"].float().permute(1, 2, 0)          # [Hkv, D, N]
    prefix_value = state["prefix_value"].float().transpose(0, 1)       # [Hkv, N, D]
    at = torch.arange(longest, device="cuda")
    total = case["prefix"] + longest + 1
    step = max(1, CHUNK // max(case["heads"] * total, 2 * kv_heads * width * total // 8))
    for a in range(0, beams, step):
        b = min(beams, a + step)
        n = b - a
        q = state["query"][a:b].float().view(n, kv_heads, group, width).transpose(0, 1)
        scores = [torch.matmul(q.reshape(kv_heads, n * group, width), prefix_key)
                  .view(kv_heads, n, group, -1)]
        slot = state["block_table"][a:b].long()[:, at // page]
        keys = state["key_cache"][slot, at % page].float()             # [n, T, Hkv, D]
        values = state["value_cache"][slot, at % page].float()
        seen = at < state["lengths"][a:b, None]
        if state["current"]:
            keys = torch.cat([keys, state["current"]["current_key"][a:b, None].float()], 1)
            values = torch.cat([values, state["current"]["current_value"][a:b, None].float()], 1)
            seen = torch.cat([seen, state["current"]["current_valid"][a:b, None]], 1)
        suffix = torch.matmul(q, keys.permute(2, 0, 3, 1))             # [Hkv, n, G, T]
        scores.append(suffix.masked_fill(~seen[None, :, None], float("-inf")))
        scores = torch.cat(scores, -1) * state["scale"]
        if not scores.shape[-1]:
            out[a:b] = 0
            continue
        weight = _softmax(scores)
        head, rest = weight.split([case["prefix"], weight.shape[-1] - case["prefix"]], -1)
        got = torch.matmul(head.reshape(kv_heads, n * group, -1), prefix_value)
        got = got.view(kv_heads, n, group, width) + torch.matmul(rest, values.permute(2, 0, 1, 3))
        out[a:b] = got.transpose(0, 1).reshape(n, case["heads"], width)
    return out


def _plain_logits(state):
    case = state["case"]
    rows, vocab, history = case["rows"], case["vocab"], case["history"]
    x = state["logits"].float()
    at = torch.arange(history, device="cuda")
    seen = (at < state["lengths"][:, None]).float()
    new = seen * (at >= state["prompt_lengths"][:, None])
    token = state["tokens"].long()
    zero = torch.zeros(rows, vocab, device="cuda")
    times = zero.scatter_add(1, token, seen)
    count = zero.scatter_add_(1, token, new)
    r = state["repetition"][:, None]
    x = torch.where(times > 0, torch.where(x > 0, x / r, x * r), x)
    x = x - state["frequency"][:, None] * count - state["presence"][:, None] * (count > 0)
    if state["bias"] is not None:
        x = x + state["bias"]
    if state["allowed"] is not None:
        bit = torch.arange(32, device="cuda", dtype=torch.int32)
        allowed = ((state["allowed"][:, :, None] >> bit) & 1).view(rows, -1)[:, :vocab] != 0
        x = x.masked_fill(~allowed, float("-inf"))
    return x.to(DTYPES[case["dtype"]])


def run(state):
    op = state["case"]["op"]
    if not own:
        return {"prompt": _plain_prompt, "prefix": _plain_prefix, "logits": _plain_logits}[op](state)
    if op == "prompt":
        from graph_rewrite_system_b200.prompt_attention import prompt_attention

        return prompt_attention(state["query"], state["key"], state["value"], state["offsets"],
                                scale=state["scale"])
    if op == "prefix":
        from graph_rewrite_system_b200.prefix_attention import shared_prefix_attention

        return shared_prefix_attention(
            state["query"], state["prefix_key"], state["prefix_value"], state["key_cache"],
            state["value_cache"], state["block_table"], state["lengths"], scale=state["scale"],
            **state["current"])
    from graph_rewrite_system_b200.token_logits import adjust_logits

    return adjust_logits(
        state["logits"], tokens=state["tokens"], lengths=state["lengths"],
        prompt_lengths=state["prompt_lengths"], repetition=state["repetition"],
        presence=state["presence"], frequency=state["frequency"], bias=state["bias"],
        allowed=state["allowed"])


# ---- the definitions in 64 bits ----------------------------------------------

def _exact_prompt(case, s):
    group = case["heads"] // case["kv_heads"]
    result = torch.zeros(s["query"].shape, device="cuda", dtype=torch.float64)
    for j in range(case["sequences"]):
        rows = slice(s["bounds"][j], s["bounds"][j + 1])
        n = rows.stop - rows.start
        for h in range(case["heads"] if n else 0):
            k = s["key"][rows, h // group].double()
            v = s["value"][rows, h // group].double()
            for a in range(0, n, 4096):
                b = min(n, a + 4096)
                q = s["query"][rows.start + a:rows.start + b, h].double()
                logit = (q @ k[:b].T) * s["scale"]
                logit += torch.full((b - a, b), -math.inf, device="cuda",
                                    dtype=torch.float64).triu(a + 1)
                norm = torch.logsumexp(logit, 1)
                result[rows.start + a:rows.start + b, h] = (logit - norm[:, None]).exp() @ v[:b]
    return result


def _exact_prefix(case, s):
    group, page = case["heads"] // case["kv_heads"], case["page"]
    lengths = _lengths(case, case["beams"])
    result = torch.zeros(s["query"].shape, device="cuda", dtype=torch.float64)
    pk, pv = s["prefix_key"].double(), s["prefix_value"].double()
    valid = s["current"]["current_valid"].tolist() if s["current"] else None
    for b, length in enumerate(lengths):
        # the beam's own rows, in order, behind the shared ones
        blocks = s["block_table"][b, :-(-length // page)].long()
        k = [pk, s["key_cache"][blocks].flatten(0, 1)[:length].double()]
        v = [pv, s["value_cache"][blocks].flatten(0, 1)[:length].double()]
        if valid is not None and valid[b]:
            k.append(s["current"]["current_key"][b:b + 1].double())
            v.append(s["current"]["current_value"][b:b + 1].double())
        k, v = torch.cat(k), torch.cat(v)
        if not k.shape[0]:
            continue
        q = s["query"][b].double().view(case["kv_heads"], group, case["width"])
        logit = torch.einsum("hgd,thd->hgt", q, k) * s["scale"]
        weight = (logit - torch.logsumexp(logit, 2, keepdim=True)).exp()
        result[b] = torch.einsum("hgt,thd->hgd", weight, v).flatten(0, 1)
    return result


def _exact_logits(case, s):
    vocab = case["vocab"]
    result = torch.empty(case["rows"], vocab, device="cuda", dtype=torch.float64)
    lengths, prompts = s["lengths"].tolist(), s["prompt_lengths"].tolist()
    for b in range(case["rows"]):
        x = s["logits"][b].double()
        history = s["tokens"][b, :lengths[b]].long()
        seen = torch.bincount(history, minlength=vocab) > 0
        count = torch.bincount(history[prompts[b]:], minlength=vocab).double()
        factor = torch.where(x > 0, 1 / s["repetition"][b].double(), s["repetition"][b].double())
        x = torch.where(seen, x * factor, x)
        x -= s["frequency"][b].double() * count + s["presence"][b].double() * count.clamp(max=1)
        if s["bias"] is not None:
            x += (s["bias"] if s["bias"].dim() == 1 else s["bias"][b]).double()
        if s["allowed"] is not None:
            v = torch.arange(vocab, device="cuda")
            x[(s["allowed"][b].long()[v // 32] >> (v % 32)) % 2 == 0] = -math.inf
        result[b] = x
    return result


def exact(case, seed):
    form = {"prompt": _exact_prompt, "prefix": _exact_prefix, "logits": _exact_logits}[case["op"]]
    return form(case, prepare(case, seed))
