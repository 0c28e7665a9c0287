"""Oracle of the grouped attention operators and the logit adjustment, in fp64.

No reference counterpart.  The attention functions return, beside the output,
what an error bound needs: the same rows with |value| in place of value (the
scale of a relative error of the weights) and the largest sum of |query * key *
scale| of the row (the scale of a rounding error of its scores).
"""
from __future__ import annotations

import math

import torch


def _row_attention(q, k, v, scale):
    """q [G, D], k/v [T, D] -> output, absolute output, score scale."""
    if not k.shape[0]:
        zero = torch.zeros_like(q)
        return zero, zero, torch.zeros(q.shape[0], dtype=torch.float64)
    scores = (q @ k.T) * scale
    weights = torch.softmax(scores, -1)
    reach = (q.abs() @ k.abs().T).amax(-1) * abs(scale)
    return weights @ v, weights @ v.abs(), reach


def prompt_attention(query, key, value, offsets, scale=None):
    """[T, H, D], [T, Hkv, D] twice, list of offsets; rows outside every
    sequence are zero."""
    q, k, v = query.double(), key.double(), value.double()
    tokens, heads, width = q.shape
    group = heads // k.shape[1]
    scale = 1.0 / math.sqrt(width) if scale is None else scale
    out, spread = torch.zeros_like(q), torch.zeros_like(q)
    reach = torch.zeros(tokens, heads, dtype=torch.float64)
    for begin, end in zip(offsets, offsets[1:]):
        for p in range(begin, end):
            for h in range(k.shape[1]):
                rows = slice(h * group, (h + 1) * group)
                out[p, rows], spread[p, rows], reach[p, rows] = _row_attention(
                    q[p, rows], k[begin:p + 1, h], v[begin:p + 1, h], scale)
    return out, spread, reach


def shared_prefix_attention(query, prefix_key, prefix_value, key_cache=None, value_cache=None,
                            block_table=None, lengths=None, *, current_key=None,
                            current_value=None, current_valid=None, scale=None):
    """[B, H, D]; page ids outside the cache hold no keys, lengths are cut to
    the table."""
    q = query.double()
    batch, heads, width = q.shape
    kv_heads = prefix_key.shape[1]
    group = heads // kv_heads
    scale = 1.0 / math.sqrt(width) if scale is None else scale
    out, spread = torch.zeros_like(q), torch.zeros_like(q)
    reach = torch.zeros(batch, heads, dtype=torch.float64)
    for b in range(batch):
        keys, values = [prefix_key], [prefix_value]
        if key_cache is not None:
            page = key_cache.shape[1]
            room = block_table.shape[1] * page
            for t in range(min(max(int(lengths[b]), 0), room)):
                slot = int(block_table[b, t // page])
                if 0 <= slot < key_cache.shape[0]:
                    keys.append(key_cache[slot, t % page][None])
                    values.append(value_cache[slot, t % page][None])
        if current_key is not None and (current_valid is None or bool(current_valid[b])):
            keys.append(current_key[b][None])
            values.append(current_value[b][None])
        k, v = torch.cat(keys).double(), torch.cat(values).double()
        for h in range(kv_heads):
            rows = slice(h * group, (h + 1) * group)
            out[b, rows], spread[b, rows], reach[b, rows] = _row_attention(
                q[b, rows], k[:, h], v[:, h], scale)
    return out, spread, reach


def attention_bound(out, spread, reach, dtype, width, keys):
    """Largest error of an output element, by first-order rounding analysis.

    Scores: products of the inputs summed over `width` terms in fp32 and scaled
    (bf16 products are exact, fp32 ones round) are off by (width + 4) 2^-24
    times the row's sum of |q k scale|, in a natural exponent; the running
    maximum subtracts exactly up to one more such term.  Exponential: 2^-21
    relative; the bf16 kernels round the weights to bf16 (2^-8).  Sums over `keys` weights
    in fp32: keys 2^-24 in the numerator and in the denominator, on partial
    sums no larger than the absolute sums.  The output rounds once (2^-8 or
    2^-24)."""
    half = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24
    weight = 2 * (width + 5) * 2.0 ** -24 * reach[..., None] + 2 * 2.0 ** -21 \
        + 2 * (keys + 8) * 2.0 ** -24
    if dtype == torch.bfloat16:
        weight = weight + 2.0 ** -8
    return 1.01 * (weight * spread + half * out.abs()) + 1e-30


def adjust_logits(logits, *, tokens=None, lengths=None, prompt_lengths=None, repetition=1.0,
                  presence=0.0, frequency=0.0, bias=None, allowed=None, fill=float("-inf")):
    """fp64 [rows, vocab], token by token."""
    x = logits.double().clone()
    rows, vocab = x.shape
    at = lambda knob, b: float(knob[b]) if isinstance(knob, torch.Tensor) else float(knob)
    for b in range(rows):
        seen, count = set(), {}
        if tokens is not None:
            n = tokens.shape[1] if lengths is None else min(max(int(lengths[b]), 0), tokens.shape[1])
            prompt = 0 if prompt_lengths is None else int(prompt_lengths[b])
            for i in range(n):
                v = int(tokens[b, i])
                if 0 <= v < vocab:
                    seen.add(v)
                    if i >= prompt:
                        count[v] = count.get(v, 0) + 1
        for v in seen:
            r = at(repetition, b)
            x[b, v] = x[b, v] / r if x[b, v] > 0 else x[b, v] * r
            if v in count:
                x[b, v] -= at(frequency, b) * count[v] + at(presence, b)
        if bias is not None:
            x[b] += (bias if bias.dim() == 1 else bias[b if bias.shape[0] > 1 else 0]).double()
        if allowed is not None:
            words = allowed if allowed.dim() == 1 else allowed[b if allowed.shape[0] > 1 else 0]
            for v in range(vocab):
                if not (int(words[v // 32]) >> (v % 32)) & 1:
                    x[b, v] = fill
    return x
