"""Oracle of the rotary positions, the append to paged caches and the attention
over 8-bit pages, in fp64 on the CPU.

No reference counterpart.  Angles are reduced with integers, so any position is
as exact as fp64; results come with what an error bound needs.
"""
from __future__ import annotations

from fractions import Fraction
import math

import torch

from .grouped_attention import _row_attention

E4M3 = torch.float8_e4m3fn


def _arctan(inverse: int, bits: int) -> int:
    """arctan(1 / inverse) * 2^bits by its series."""
    total, term, k = 0, (1 << bits) // inverse, 0
    while term:
        total += term // (2 * k + 1) * (1 if k % 2 == 0 else -1)
        term //= inverse * inverse
        k += 1
    return total


_BITS = 320
_TWO_PI = 8 * (4 * _arctan(5, _BITS) - _arctan(239, _BITS))       # Machin's formula


def angle(position: int, frequency: float) -> float:
    """position * frequency modulo 2 pi, in (-pi, pi]."""
    f = Fraction(frequency) * position
    whole = (f.numerator << _BITS) // f.denominator
    part = whole % _TWO_PI
    if 2 * part > _TWO_PI:
        part -= _TWO_PI
    return float(Fraction(part, 1 << _BITS))


def turn(x, positions, frequencies, interleaved, magnitude=1.0):
    """x [T, H, D] turned, fp64, and the sum of a pair's absolute values at each
    of its elements (zero for those that are copied)."""
    x = x.double()
    out, reach = x.clone(), torch.zeros_like(x)
    half = len(frequencies)
    for t, p in enumerate(positions.tolist()):
        a = torch.tensor([angle(p, f) for f in frequencies.tolist()], dtype=torch.float64)
        c, s = torch.cos(a) * magnitude, torch.sin(a) * magnitude
        i = torch.arange(half)
        u, v = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        out[t][:, u] = x[t][:, u] * c - x[t][:, v] * s
        out[t][:, v] = x[t][:, u] * s + x[t][:, v] * c
        both = (x[t][:, u].abs() + x[t][:, v].abs()) * abs(magnitude)
        reach[t][:, u] = reach[t][:, v] = both
    return out, reach


def turn_bound(out, reach, dtype):
    """fp32 (cos, sin): the reduced angle, at most pi / 4, is rounded three times,
    the series' rest and roundings add less than 2^-23: 5 2^-24 in all; the
    magnitude, a product and a multiply-add round once each; then the output."""
    half = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24
    return 1.01 * (9 * 2.0 ** -24 * reach + half * out.abs() * (reach > 0))


def page_scale(amax: float) -> float:
    """The smallest power of two that holds amax within 448."""
    e = -118
    while e < 119 and amax > 448.0 * 2.0 ** e:
        e += 1
    return 2.0 ** e


def to_e4m3(x):
    """Codes of fp32 values (round to nearest even, at most 448, not finite: NaN)."""
    x = torch.where(torch.isfinite(x), x.float().clamp(-448, 448), torch.tensor(math.nan))
    return x.to(E4M3)


def append_tokens(key, value, key_cache, value_cache, block_table, lengths, *, key_scale=None,
                  value_scale=None, offsets=None, source_table=None, frequencies=None,
                  interleaved=False, magnitude=1.0, positions=None, query=None):
    """What the call leaves: a dict with "query" (fp64 and reach, zero rows for
    tokens of no sequence) and for "key" and "value" the cache (the given one with
    kept rows moved; rows of new tokens as given), `fresh` (bool [pages, page]),
    the new rows' exact values in units of the scale and their reach (fp64, zero
    elsewhere), and the scales (or None).  Bad pages and places are skipped."""
    rows = lengths.shape[0]
    offsets = list(range(rows + 1)) if offsets is None else offsets.tolist()
    tokens = key.shape[0]
    pages, page = key_cache.shape[:2]
    source_table = block_table if source_table is None else source_table
    place = torch.zeros(tokens, dtype=torch.int64)
    mine = torch.zeros(tokens, dtype=torch.bool)
    for b in range(rows):
        for i, t in enumerate(range(offsets[b], offsets[b + 1])):
            place[t], mine[t] = min(max(int(lengths[b]), 0), 1 << 30) + i, True
    turns = place if positions is None else positions
    out = {}
    if query is not None:
        q, reach = turn(query, turns, frequencies, interleaved, magnitude)
        out["query"] = (torch.where(mine[:, None, None], q, 0.0),
                        torch.where(mine[:, None, None], reach, 0.0))
    for name, x, cache, scale in (("key", key, key_cache, key_scale),
                                  ("value", value, value_cache, value_scale)):
        exact, reach = x.double(), torch.zeros_like(x, dtype=torch.float64)
        most = 1.0
        if name == "key" and frequencies is not None:
            exact, reach = turn(x, turns, frequencies, interleaved, magnitude)
            most = max(1.0, 1.41421366 * abs(magnitude))
        after, new_scale = cache.clone(), None if scale is None else scale.clone()
        fresh = torch.zeros(pages, page, dtype=torch.bool)
        real = torch.zeros(cache.shape, dtype=torch.float64)
        real_reach = torch.zeros_like(real)
        for b in range(rows):
            n, past = offsets[b + 1] - offsets[b], int(lengths[b])
            if past < 0 or past > 1 << 30:
                continue
            for column in range(past // page, -(-(past + n) // page) if n else 0):
                if column >= block_table.shape[1]:
                    continue
                to, origin = int(block_table[b, column]), int(source_table[b, column])
                if not 0 <= to < pages:
                    continue
                low, high = max(past, column * page), min(past + n, (column + 1) * page)
                kept = low - column * page
                there = slice(offsets[b] + low - past, offsets[b] + high - past)
                place_ = slice(kept, kept + high - low)
                fresh[to, place_] = True
                if not 0 <= origin < pages:
                    kept = 0
                if scale is None:
                    if kept:
                        after[to, :kept] = cache[origin, :kept]
                    real[to, place_], real_reach[to, place_] = exact[there], reach[there]
                    continue
                for h in range(x.shape[1]):
                    size = x[there, h].float().abs()
                    size = size[torch.isfinite(size)]
                    amax = torch.tensor(0.0) if not len(size) else size.max()
                    s = page_scale(float(amax * torch.tensor(most, dtype=torch.float32)))
                    if kept:
                        before = float(scale[origin, h])
                        s = max(s, before)
                        after[to, :kept, h] = to_e4m3(
                            cache[origin, :kept, h].float() * (before / s)).view(cache.dtype)
                    new_scale[to, h] = s
                    real[to, place_, h] = exact[there, h] / s
                    real_reach[to, place_, h] = reach[there, h] / s
        out[name] = (after, fresh, real, real_reach, new_scale)
    return out


def quantized_attention(query, key_cache, value_cache, key_scale, value_scale, block_table,
                        lengths, *, scale=None):
    """Output, absolute output, score reach and, for the bound, the largest query
    element times the sum of |k| and the largest p * value scale times the sum of
    |codes|; [B, H, ...]."""
    q = query.double()
    batch, heads, width = q.shape
    pages, page, kv_heads, _ = key_cache.shape
    group = heads // kv_heads
    scale = 1.0 / math.sqrt(width) if scale is None else scale
    out, spread, tail = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(q)
    reach, far = (torch.zeros(batch, heads, dtype=torch.float64) for _ in range(2))
    codes = [key_cache.double(), value_cache.double()]
    for b in range(batch):
        room = block_table.shape[1] * page
        at = torch.arange(min(max(int(lengths[b]), 0), room))
        slot = block_table[b, at // page].long() if len(at) else at
        fine = (slot >= 0) & (slot < pages)
        slot, row = slot[fine], at[fine] % page
        if not len(slot):
            continue
        ks, vs = key_scale[slot].double(), value_scale[slot].double()
        for h in range(kv_heads):
            k = codes[0][slot, row, h] * ks[:, h, None]
            c = codes[1][slot, row, h]
            r = slice(h * group, (h + 1) * group)
            out[b, r], spread[b, r], reach[b, r] = _row_attention(q[b, r], k, c * vs[:, h, None],
                                                                  scale)
            p = torch.softmax(q[b, r] @ k.T * scale, -1)
            far[b, r] = q[b, r].abs().amax(-1) * k.abs().sum(-1).max() * abs(scale)
            tail[b, r] = (p * vs[:, h]).amax(-1, keepdim=True) * c.abs().sum(0)
    return out, spread, reach, far, tail


def quantized_bound(results, dtype, width, keys, scales=None):
    """First-order roundings.  Scores: (width + 8) fp32 roundings of the absolute
    sum, twice that for the tensor cores' sums; queries in f16 (bf16 exactly, fp32
    in two parts to 2^-22) but for elements 2^38 below the largest.  Weights: two
    exponentials to 2^-21, f16 once (2^-11) or in two parts (2^-22), and 2^-34 of
    the largest where f16 runs out; the log2 of a value scale that is no power of
    two is rounded at its size.  Sums over `keys`; the output rounds once."""
    out, spread, reach, far, tail = results
    bf16 = dtype == torch.bfloat16
    half = 2.0 ** -8 if bf16 else 2.0 ** -24
    logs = 0.0 if scales is None else float(scales.double().log2().abs().max())
    weight = (2 * (width + 8) * 2.0 ** -24 + (0 if bf16 else 2.0 ** -22)) * reach \
        + 2.0 ** -38 * far
    weight = weight[..., None] + 2 * 2.0 ** -21 + 2 * (keys + 16) * 2.0 ** -24 \
        + (2.0 ** -11 if bf16 else 2.0 ** -22) + 2 * 2.0 ** -24 * logs
    return 1.01 * (weight * spread + 2.0 ** -34 * tail + half * out.abs()) + 1e-30
