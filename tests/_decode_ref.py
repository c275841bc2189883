"""The operators of a decoding step from their definitions, in 64 bits on the CPU, element by element where that is shortest."""
import math

import numpy as np
import torch

HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def owners(starts, past, max_new, tokens):
    """(sequence, own index) of each row, or None for rows that belong to no sequence."""
    rows = [None] * tokens
    for b in range(len(past)):
        first, end = (b * max_new, (b + 1) * max_new) if starts is None else (starts[b], starts[b + 1])
        for j in range(min(end - first, max_new)):
            rows[first + j] = (b, max(past[b], 0) + j)
    return rows


def norm_rotate(x, weight, eps, inv_freq, interleaved, position):
    """x: float64 [heads, dim]."""
    x = x.clone()
    if weight is not None:
        x = x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt() * weight
    half = 0 if inv_freq is None else len(inv_freq)
    y = x.clone()
    for i in range(half):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        c, s = math.cos(position * inv_freq[i]), math.sin(position * inv_freq[i])
        y[:, a], y[:, b] = x[:, a] * c - x[:, b] * s, x[:, b] * c + x[:, a] * s
    return y


def gather(cache, table, count):
    """Keys or values of the first `count` tokens of a table: float64 [count, heads, dim], and which of them are in a page of the cache."""
    pages, heads, size, dim = cache.shape
    out, there = torch.zeros((count, heads, dim), dtype=torch.float64), torch.zeros(count, dtype=torch.bool)
    for i in range(count):
        if i // size < len(table) and 0 <= table[i // size] < pages:
            out[i] = cache[table[i // size], :, i % size].double()
            there[i] = True
    return out, there


def attention(q, k, v, rows, tables, prefix_table, prefix_len, scale):
    """q [tokens, heads, dim] on the CPU.  Returns the outputs, and per row and head what errors are relative to: the weighted mean of |v| and the largest sum of |q k| * scale."""
    heads, dim = q.shape[1:]
    per_kv = heads // k.shape[1]
    shared = [gather(t, prefix_table, prefix_len) for t in (k, v)]
    out = torch.zeros(q.shape, dtype=torch.float64)
    weight, products = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape[:2], dtype=torch.float64)
    held = {}
    for t, owner in enumerate(rows):
        if owner is None:
            continue
        b, own = owner
        if b not in held or held[b][0][0].shape[0] < own + 1:
            most = max(o[1] for o in rows if o is not None and o[0] == b) + 1
            held[b] = [gather(x, tables[b], most) for x in (k, v)]
        keys = torch.cat((shared[0][0], held[b][0][0][:own + 1]))
        values = torch.cat((shared[1][0], held[b][1][0][:own + 1]))
        there = torch.cat((shared[0][1], held[b][0][1][:own + 1]))
        keys, values = keys[there], values[there]
        if not len(keys):
            continue
        for h in range(heads):
            x = keys[:, h // per_kv] @ q[t, h].double() * scale
            p = torch.softmax(x, 0)
            out[t, h] = p @ values[:, h // per_kv]
            weight[t, h] = p @ values[:, h // per_kv].abs()
            products[t, h] = (keys[:, h // per_kv].abs() @ q[t, h].double().abs()).max() * abs(scale)
    return out, weight, products


def attention_bound(out, weight, products, dtype, keys):
    """How far a result may be: its own rounding; that of the probabilities to the type that the second product takes them in (fp32: none), each at most half a step, in the weighted
    sum; and what 32-bit sums add -- a score of dim products is off by dim * 2^-24 of the sum of their magnitudes, which is the relative error of its probability above and below the
    line, and a sum of n terms by n * 2^-24."""
    dim = out.shape[-1]
    p = 0.0 if dtype == torch.float32 else HALF_STEP[dtype]
    f32 = 2.0 ** -24 * (2 * dim * products[..., None] + 2 * keys + 64)
    tiny = 2.0 ** -24 if dtype == torch.float16 else 0.0   # fp16's smallest step, of outputs and of probabilities
    return HALF_STEP[dtype] * out.abs() + (p + f32) * weight * 1.01 + tiny * (1 + weight * keys)


def select(logits, scores, finished, pad, count):
    """Lists of (value, parent, token) per group; -inf, -1, -1 where there is no continuation left."""
    groups, beams, vocab = logits.shape
    res = []
    for g in range(groups):
        cand = []
        for w in range(beams):
            s = float(scores[g, w])
            if finished is not None and finished[g, w]:
                cand.append((s, w, pad))
                continue
            x = logits[g, w].double().numpy().copy()
            x[np.isnan(x)] = -np.inf
            if np.isposinf(x).any() or np.isneginf(x).all():
                continue
            top = x.max()
            value = s + (x - (top + math.log(np.exp(x - top).sum())))
            best = np.lexsort((np.arange(vocab), -value))[:count]
            cand += [(float(value[t]), w, int(t)) for t in best]
        cand = [c for c in cand if math.isfinite(c[0])]
        cand.sort(key=lambda c: (-c[0], c[1] * vocab + c[2]))
        res.append((cand + [(-math.inf, -1, -1)] * count)[:count])
    return res


def reorder(k, v, parents, past, tables, spare, tables_out):
    """In place on k, v and tables_out (CPU); returns the children's lengths."""
    groups, count = parents.shape
    beams, size, pages = len(past) // groups, k.shape[2], k.shape[0]
    old_k, old_v = k.clone(), v.clone()
    out = []
    for g in range(groups):
        for c in range(count):
            p, row = int(parents[g, c]), g * count + c
            if not 0 <= p < beams:
                out.append(0)
                continue
            n = max(int(past[g * beams + p]), 0)
            full, rest = divmod(n, size)
            out.append(n)
            tables_out[row, :full] = tables[g * beams + p, :full]
            if full >= tables.shape[1]:
                continue
            last = int(tables[g * beams + p, full])
            first = p not in [int(x) for x in parents[g, :c]]
            if rest and first:
                tables_out[row, full] = last
                continue
            tables_out[row, full] = spare[row]
            if rest and 0 <= last < pages and 0 <= int(spare[row]) < pages:
                k[spare[row], :, :rest], v[spare[row], :, :rest] = old_k[last, :, :rest], old_v[last, :, :rest]
    return out
