"""The operators over long caches from their definitions, in 64 bits on the CPU, token by token."""
import torch

import _decode_ref as ref


class Sequences:
    """A batch as the host sees it: rows' owners, and where the tokens of a sequence lie."""

    def __init__(self, starts, past, max_new, tokens, tables, prefix_table, prefix_len, page, num_pages):
        self.rows = ref.owners(starts, past, max_new, tokens)
        self.tables, self.prefix_table, self.prefix_len, self.page, self.num_pages = tables, prefix_table, prefix_len, page, num_pages
        self.shared = -(-prefix_len // page)
        self.past = [max(p, 0) for p in past]

    def new(self, b):
        return [t for t, o in enumerate(self.rows) if o is not None and o[0] == b]

    def physical(self, b, e):
        """The page of the cache that page e along sequence b is, or None."""
        if e < 0 or e >= self.shared + len(self.tables[b]):
            return None
        p = int(self.prefix_table[e] if e < self.shared else self.tables[b][e - self.shared])
        return p if 0 <= p < self.num_pages else None

    def seen_in(self, b, own, e):
        """How many tokens of page e the token with index `own` sees."""
        if e < self.shared:
            return min(self.page, self.prefix_len - e * self.page)
        return max(0, min(self.page, own + 1 - (e - self.shared) * self.page))

    def pages_seen(self, own, b):
        return self.shared + min(own // self.page + 1, len(self.tables[b]))


def bounds(s, k, old):
    """old: [num_pages, kv_heads, 2, dim]; returns them with the touched pages' made anew."""
    out = old.clone()
    for b in range(len(s.past)):
        rows = s.new(b)
        if not rows:
            continue
        end = s.past[b] + len(rows)
        for e in range(s.past[b] // s.page, (end - 1) // s.page + 1):
            p = s.physical(b, s.shared + e)
            if p is None:
                continue
            keys = k[p, :, :min(s.page, end - e * s.page)]
            out[p, :, 0] = torch.where(keys.isnan(), torch.inf, keys.float()).amin(1).to(k.dtype)
            out[p, :, 1] = torch.where(keys.isnan(), -torch.inf, keys.float()).amax(1).to(k.dtype)
    return out


def pick(s, q, bounds, count, first, last):
    """int32 [tokens, kv_heads, count]; rows without an owner keep -7."""
    tokens, heads, dim = q.shape
    kv_heads = bounds.shape[1]
    group = heads // kv_heads
    out = torch.full((tokens, kv_heads, count), -7, dtype=torch.int32)
    for t, owner in enumerate(s.rows):
        if owner is None:
            continue
        b, own = owner
        n = s.pages_seen(own, b)
        where = [s.physical(b, e) for e in range(n)]
        there = [e for e in range(n) if where[e] is not None]
        for h in range(kv_heads):
            out[t, h] = -1
            if not there:
                continue
            limits = bounds[[where[e] for e in there], h].double()
            x = q[t, h * group:(h + 1) * group].double()[:, None]
            worth = torch.maximum(x * limits[None, :, 0], x * limits[None, :, 1]).sum(-1).amax(0)
            worth[worth.isnan()] = torch.inf
            forced = [e < first or e >= n - last for e in there]
            order = sorted(range(len(there)), key=lambda i: (not forced[i], 0.0 if forced[i] else -float(worth[i]), there[i]))[:count]
            taken = sorted(there[i] for i in order)
            out[t, h, :len(taken)] = torch.tensor(taken, dtype=torch.int32)
    return out


def attend(s, q, k, v, pages, scale):
    """As _decode_ref.attention: outputs, and what errors are relative to; and how many keys the longest row has."""
    tokens, heads, dim = q.shape
    kv_heads = k.shape[1]
    group = heads // kv_heads
    out, weight, products = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape[:2], dtype=torch.float64)
    most = 0
    for t, owner in enumerate(s.rows):
        if owner is None:
            continue
        b, own = owner
        for h in range(kv_heads):
            keys, values = [], []
            for e in pages[t, h].tolist():
                p = s.physical(b, e)
                n = 0 if p is None else s.seen_in(b, own, e)
                if n > 0:
                    keys.append(k[p, h, :n].double())
                    values.append(v[p, h, :n].double())
            if not keys:
                continue
            keys, values = torch.cat(keys), torch.cat(values)
            most = max(most, len(keys))
            for g in range(h * group, (h + 1) * group):
                x = keys @ q[t, g].double() * scale
                w = torch.softmax(x, 0)
                out[t, g], weight[t, g] = w @ values, w @ values.abs()
                products[t, g] = (keys.abs() @ q[t, g].double().abs()).max() * abs(scale)
    return out, weight, products, most


def weigh(s, q, k, weights, scale):
    """The weights [sequences, kv_heads, places] after a call, and how far a result may be: a weight's relative error is that of its exponential and of the sum that it is divided by -- each a score's
    error, dim * 2^-24 of the sum of its products' magnitudes (which 2^24 keeps in powers of e; in powers of two 1.5 times as much), and a few roundings; a sum of n terms adds n * 2^-24 of itself."""
    tokens, heads, dim = q.shape
    kv_heads = k.shape[1]
    group = heads // kv_heads
    out, error = weights.double().clone(), torch.zeros(weights.shape, dtype=torch.float64)
    places = weights.shape[2]
    for b in range(len(s.past)):
        rows = s.new(b)
        if not rows:
            continue
        end = min(s.past[b] + len(rows), places)
        out[b, :, s.past[b]:end] = 0.0
        error[b, :, :end] += 2.0 ** -24 * out[b, :, :end].abs() * (1 + len(rows) * group / 64.0)
        for t in rows:
            own = s.rows[t][1]
            at = [(e, i) for e in range(s.pages_seen(own, b)) if s.physical(b, e) is not None for i in range(s.seen_in(b, own, e))]
            if not at:
                continue
            pages, slots = torch.tensor([s.physical(b, e) for e, _ in at]), torch.tensor([i for _, i in at])
            index = torch.tensor([(e - s.shared) * s.page + i if e >= s.shared else -1 for e, i in at])
            mine = index >= 0
            for h in range(kv_heads):
                keys = k[pages, h, slots].double()
                for g in range(h * group, (h + 1) * group):
                    x = keys @ q[t, g].double() * scale
                    p = torch.softmax(x, 0)
                    products = (keys.abs() @ q[t, g].double().abs()).max() * abs(scale)
                    out[b, h, index[mine]] += p[mine]
                    error[b, h, index[mine]] += 2.0 ** -24 * p[mine] * (3 * dim * float(products) + 2 * len(at) + 64 + len(rows) * group)
    return out, error + 2.0 ** -126


def evict(s_past, tables, num_pages, k, v, weights, keep, first, recent):
    """In place on k, v and weights (CPU); returns kept and the lengths."""
    sequences, kv_heads, places = weights.shape
    page = k.shape[2]
    kept, lengths = torch.full((sequences, kv_heads, keep), -1, dtype=torch.int32), []
    for b in range(sequences):
        n = min(max(s_past[b], 0), places)
        lengths.append(min(n, keep))
        for h in range(kv_heads):
            if n <= keep:
                kept[b, h, :n] = torch.arange(n)
                continue
            w = weights[b, h].tolist()
            order = sorted(range(first, n - recent), key=lambda i: ((0, -w[i]) if w[i] == w[i] else (1, 0.0)) + (i,))[:keep - first - recent]
            stay = sorted(list(range(first)) + order + list(range(n - recent, n)))
            kept[b, h] = torch.tensor(stay, dtype=torch.int32)
            for to, i in enumerate(stay):
                weights[b, h, to] = weights[b, h, i]
                src, dst = int(tables[b][i // page]), int(tables[b][to // page])
                if 0 <= src < num_pages and 0 <= dst < num_pages:
                    k[dst, h, to % page], v[dst, h, to % page] = k[src, h, i % page].clone(), v[src, h, i % page].clone()
    return kept, lengths
