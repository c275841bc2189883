"""The operators that keep a long cache from being read whole and from being kept whole, as cases that can be timed: their plain forms and the framework's kernels.

  bounds   per page and key head the least and the largest value that its keys have in each dimension, for the pages that new tokens went to
  pick     per new token and key head the pages whose bounds allow the largest products with its queries
  attend   attention of each new token over the pages that were picked for it
  weigh    the softmax weights that each token of a sequence gets from the new tokens, added up
  evict    the tokens with the largest of these sums, the first and the most recent ones stay and move together; the rest is gone

Caches are [pages][heads][tokens of a page][head size], one tensor for keys and one for values; a sequence's own tokens lie in the pages that its row of
the page table names, a prefix that all sequences share in those of a table of its own.  Pages are counted along a sequence: the prefix's, then its own.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # A served batch's step: every sequence's last page has one token more.  Latency.
        {"name": "bounds_step_bf16", "kind": "bounds", "dtype": "bf16", "kv_heads": 8, "dim": 128, "page": 64, "sequences": 64, "new": 1, "ragged": False, "past": 4000},
        # Prompts of several requests at once, ragged.
        {"name": "bounds_prompts_f16", "kind": "bounds", "dtype": "f16", "kv_heads": 8, "dim": 64, "page": 32, "sequences": 7, "new": 12000, "ragged": True, "past": 100},
        # Three requests of a small fp32 model: the smallest call.
        {"name": "pick_small_f32", "kind": "pick", "dtype": "f32", "heads": 8, "kv_heads": 2, "dim": 64, "page": 16, "sequences": 3, "new": 1, "ragged": False,
         "past": 900, "prefix": 0, "count": 16, "first": 1, "last": 2},
        # A served batch with long histories.
        {"name": "pick_batch_bf16", "kind": "pick", "dtype": "bf16", "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "sequences": 32, "new": 1, "ragged": False,
         "past": 65536, "prefix": 0, "count": 64, "first": 1, "last": 2},
        # One request's drafted tokens behind a shared document and a history of half a million tokens, three query heads to a key head.
        {"name": "pick_drafts_f16", "kind": "pick", "dtype": "f16", "heads": 24, "kv_heads": 8, "dim": 64, "page": 32, "sequences": 1, "new": 4, "ragged": False,
         "past": 500000, "prefix": 20011, "count": 200, "first": 4, "last": 4},
        # The smallest call's attention.
        {"name": "attend_small_f32", "kind": "attend", "dtype": "f32", "heads": 8, "kv_heads": 2, "dim": 64, "page": 16, "sequences": 3, "new": 1, "ragged": False,
         "past": 900, "prefix": 0, "count": 16},
        # A served batch: a sixteenth of up to 16384 tokens each.
        {"name": "attend_batch_bf16", "kind": "attend", "dtype": "bf16", "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "sequences": 64, "new": 1, "ragged": False,
         "past": 16384, "prefix": 0, "count": 64},
        # Drafted tokens of a few requests behind a shared instruction, small pages.
        {"name": "attend_drafts_f16", "kind": "attend", "dtype": "f16", "heads": 24, "kv_heads": 8, "dim": 128, "page": 16, "sequences": 6, "new": 5, "ragged": True,
         "past": 20000, "prefix": 3001, "count": 100},
        # A served batch's step.
        {"name": "weigh_step_bf16", "kind": "weigh", "dtype": "bf16", "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "sequences": 32, "new": 1, "ragged": False,
         "past": 16384, "prefix": 0},
        # The last tokens of long prompts behind a shared instruction, whose weights decide what is kept of the prompts.
        {"name": "weigh_window_bf16", "kind": "weigh", "dtype": "bf16", "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "sequences": 4, "new": 32, "ragged": False,
         "past": 16000, "prefix": 1001},
        # One request of a small fp32 model.
        {"name": "evict_one_f32", "kind": "evict", "dtype": "f32", "kv_heads": 2, "dim": 64, "page": 16, "sequences": 1, "past": 3000, "keep": 1000, "first": 4, "recent": 100},
        # A batch of long histories, some of which are short enough to stay as they are.
        {"name": "evict_batch_bf16", "kind": "evict", "dtype": "bf16", "kv_heads": 8, "dim": 128, "page": 64, "sequences": 24, "past": 16384, "keep": 4096, "first": 16, "recent": 512},
    ]


def _log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(["bounds", "pick", "pick", "attend", "attend", "weigh", "evict"])
    c = {"kind": kind, "dtype": rng.choice(["f32", "bf16", "bf16", "f16"]), "kv_heads": rng.choice([1, 2, 4, 8, 8]), "dim": rng.choice([64, 128, 128, 256]),
         "page": rng.choice([8, 16, 32, 64, 64, 128])}
    row = c["kv_heads"] * c["dim"]

    def most(values, each, limit):  # how long something may be for the whole of it to stay under `values`
        return max(2, min(limit, values // each))

    if kind == "bounds":
        c["sequences"] = _log_int(rng, 1, 64)
        c["new"] = rng.choice([1, 1, rng.randint(2, 8), _log_int(rng, 8, most(2 ** 25, c["sequences"] * row, 12000))])
        c["ragged"] = c["new"] > 1 and rng.random() < 0.6
        c["past"] = _log_int(rng, 1, most(2 ** 27, c["sequences"] * row, 8000))
        return c
    if kind == "evict":
        c["sequences"] = _log_int(rng, 1, 32)
        c["past"] = _log_int(rng, 2, most(2 ** 27, c["sequences"] * row, 100000))
        c["keep"] = _log_int(rng, 1, c["past"])
        c["first"] = rng.choice([0, min(c["keep"], rng.randint(0, 16))])
        c["recent"] = rng.choice([0, rng.randint(0, c["keep"] - c["first"])])
        return c
    c["heads"] = c["kv_heads"] * rng.choice([1, 2, 3, 4, 4, 8])
    c["prefix"] = rng.choice([0, 0, _log_int(rng, 1, 16000)])
    c["sequences"] = _log_int(rng, 1, 64)
    if kind == "pick":
        c["new"] = rng.choice([1, 1, rng.randint(2, 6)])
        pages = min(most(2 ** 24, c["sequences"] * row, 16000), most(2 ** 31, c["sequences"] * row, 800000) // c["page"])
        c["past"] = _log_int(rng, 48 * c["page"], max(64, pages) * c["page"])  # histories of which most is left out
        c["first"], c["last"] = rng.choice([0, 1, 4]), rng.choice([1, 2, 5])
        c["count"] = c["first"] + c["last"] + _log_int(rng, 4, min(256, c["past"] // (4 * c["page"])))
    elif kind == "attend":
        c["new"] = rng.choice([1, 1, rng.randint(2, 6)])
        each = most(2 ** 27, c["sequences"] * c["new"] * row, 16000)
        c["count"] = max(1, _log_int(rng, 1, each) // c["page"])
        c["past"] = _log_int(rng, 1, most(2 ** 29, c["sequences"] * row, 60000))
    else:
        c["new"] = rng.choice([1, 1, rng.randint(2, 6), _log_int(rng, 8, 64)])
        each = most(2 ** 27, c["sequences"] * row, 32000)
        c["past"] = _log_int(rng, 1, min(each, most(2 ** 27, c["sequences"] * c["new"] * c["heads"], 32000)))
        c["prefix"] = min(c["prefix"], each)
    c["ragged"] = c["new"] > 1 and rng.random() < 0.6
    return c


# ---------------------------------------------------------------- preparation

def _new_tokens(c):
    """Tokens that a ragged batch has in each sequence: fixed by the case, from one to `new`, the last one `new`."""
    n = c["sequences"]
    if not c["ragged"]:
        return [c["new"]] * n
    return [1 + (c["new"] - 1) * ((7 * i + 3) % (n + 1)) // (n + 1) for i in range(n - 1)] + [c["new"]]


def _pages(tokens, page):
    return -(-tokens // page)


def _randn(shape, dtype, gen, scale=1.0):
    t = torch.empty(shape, dtype=dtype, device="cuda")
    return t.normal_(0.0, scale, generator=gen)


def _paged(c, gen, capacity):
    """A cache with room for `capacity` own tokens of each sequence, and its page tables; the pages in any order.  Where only bounds are read, what keys and values hold is left open."""
    page, prefix, sequences = c["page"], c.get("prefix", 0), c["sequences"]
    each, shared = _pages(capacity, page), _pages(prefix, page)
    total = sequences * each + shared
    order = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)
    shape, dtype = (total, c["kv_heads"], page, c["dim"]), DTYPES[c["dtype"]]
    k, v = (torch.empty(shape, dtype=dtype, device="cuda") if c["kind"] == "pick" else _randn(shape, dtype, gen) for _ in range(2))
    return {"k": k, "v": v, "tables": order[:sequences * each].view(sequences, each).contiguous(), "prefix_table": order[sequences * each:].contiguous()}


def _past(c, gen):
    """Own tokens of each sequence: from half of `past` on, the first one all of it."""
    past = torch.randint(c["past"] // 2, c["past"] + 1, (c["sequences"],), generator=gen, device="cuda", dtype=torch.int32)
    past[0] = c["past"]
    return past


def prepare(case, seed):
    c = dict(case)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    kind, dtype, page = c["kind"], DTYPES[c["dtype"]], c["page"]
    s = _paged(c, gen, c["past"] + c.get("new", 0))
    s["past"], s["case"] = _past(c, gen), c
    places = s["tables"].shape[1] * page
    if kind == "evict":
        # what attention leaves: a few tokens with most of the weight
        s["weights"] = torch.rand((c["sequences"], c["kv_heads"], places), generator=gen, device="cuda").pow_(12.0).mul_(40.0)
    else:
        counts = _new_tokens(c)
        starts = [0]
        for n in counts:
            starts.append(starts[-1] + n)
        s["tokens"] = starts[-1]
        s["starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda") if c["ragged"] else None
        if kind != "bounds":
            s["q"] = _randn((starts[-1], c["heads"], c["dim"]), dtype, gen, 1.5)
    if kind == "bounds":
        s["bounds"] = torch.zeros((s["k"].shape[0], c["kv_heads"], 2, c["dim"]), dtype=dtype, device="cuda")
    if kind == "pick":  # as those of a page of normal values
        low = _randn((s["k"].shape[0], c["kv_heads"], c["dim"]), torch.float32, gen, 0.4).sub_(2.0)
        s["bounds"] = torch.stack((low, low + _randn(low.shape, torch.float32, gen, 0.4).abs_().add_(3.6)), 2).to(dtype)
    if kind == "attend":
        # any pages that a token sees, its own one always, as a selection leaves them: in order, and -1 behind
        seq, j = _rows(s)
        shared = _pages(c["prefix"], page)
        seen = shared + (s["past"][seq].long() + j) // page + 1
        key = torch.rand((s["tokens"], c["kv_heads"], shared + s["tables"].shape[1]), generator=gen, device="cuda")
        at = torch.arange(key.shape[2], device="cuda")
        key = torch.where(at == (seen - 1)[:, None, None], 2.0, torch.where(at < seen[:, None, None], key, -1.0))
        value, order = key.topk(min(c["count"], key.shape[2]), -1)
        order = order.masked_fill(value < 0, key.shape[2]).sort(-1).values
        s["pages"] = torch.full((s["tokens"], c["kv_heads"], c["count"]), -1, dtype=torch.int32, device="cuda")
        s["pages"][..., :order.shape[2]] = order.masked_fill(order == key.shape[2], -1).to(torch.int32)
    if kind == "weigh":
        s["weights"] = torch.rand((c["sequences"], c["kv_heads"], places), generator=gen, device="cuda")
    if own:
        from paella_amd import decode, long_cache
        s["cache"] = decode.KVCache(s["k"], s["v"])
        if kind == "evict":
            s["plan"] = long_cache.Evict(s["cache"], c["sequences"], s["tables"].shape[1], c["keep"], first=c["first"], recent=c["recent"])
        else:
            s["batch"] = decode.KVBatch(s["past"], s["tables"], max_new=c["new"], starts=s["starts"], tokens=s["tokens"], prefix_table=s["prefix_table"],
                                        prefix_len=c.get("prefix", 0))
        if kind == "pick":
            s["plan"] = long_cache.PageSelect(c["heads"], s["cache"], s["batch"], c["count"], first=c["first"], last=c["last"])
        if kind == "attend":
            s["plan"] = long_cache.PageAttention(c["heads"], s["cache"], s["batch"], c["count"])
        if kind == "weigh":
            s["plan"] = long_cache.KeyWeights(c["heads"], s["cache"], s["batch"])
    return s


# ---------------------------------------------------------------- the framework's operators

def _run_own(s):
    kind = s["case"]["kind"]
    if kind == "bounds":
        from paella_amd import long_cache
        return {"bounds": long_cache.page_bounds(s["cache"], s["bounds"], s["batch"])}
    if kind == "pick":
        return {"pages": s["plan"](s["q"], s["bounds"], s["cache"], s["batch"])}
    if kind == "attend":
        return {"out": s["plan"](s["q"], s["cache"], s["batch"], s["pages"])}
    if kind == "weigh":
        return {"weights": s["plan"](s["q"], s["cache"], s["batch"], s["weights"])}
    past, kept = s["plan"](s["cache"], s["weights"], s["past"], s["tables"])
    return {"past": past, "kept": kept, "k": s["k"], "v": s["v"], "weights": s["weights"]}


# ---------------------------------------------------------------- plain forms

def _rows(s):
    """(sequence, index among its new tokens) of each row of the batch."""
    c = s["case"]
    starts = s["starts"] if s["starts"] is not None else torch.arange(0, (c["sequences"] + 1) * c["new"], c["new"], dtype=torch.int32, device="cuda")
    row = torch.arange(s["tokens"], device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(starts[1:].contiguous(), row, right=True)
    return seq, (row - starts[seq]).long()


def _counts(s):
    c = s["case"]
    if s["starts"] is None:
        return torch.full((c["sequences"],), c["new"], dtype=torch.int64, device="cuda")
    return (s["starts"][1:] - s["starts"][:-1]).long()


def _bounds(s):
    c = s["case"]
    page, n = c["page"], s["tables"].shape[1]
    past = s["past"].long()
    first, end = past // page, past + _counts(s)
    at = first[:, None] + torch.arange(_pages(c["new"] - 1, page) + 1, device="cuda")  # the pages that new tokens lie in
    held = (end[:, None] - at * page).clamp(max=page)                                   # tokens in each
    seq, which = (held > 0).nonzero(as_tuple=True)
    at, held = at[seq, which], held[seq, which]
    to = s["tables"][seq, at.clamp(max=n - 1)].long()
    k = s["k"][to].float()
    absent = (torch.arange(page, device="cuda") >= held[:, None])[:, None, :, None]
    low, high = k.masked_fill(absent, math.inf).amin(2), k.masked_fill(absent, -math.inf).amax(2)
    s["bounds"][to] = torch.stack((low, high), 2).to(s["bounds"].dtype)
    return {"bounds": s["bounds"]}


def _by_sequence(s, x):
    """Rows [tokens, heads, dim] as [sequences, key heads, new tokens * heads of a key head, dim], with zeros where a sequence has fewer new tokens."""
    c = s["case"]
    seq, j = _rows(s)
    h, g = c["kv_heads"], c["heads"] // c["kv_heads"]
    y = x.new_zeros((c["sequences"], c["new"], h, g, c["dim"]))
    y[seq, j] = x.view(-1, h, g, c["dim"])
    return y.permute(0, 2, 1, 3, 4).reshape(c["sequences"], h, c["new"] * g, c["dim"])


def _pick(s):
    c = s["case"]
    b, n, h, d, page = c["sequences"], c["new"], c["kv_heads"], c["dim"], c["page"]
    g, shared = c["heads"] // h, _pages(c["prefix"], page)
    seq, j = _rows(s)
    table = torch.cat((s["prefix_table"][None].expand(b, -1), s["tables"]), 1).long()
    q = _by_sequence(s, s["q"].double())  # 64 bits: which of two neighbours comes first is decided by their last digits
    q = torch.cat((q.clamp(max=0.0), q.clamp(min=0.0)), -1)
    value = torch.empty((b, h, n, table.shape[1]), dtype=torch.float64, device="cuda")
    for i in range(b):
        bounds = s["bounds"][table[i]].double().permute(1, 2, 3, 0).reshape(h, 2 * d, -1)
        value[i] = torch.matmul(q[i], bounds.contiguous()).view(h, n, g, -1).amax(2)
    value = value.permute(0, 2, 1, 3)[seq, j]
    seen = (shared + (s["past"][seq].long() + j) // page + 1)[:, None, None]
    at = torch.arange(table.shape[1], device="cuda")
    value = value.masked_fill((at < c["first"]) | (at >= seen - c["last"]), math.inf).masked_fill(at >= seen, -math.inf)
    value, order = value.sort(dim=-1, descending=True, stable=True)
    value, order = value[..., :c["count"]], order[..., :c["count"]]
    order = order.masked_fill(value == -math.inf, table.shape[1]).sort(-1).values
    pages = torch.full((s["tokens"], h, c["count"]), -1, dtype=torch.int32, device="cuda")
    pages[..., :order.shape[2]] = order.masked_fill(order == table.shape[1], -1).to(torch.int32)
    return {"pages": pages}


def _attend(s):
    c = s["case"]
    h, d, page = c["kv_heads"], c["dim"], c["page"]
    g, shared = c["heads"] // h, _pages(c["prefix"], page)
    seq, j = _rows(s)
    listed_, at = s["pages"].long(), s["past"][seq].long() + j
    which = listed_.clamp(min=0)
    if shared:
        physical = torch.where(which < shared, s["prefix_table"][which.clamp(max=shared - 1)], s["tables"][seq[:, None, None], (which - shared).clamp(min=0)]).long()
    else:
        physical = s["tables"][seq[:, None, None], which].long()
    # how many of each page's tokens a row sees
    held = torch.where(which < shared, c["prefix"] - which * page, at[:, None, None] + 1 - (which - shared) * page).clamp(0, page)
    held = held.masked_fill(listed_ < 0, 0)
    hidden = (torch.arange(page, device="cuda") >= held[..., None]).flatten(2)
    head = torch.arange(h, device="cuda")[None, :, None]
    k, v = (t[physical, head].float().flatten(2, 3).view(-1, listed_.shape[2] * page, d) for t in (s["k"], s["v"]))
    q = s["q"].float().view(-1, g, d) / math.sqrt(d)
    x = torch.matmul(q, k.transpose(1, 2).contiguous()).masked_fill(hidden.flatten(0, 1)[:, None], -math.inf)
    p = (x - x.amax(-1, keepdim=True)).exp()
    out = torch.matmul(p, v) / p.sum(-1, keepdim=True)
    return {"out": out.view(-1, c["heads"], d).to(s["q"].dtype)}


def _weigh(s):
    c = s["case"]
    b, n, h, d, page = c["sequences"], c["new"], c["kv_heads"], c["dim"], c["page"]
    g = c["heads"] // h
    counts, past = _counts(s), s["past"].long()
    q = _by_sequence(s, s["q"].float()) / math.sqrt(d)
    keys = s["k"][s["tables"].long()].float().transpose(1, 2).reshape(b, h, -1, d)
    at = torch.arange(keys.shape[2], device="cuda")
    row = torch.arange(n, device="cuda")
    x = torch.matmul(q, keys.transpose(2, 3).contiguous())
    hidden = at >= (past[:, None] + row + 1).repeat_interleave(g, 1)[:, :, None]
    x = x.masked_fill_(hidden[:, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    total = 0.0
    if c["prefix"]:
        shared = s["k"][s["prefix_table"].long()].float().transpose(0, 1).reshape(h, -1, d)[:, :c["prefix"]]
        y = torch.matmul(q.transpose(0, 1).reshape(h, -1, d), shared.transpose(1, 2).contiguous()).view(h, b, n * g, -1).transpose(0, 1)
        top = torch.maximum(top, y.amax(-1, keepdim=True))
        total = (y - top).exp().sum(-1, keepdim=True)
    p = (x - top).exp_()
    p = p / (total + p.sum(-1, keepdim=True))
    p = p.masked_fill_((row >= counts[:, None]).repeat_interleave(g, 1)[:, None, :, None], 0.0).sum(2)
    old = torch.where((at < past[:, None])[:, None], s["weights"], 0.0)
    s["weights"].copy_(torch.where((at < (past + counts)[:, None])[:, None], old + p, s["weights"]))
    return {"weights": s["weights"]}


def _evict(s):
    c = s["case"]
    b, h, page, keep = c["sequences"], c["kv_heads"], c["page"], c["keep"]
    past = s["past"].long()[:, None, None]
    at = torch.arange(s["weights"].shape[2], device="cuda")
    rank = s["weights"].masked_fill((at < c["first"]) | (at >= past - c["recent"]), math.inf).masked_fill(at >= past, -math.inf)
    value, order = rank.sort(dim=-1, descending=True, stable=True)
    order = order[..., :keep].masked_fill(value[..., :keep] == -math.inf, at.shape[0]).sort(-1).values
    there = order < at.shape[0]
    source = order.masked_fill(~there, 0)
    to = at[:order.shape[2]].expand_as(source)
    seq, head = torch.arange(b, device="cuda")[:, None, None].expand_as(source), torch.arange(h, device="cuda")[None, :, None].expand_as(source)
    seq, head, source, to = seq[there], head[there], source[there], to[there]
    where, whence = (s["tables"][seq, i // page].long() for i in (to, source))
    for t in (s["k"], s["v"]):
        t[where, head, to % page] = t[whence, head, source % page]
    s["weights"][seq, head, to] = s["weights"][seq, head, source]
    kept = torch.full((b, h, keep), -1, dtype=torch.int32, device="cuda")
    kept[..., :order.shape[2]] = order.masked_fill(~there, -1).to(torch.int32)
    return {"past": s["past"].clamp(max=keep), "kept": kept, "k": s["k"], "v": s["v"], "weights": s["weights"]}


def run(state):
    if own:
        return _run_own(state)
    return {"bounds": _bounds, "pick": _pick, "attend": _attend, "weigh": _weigh, "evict": _evict}[state["case"]["kind"]](state)


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    c = case
    size, row = 4 if c["dtype"] == "f32" else 2, c["kv_heads"] * c["dim"]
    n, page = c["sequences"], c["page"]
    own_tokens = c["past"] + (n - 1) * 0.75 * c["past"]  # lengths are spread evenly from half of the longest on, the first one the longest
    if c["kind"] == "evict":
        long = [max(0.0, min(1.0, (c["past"] - c["keep"]) / max(1.0, 0.5 * c["past"])))] * (n - 1) + [float(c["past"] > c["keep"])]
        moved = sum(long) * max(0, c["keep"] - c["first"])  # the first ones lie where they stay
        return {"bytes": 4.0 * own_tokens * c["kv_heads"] + moved * c["kv_heads"] * (4.0 * c["dim"] * size + 8.0) + 4.0 * n * c["kv_heads"] * c["keep"], "flops": 0.0}
    counts = _new_tokens(c)
    if c["kind"] == "bounds":
        tokens = sum(counts) + n * (min(page, c["past"]) - 1) / 2  # those that the first of the pages holds already
        pages = sum((k + page - 1) / page for k in counts)
        return {"bytes": (tokens + 2.0 * pages) * row * size, "flops": 2.0 * tokens * row}
    rows = sum(counts) * c["heads"] * c["dim"]
    if c["kind"] == "pick":
        pages = _pages(c["prefix"], page) + own_tokens / page
        seen = sum(counts) * _pages(c["prefix"], page) + sum(k * (1.0 if i == 0 else 0.75) * c["past"] / page for i, k in enumerate(counts))
        return {"bytes": 2.0 * pages * row * size + rows * size + 4.0 * sum(counts) * c["kv_heads"] * c["count"], "flops": 4.0 * seen * c["heads"] * c["dim"]}
    if c["kind"] == "attend":
        keys = sum(k * min(c["count"] * page, c["prefix"] + (1.0 if i == 0 else 0.75) * c["past"]) for i, k in enumerate(counts))  # of all rows together
        held = c["prefix"] + own_tokens + sum(counts)  # what rows of one sequence, and the prefix, share is read once
        return {"bytes": 2.0 * min(keys, held) * row * size + 2.0 * rows * size + 4.0 * sum(counts) * c["kv_heads"] * c["count"], "flops": 4.0 * keys * c["heads"] * c["dim"]}
    keys = sum(k * (c["prefix"] + (1.0 if i == 0 else 0.75) * c["past"] + (k + 1) / 2) for i, k in enumerate(counts))
    held = own_tokens + sum(counts)
    return {"bytes": (c["prefix"] + held) * row * size + rows * size + 8.0 * held * c["kv_heads"], "flops": 2.0 * keys * c["heads"] * c["dim"]}


# ---------------------------------------------------------------- in 64 bits, from the definitions

def _exact_bounds(s):
    c = s["case"]
    out, past = s["bounds"].double(), s["past"].tolist()
    for i, n in enumerate(_new_tokens(c)):
        for p in range(past[i] // c["page"], (past[i] + n - 1) // c["page"] + 1):
            where = int(s["tables"][i, p])
            keys = s["k"][where, :, :min(c["page"], past[i] + n - p * c["page"])].double()
            out[where, :, 0], out[where, :, 1] = keys.min(1).values, keys.max(1).values
    return {"bounds": out}


def _exact_attend(s):
    c = s["case"]
    h, d, page, shared = c["kv_heads"], c["dim"], c["page"], _pages(c["prefix"], c["page"])
    past, tables, prefix_table, pages = s["past"].tolist(), s["tables"].tolist(), s["prefix_table"].tolist(), s["pages"].tolist()
    out, t = [], 0
    for i, n in enumerate(_new_tokens(c)):
        for j in range(n):
            for head in range(h):
                which, places = [], []
                for e in pages[t][head]:
                    if e < 0:
                        continue
                    table, index, length = (prefix_table, e, c["prefix"]) if e < shared else (tables[i], e - shared, past[i] + j + 1)
                    which.append(table[index])
                    places.append(min(page, length - index * page))
                at = torch.tensor(which, device="cuda")
                seen = (torch.arange(page, device="cuda") < torch.tensor(places, device="cuda")[:, None]).flatten()
                k, v = (x[at, head].reshape(-1, d)[seen].double() for x in (s["k"], s["v"]))
                q = s["q"][t].view(h, -1, d)[head].double()
                out.append(torch.softmax(q @ k.t().contiguous() / d ** 0.5, -1) @ v)
            t += 1
    return {"out": torch.cat(out).view(t, c["heads"], d)}


def _exact_weigh(s):
    c = s["case"]
    h, d, g = c["kv_heads"], c["dim"], c["heads"] // c["kv_heads"]
    out, past, row = s["weights"].double(), s["past"].tolist(), 0
    prefix = s["k"][s["prefix_table"].long()].double().transpose(1, 2).reshape(-1, h, d)[:c["prefix"]]
    for i, n in enumerate(_new_tokens(c)):
        length = past[i] + n
        keys = s["k"][s["tables"][i, :_pages(length, c["page"])].long()].double().transpose(1, 2).reshape(-1, h, d)[:length]
        keys = torch.cat((prefix, keys))
        reach = c["prefix"] + past[i] + 1 + torch.arange(n, device="cuda").repeat_interleave(g)
        unseen = torch.arange(len(keys), device="cuda")[None] >= reach[:, None]
        out[i, :, past[i]:length] = 0.0
        for head in range(h):
            q = s["q"][row:row + n].view(n, h, g, d)[:, head].reshape(n * g, d).double()
            x = q @ keys[:, head].t().contiguous() / d ** 0.5
            x[unseen] = -math.inf
            out[i, head, :length] += torch.softmax(x, -1)[:, c["prefix"]:].sum(0)
        row += n
    return {"weights": out}


def _exact_evict(s):
    c = s["case"]
    page, keep = c["page"], c["keep"]
    k, v, w = s["k"].double(), s["v"].double(), s["weights"].double()
    for i, n in enumerate(s["past"].tolist()):
        if n <= keep:
            continue
        table = s["tables"][i].long()
        between = slice(c["first"], n - c["recent"])
        middle = keep - c["first"] - c["recent"]
        for head in range(c["kv_heads"]):
            order = torch.sort(s["weights"][i, head, between], descending=True, stable=True).indices[:middle] + c["first"]
            source = torch.cat((torch.arange(c["first"], device="cuda"), order.sort().values, torch.arange(n - c["recent"], n, device="cuda")))
            to = torch.arange(keep, device="cuda")
            for t, old in ((k, s["k"]), (v, s["v"])):
                t[table[to // page], head, to % page] = old[table[source // page], head, source % page].double()
            w[i, head, :keep] = s["weights"][i, head, source].double()
    return {"past": None, "kept": None, "k": k, "v": v, "weights": w}


def exact(case, seed):
    if case["kind"] == "pick":  # whole numbers alone
        return None
    s = prepare(case, seed)
    return {"bounds": _exact_bounds, "attend": _exact_attend, "weigh": _exact_weigh, "evict": _exact_evict}[case["kind"]](s)
