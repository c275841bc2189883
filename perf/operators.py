"""The operators of a decoding step over a paged cache, as cases that can be timed: their plain forms and the framework's kernels.

  append   the new tokens' queries and keys normed per head and rotated to their positions, keys and values stored in the cache
  attend   attention of a batch that shares a prefix: every new token over the prefix and its own sequence's tokens
  select   beam search: the best continuations over a group's beams and the vocabulary, from logits
  reorder  beam search: the beams' page tables and half-filled pages after a selection

Caches are [pages][heads][tokens of a page][head size], one tensor for keys and one for values; a sequence's own tokens lie in the pages
that its row of the page table names, the shared prefix in those of a table of its own.  Position of a sequence's own token i: prefix + i.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-6


def listed():
    return [
        # One token each for a few sequences of a small model in fp32, no norms: the smallest call, latency.
        {"name": "append_token_f32", "kind": "append", "dtype": "f32", "heads": 8, "kv_heads": 2, "dim": 64, "rotary": 64, "interleaved": False, "norm": False,
         "page": 16, "sequences": 4, "new": 1, "ragged": False, "past": 300, "prefix": 0},
        # A served batch's step: 64 sequences, a token each, behind a prefix of some thousand tokens.
        {"name": "append_step_bf16", "kind": "append", "dtype": "bf16", "heads": 32, "kv_heads": 8, "dim": 128, "rotary": 128, "interleaved": False, "norm": True,
         "page": 64, "sequences": 64, "new": 1, "ragged": False, "past": 2000, "prefix": 6001},
        # Prompts of several requests at once, ragged, positions that pass 100000.
        {"name": "append_prompts_bf16", "kind": "append", "dtype": "bf16", "heads": 32, "kv_heads": 8, "dim": 128, "rotary": 64, "interleaved": True, "norm": True,
         "page": 64, "sequences": 7, "new": 2500, "ragged": True, "past": 100, "prefix": 131000},
        # Three requests of a small fp32 model behind a short instruction: the smallest call.
        {"name": "attend_small_f32", "kind": "attend", "dtype": "f32", "heads": 8, "kv_heads": 2, "dim": 64, "page": 16, "sequences": 3, "new": 1, "ragged": False,
         "past": 40, "prefix": 333},
        # Beams of one request: eight hypotheses over one prompt, few tokens of their own, a key head per query head.
        {"name": "attend_beams_f16", "kind": "attend", "dtype": "f16", "heads": 16, "kv_heads": 16, "dim": 64, "page": 32, "sequences": 8, "new": 1, "ragged": False,
         "past": 100, "prefix": 2011},
        # A served batch under a common instruction; several drafted tokens each, checked at once.
        {"name": "attend_drafts_bf16", "kind": "attend", "dtype": "bf16", "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "sequences": 32, "new": 5, "ragged": True,
         "past": 1000, "prefix": 8190},
        # Many requests about one long document.
        {"name": "attend_document_bf16", "kind": "attend", "dtype": "bf16", "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "sequences": 64, "new": 1, "ragged": False,
         "past": 4000, "prefix": 65536},
        # One request with four beams over a middling vocabulary: latency.
        {"name": "select_one_f32", "kind": "select", "dtype": "f32", "groups": 1, "beams": 4, "vocab": 32000, "count": 4, "finished": False},
        # A batch of requests with four beams each over a large vocabulary, twice as many candidates as beams.
        {"name": "select_batch_bf16", "kind": "select", "dtype": "bf16", "groups": 32, "beams": 4, "vocab": 131072, "count": 8, "finished": False},
        # Wide beams, some of which have ended, over a vocabulary of odd size.
        {"name": "select_wide_f32", "kind": "select", "dtype": "f32", "groups": 4, "beams": 16, "vocab": 50021, "count": 32, "finished": True},
        # One request's four beams.
        {"name": "reorder_one_f32", "kind": "reorder", "dtype": "f32", "kv_heads": 2, "dim": 64, "page": 16, "groups": 1, "beams": 4, "count": 4, "parents": 2, "past": 90},
        # A batch's beams, long hypotheses, large pages.
        {"name": "reorder_batch_bf16", "kind": "reorder", "dtype": "bf16", "kv_heads": 8, "dim": 128, "page": 64, "groups": 32, "beams": 8, "count": 8, "parents": 3,
         "past": 700},
    ]


def _log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(["append", "attend", "attend", "select", "reorder"])
    dtype = rng.choice(["f32", "bf16", "bf16", "f16"])
    kv_heads = rng.choice([1, 2, 4, 8, 8])
    dim = rng.choice([64, 128, 128, 256])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 4, 8])
    page = rng.choice([8, 16, 32, 64, 64, 128])
    prefix = rng.choice([0, _log_int(rng, 1, 32000), _log_int(rng, 100, 32000)])

    def most(values, each, limit):  # how long something may be for the whole of it to stay under `values`
        return max(2, min(limit, values // each))

    if kind == "append":
        sequences = _log_int(rng, 1, 64)
        new = rng.choice([1, 1, _log_int(rng, 2, most(60_000_000, sequences * (heads + 2 * kv_heads) * dim, 12000))])
        return {"kind": kind, "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "dim": dim, "rotary": dim // rng.choice([1, 1, 2, 4]),
                "interleaved": rng.random() < 0.3, "norm": rng.random() < 0.7, "page": page, "sequences": sequences, "new": new,
                "ragged": new > 1 and rng.random() < 0.6, "past": _log_int(rng, 1, most(2 ** 26, sequences * kv_heads * dim, 2000)), "prefix": prefix}
    if kind == "attend":
        sequences = _log_int(rng, 1, 96)
        new = rng.choice([1, 1, rng.randint(2, 8)])
        rows = sequences * new * heads * dim
        return {"kind": kind, "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page, "sequences": sequences, "new": new,
                "ragged": new > 1 and rng.random() < 0.6, "past": _log_int(rng, 1, min(most(2 ** 26, sequences * kv_heads * dim, 6000), most(10 ** 10, rows, 6000))),
                "prefix": min(prefix, 10 ** 10 // rows)}
    if kind == "select":
        groups, beams = _log_int(rng, 1, 32), rng.choice([1, 2, 3, 4, 5, 8, 16])
        return {"kind": kind, "dtype": dtype, "groups": groups, "beams": beams, "vocab": _log_int(rng, 200, most(2 ** 23, groups * beams, 150000)),
                "count": beams * rng.choice([1, 1, 2]), "finished": rng.random() < 0.3}
    groups, beams = _log_int(rng, 1, 32), rng.choice([2, 3, 4, 8, 16])
    return {"kind": kind, "dtype": dtype, "kv_heads": kv_heads, "dim": dim, "page": page, "groups": groups, "beams": beams, "count": beams,
            "parents": rng.randint(1, beams), "past": _log_int(rng, 1, most(2 ** 26, groups * beams * kv_heads * dim, 2000))}


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


def _paged(c, gen, sequences, capacity, spare=0):
    """A cache with room for `capacity` own tokens of each sequence, its page table, and `spare` further pages; the pages in any order."""
    page, prefix = c["page"], c.get("prefix", 0)
    each, shared = _pages(capacity, page), _pages(prefix, page)
    total = sequences * each + shared + spare
    order = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)
    shape = (total, c["kv_heads"], page, c["dim"])
    s = {"k": _randn(shape, DTYPES[c["dtype"]], gen), "v": _randn(shape, DTYPES[c["dtype"]], gen),
         "tables": order[:sequences * each].view(sequences, each).contiguous(), "prefix_table": order[sequences * each:sequences * each + shared].contiguous(),
         "spare": order[sequences * each + shared:].contiguous()}
    return s


def _past(c, gen, sequences):
    """Own tokens of each sequence: anything up to `past`, the first one all of it."""
    past = torch.randint(0, c["past"] + 1, (sequences,), generator=gen, device="cuda", dtype=torch.int32)
    past[0] = c["past"]
    return past


def prepare(case, seed):
    c = dict(case)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    kind, dtype = c["kind"], DTYPES[c["dtype"]]
    if kind in ("append", "attend"):
        counts = _new_tokens(c)
        tokens = sum(counts)
        s = _paged(c, gen, c["sequences"], c["past"] + c["new"])
        s["past"] = _past(c, gen, c["sequences"])
        starts = [0]
        for n in counts:
            starts.append(starts[-1] + n)
        s["starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda") if c["ragged"] else None
        if kind == "append":
            # queries, keys and values side by side, as one projection leaves them
            qkv = _randn((tokens, c["heads"] + 2 * c["kv_heads"], c["dim"]), dtype, gen)
            s["q"], s["kn"], s["vn"] = qkv[:, :c["heads"]], qkv[:, c["heads"]:c["heads"] + c["kv_heads"]], qkv[:, c["heads"] + c["kv_heads"]:]
            s["inv_freq"] = torch.tensor([10000.0 ** (-2.0 * i / c["rotary"]) for i in range(c["rotary"] // 2)], dtype=torch.float32, device="cuda")
            s["q_norm"] = s["k_norm"] = None
            if c["norm"]:
                s["q_norm"], s["k_norm"] = (_randn((c["dim"],), torch.float32, gen, 0.2) + 1.0 for _ in range(2))
        else:
            s["q"] = _randn((tokens, c["heads"], c["dim"]), dtype, gen, 1.5)
    elif kind == "select":
        # a language model's logits: most tokens unlikely, a few far ahead of the rest
        x = _randn((c["groups"], c["beams"], c["vocab"]), torch.float32, gen, 2.0)
        x += torch.rand(x.shape, generator=gen, device="cuda").pow_(24.0).mul_(9.0)
        s = {"logits": x.to(dtype), "scores": _randn((c["groups"], c["beams"]), torch.float32, gen).abs_().mul_(-2.0)}
        s["finished"] = None
        if c["finished"]:
            s["finished"] = (torch.rand((c["groups"], c["beams"]), generator=gen, device="cuda") < 0.25).to(torch.uint8)
    else:
        rows = c["groups"] * c["beams"]
        s = _paged(c, gen, rows, c["past"] + 1, spare=c["groups"] * c["count"])
        s["past"] = _past(c, gen, c["groups"])[:, None].expand(c["groups"], c["beams"]).reshape(-1).contiguous()  # beams of one request are equally long
        # `parents` of the beams survive, each of them at least once, in any order
        alive = torch.rand((c["groups"], c["beams"]), generator=gen, device="cuda").argsort(1)[:, :c["parents"]]
        pick = torch.randint(0, c["parents"], (c["groups"], c["count"]), generator=gen, device="cuda")
        pick[:, :c["parents"]] = torch.arange(c["parents"], device="cuda")
        shuffle = torch.rand((c["groups"], c["count"]), generator=gen, device="cuda").argsort(1)
        s["parents"] = alive.gather(1, pick.gather(1, shuffle)).to(torch.int32).contiguous()
        s["tables_out"] = torch.full((c["groups"] * c["count"], s["tables"].shape[1]), -1, dtype=torch.int32, device="cuda")
    s["case"] = c
    if own:
        from paella_amd import decode
        if kind != "select":
            s["cache"] = decode.KVCache(s["k"], s["v"])
        if kind in ("append", "attend"):
            s["batch"] = decode.KVBatch(s["past"], s["tables"], max_new=c["new"], starts=s["starts"], tokens=tokens, prefix_table=s["prefix_table"],
                                        prefix_len=c["prefix"])
        if kind == "attend":
            s["attend"] = decode.PrefixAttention(c["heads"], s["cache"], s["batch"])
        if kind == "select":
            s["select"] = decode.BeamSelect(c["groups"], c["beams"], c["vocab"], c["count"], dtype)
    return s


# ---------------------------------------------------------------- the framework's operators

def _run_own(s):
    from paella_amd import decode
    kind = s["case"]["kind"]
    if kind == "append":
        q = decode.kv_append(s["cache"], s["batch"], s["kn"], s["vn"], q=s["q"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS, inv_freq=s["inv_freq"],
                             interleaved=s["case"]["interleaved"])
        return {"q": q, "k": s["k"], "v": s["v"]}
    if kind == "attend":
        return {"out": s["attend"](s["q"], s["cache"], s["batch"])}
    if kind == "select":
        scores, parents, tokens = s["select"](s["logits"], s["scores"], finished=s["finished"], pad_token=1)
        return {"scores": scores, "parents": parents, "tokens": tokens}
    past = decode.beam_reorder(s["cache"], s["parents"], s["past"], s["tables"], s["tables_out"], s["spare"])
    return {"past": past, "tables": s["tables_out"], "k": s["k"], "v": s["v"]}


# ---------------------------------------------------------------- plain forms

def _rows(s):
    """(sequence, index among its new tokens) of each row of the batch."""
    c = s["case"]
    starts = s["starts"] if s["starts"] is not None else torch.arange(0, (c["sequences"] + 1) * c["new"], c["new"], dtype=torch.int32, device="cuda")
    row = torch.arange(s["q"].shape[0], device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(starts[1:].contiguous(), row, right=True)
    return seq, (row - starts[seq]).long()


def _rotate(x, cos, sin, rotary, interleaved):
    r = x[..., :rotary]
    a, b = (r[..., 0::2], r[..., 1::2]) if interleaved else (r[..., :rotary // 2], r[..., rotary // 2:])
    p, q = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack((p, q), -1).flatten(-2) if interleaved else torch.cat((p, q), -1)
    return torch.cat((turned, x[..., rotary:]), -1)


def _normed(x, weight):
    return x if weight is None else x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight


def _append(s):
    c = s["case"]
    seq, j = _rows(s)
    at = s["past"][seq].long() + j
    angle = (c["prefix"] + at).double()[:, None] * s["inv_freq"].double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    q = _rotate(_normed(s["q"].float(), s["q_norm"]), cos, sin, c["rotary"], c["interleaved"]).to(s["q"].dtype)
    k = _rotate(_normed(s["kn"].float(), s["k_norm"]), cos, sin, c["rotary"], c["interleaved"])
    page, slot = s["tables"][seq, at // c["page"]].long(), at % c["page"]
    s["k"][page, :, slot] = k.to(s["k"].dtype)
    s["v"][page, :, slot] = s["vn"]
    return {"q": q, "k": s["k"], "v": s["v"]}


def _attend(s):
    c = s["case"]
    b, n, h, d = c["sequences"], c["new"], c["kv_heads"], c["dim"]
    g = c["heads"] // h
    seq, j = _rows(s)
    q = torch.zeros((b, n, h, g, d), device="cuda")
    q[seq, j] = s["q"].float().view(-1, h, g, d)
    q = q.permute(0, 2, 1, 3, 4).reshape(b, h, n * g, d) / math.sqrt(d)
    # own tokens, page by page, those a new token may not see masked
    most = min(_pages(c["past"] + n, c["page"]), s["tables"].shape[1])
    pages = s["tables"][:, :most].long()
    keys, values = (t[pages].float().transpose(1, 2).reshape(b, h, -1, d) for t in (s["k"], s["v"]))
    seen = s["past"].long()[:, None] + torch.arange(n, device="cuda") + 1
    hidden = torch.arange(keys.shape[2], device="cuda") >= seen.repeat_interleave(g, 1)[:, :, None]
    so = torch.matmul(q, keys.transpose(2, 3).contiguous()).masked_fill(hidden[:, None], -math.inf)
    top = so.amax(-1, keepdim=True)
    if c["prefix"]:
        at = s["prefix_table"].long()
        pk, pv = (t[at].float().transpose(0, 1).reshape(h, -1, d)[:, :c["prefix"]] for t in (s["k"], s["v"]))
        sp = torch.matmul(q.transpose(0, 1).reshape(h, -1, d), pk.transpose(1, 2).contiguous()).view(h, b, n * g, -1).transpose(0, 1)
        top = torch.maximum(top, sp.amax(-1, keepdim=True))
    eo = (so - top).exp()
    total, out = eo.sum(-1, keepdim=True), torch.matmul(eo, values)
    if c["prefix"]:
        ep = (sp - top).exp()
        total = total + ep.sum(-1, keepdim=True)
        out = out + torch.matmul(ep.transpose(0, 1).reshape(h, b * n * g, -1), pv.contiguous()).view(h, b, n * g, d).transpose(0, 1)
    out = (out / total).view(b, h, n, g, d).permute(0, 2, 1, 3, 4)[seq, j]
    return {"out": out.reshape(-1, c["heads"], d).to(s["q"].dtype)}


def _select(s):
    c = s["case"]
    x = s["logits"].double()  # 64 bits: which of two neighbours comes first is decided by their last digits
    top = x.amax(-1, keepdim=True)
    value = s["scores"].double()[..., None] + (x - (top + (x - top).exp().sum(-1, keepdim=True).log()))
    if s["finished"] is not None:  # an ended beam goes on with the padding token alone
        ended = torch.full_like(value, -math.inf)
        ended[..., 1] = s["scores"].double()
        value = torch.where(s["finished"].bool()[..., None], ended, value)
    value, at = value.view(c["groups"], -1).sort(dim=1, descending=True, stable=True)
    value, at = value[:, :c["count"]], at[:, :c["count"]]
    none = value == -math.inf
    return {"scores": value.float(), "parents": (at // c["vocab"]).to(torch.int32).masked_fill(none, -1), "tokens": (at % c["vocab"]).to(torch.int32).masked_fill(none, -1)}


def _reorder(s):
    c = s["case"]
    page, rows = c["page"], c["groups"] * c["count"]
    parent = s["parents"].long()
    source = (parent + torch.arange(c["groups"], device="cuda")[:, None] * c["beams"]).view(-1)
    earlier = torch.ones((c["count"], c["count"]), dtype=torch.bool, device="cuda").tril(-1)
    first = ~((parent[:, :, None] == parent[:, None, :]) & earlier).any(-1).view(-1)
    past = s["past"][source]
    full, rest = past.long() // page, past.long() % page
    column = torch.arange(s["tables"].shape[1], device="cuda")
    fresh = (rest == 0) | ~first  # the page of the next token: the parent's last one goes on with its first child
    table = torch.where(column < full[:, None], s["tables"][source], s["tables_out"])
    last = s["tables"][source, full]
    s["tables_out"].copy_(torch.where(column == full[:, None], torch.where(fresh, s["spare"], last)[:, None], table))
    copied = ((rest > 0) & ~first)[:, None, None, None] & (torch.arange(page, device="cuda") < rest[:, None])[:, None, :, None]
    to = s["spare"][:rows].long()
    for t in (s["k"], s["v"]):
        t[to] = torch.where(copied, t[last.long()], t[to])
    return {"past": past, "tables": s["tables_out"], "k": s["k"], "v": s["v"]}


def run(state):
    if own:
        return _run_own(state)
    return {"append": _append, "attend": _attend, "select": _select, "reorder": _reorder}[state["case"]["kind"]](state)


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    c = case
    size = 4 if c["dtype"] == "f32" else 2
    if c["kind"] == "append":
        tokens = sum(_new_tokens(c))
        values = tokens * c["dim"] * (c["heads"] + 2 * c["kv_heads"])
        return {"bytes": 2.0 * values * size, "flops": values * 8.0}
    if c["kind"] == "attend":
        counts = _new_tokens(c)
        row, rows = c["kv_heads"] * c["dim"], sum(counts) * c["heads"] * c["dim"]
        held = c["past"] + (c["sequences"] - 1) * c["past"] / 2 + sum(counts)  # lengths are spread evenly, the first one the longest
        seen = counts[0] * c["past"] + sum(counts[1:]) * c["past"] / 2 + sum(n * (n + 1) / 2 for n in counts) + sum(counts) * c["prefix"]
        return {"bytes": 2.0 * (c["prefix"] + held) * row * size + 2.0 * rows * size, "flops": 4.0 * seen * c["heads"] * c["dim"]}
    if c["kind"] == "select":
        live = c["groups"] * c["beams"] * c["vocab"] * (0.75 if c["finished"] else 1.0)
        return {"bytes": live * size + c["groups"] * (c["beams"] * 4.0 + c["count"] * 12.0), "flops": live * 4.0}
    rows, copies = c["groups"] * c["count"], c["groups"] * (c["count"] - c["parents"])
    table = 8.0 * rows * (c["past"] / 2 / c["page"] + 1)
    return {"bytes": table + 4.0 * copies * c["kv_heads"] * c["page"] / 2 * c["dim"] * size, "flops": 0.0}


# ---------------------------------------------------------------- in 64 bits, from the definitions

def _exact_append(s):
    c = s["case"]
    counts = _new_tokens(c)
    seq = torch.tensor([i for i, n in enumerate(counts) for _ in range(n)], device="cuda")
    at = torch.cat([torch.arange(n) for n in counts]).cuda() + s["past"].long()[seq]
    # a turn by the angle of each pair, as a product of complex numbers
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), (at + c["prefix"]).double().outer(s["inv_freq"].double()))[:, None]
    half = c["rotary"] // 2

    def turned(x, weight):
        x = x.double()
        if weight is not None:
            x = x / (x.square().sum(-1, keepdim=True) / c["dim"] + EPS).sqrt() * weight.double()
        lead = list(range(0, c["rotary"], 2)) if c["interleaved"] else list(range(half))
        follow = [i + 1 for i in lead] if c["interleaved"] else [i + half for i in lead]
        z = torch.complex(x[..., lead], x[..., follow]) * turn
        y = x.clone()
        y[..., lead], y[..., follow] = z.real, z.imag
        return y

    k, v = s["k"].double(), s["v"].double()
    place = s["tables"][seq, at // c["page"]].long()
    k[place, :, at % c["page"]] = turned(s["kn"], s["k_norm"])
    v[place, :, at % c["page"]] = s["vn"].double()
    return {"q": turned(s["q"], s["q_norm"]), "k": k, "v": v}


def _exact_attend(s):
    c = s["case"]
    h, d, g = c["kv_heads"], c["dim"], c["heads"] // c["kv_heads"]
    prefix = [t[s["prefix_table"].long()].double().transpose(1, 2).reshape(-1, h, d)[:c["prefix"]] for t in (s["k"], s["v"])]
    past, row, out = s["past"].tolist(), 0, []
    for i, n in enumerate(_new_tokens(c)):
        length = past[i] + n
        pages = s["tables"][i, :_pages(length, c["page"])].long()
        k, v = (torch.cat((p, t[pages].double().transpose(1, 2).reshape(-1, h, d)[:length])) for p, t in zip(prefix, (s["k"], s["v"])))
        q = s["q"][row:row + n].double().view(n, h, g, d)
        for kv in range(h):
            x = torch.matmul(q[:, kv].reshape(n * g, d), k[:, kv].t().contiguous()) / d ** 0.5
            reach = c["prefix"] + past[i] + 1 + torch.arange(n, device="cuda").repeat_interleave(g)
            x[torch.arange(len(k), device="cuda")[None] >= reach[:, None]] = -math.inf
            out.append(torch.matmul(torch.softmax(x, -1), v[:, kv].contiguous()).view(n, g, d))
        row += n
    parts, at = [], 0
    for n in _new_tokens(c):
        parts.append(torch.stack(out[at:at + h], 1).reshape(n, h * g, d))
        at += h
    return {"out": torch.cat(parts)}


def _exact_select(s):
    c = s["case"]
    value = torch.log_softmax(s["logits"].double(), -1) + s["scores"].double()[..., None]
    if s["finished"] is not None:
        gone = s["finished"].bool()
        value[gone] = -math.inf
        value[..., 1] = torch.where(gone, s["scores"].double(), value[..., 1])
    return {"scores": value.flatten(1).topk(c["count"]).values, "parents": None, "tokens": None}


def _exact_reorder(s):
    c = s["case"]
    page, k, v = c["page"], s["k"].double(), s["v"].double()
    parents, past, tables, spare = s["parents"].tolist(), s["past"].tolist(), s["tables"].tolist(), s["spare"].tolist()
    for i in range(c["groups"]):
        for j, p in enumerate(parents[i]):
            full, rest = divmod(past[i * c["beams"] + p], page)
            if rest and p in parents[i][:j]:
                a, b = tables[i * c["beams"] + p][full], spare[i * c["count"] + j]
                k[b, :, :rest], v[b, :, :rest] = k[a, :, :rest], v[a, :, :rest]
    return {"past": None, "tables": None, "k": k, "v": v}


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "select": _exact_select, "reorder": _exact_reorder}[case["kind"]](s)
