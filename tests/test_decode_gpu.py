"""The operators of a decoding step against their definitions in 64 bits (_decode_ref.py), at the sizes, lengths, tables and masks where they can go wrong, and a run of
them together as a beam search uses them."""
import math

import pytest
import torch

import _decode_ref as ref

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def randn(g, *shape, dtype=F32, scale=1.0):
    return (torch.randn(shape, generator=g) * scale).to(dtype)


def paged(g, pages, heads, size, dim, dtype):
    return randn(g, pages, heads, size, dim, dtype=dtype), randn(g, pages, heads, size, dim, dtype=dtype)


def tables_for(g, sequences, each, shared, spare=0):
    """Page numbers for `sequences` rows of `each` pages, a prefix of `shared` pages and `spare` more, in any order; the number of all."""
    total = sequences * each + shared + spare
    order = torch.randperm(total, generator=g).to(torch.int32)
    return order[:sequences * each].view(sequences, each), order[sequences * each:sequences * each + shared], order[sequences * each + shared:], total


def within(got, want, bound):
    err = (got.double().cpu() - want).abs()
    bad = ~(err <= bound)
    assert not bad.any(), "%d of %d off, worst %g over %g" % (bad.sum(), bad.numel(), (err - bound).max(), bound.flatten()[(err - bound).argmax()])


# ------------------------------------------------------------------ append

# dtype, heads, kv heads, dim, rotary, interleaved, norms, page, sequences, new, starts
APPEND = [
    (F32, 8, 2, 64, 64, False, "", 16, 4, 1, None),
    (BF16, 32, 8, 128, 128, False, "qk", 64, 9, 1, None),
    (F16, 6, 2, 128, 64, True, "qk", 24, 3, 5, None),
    (BF16, 12, 4, 96, 32, False, "k", 8, 3, 7, [0, 3, 3, 10]),       # head size no power of two; a sequence without new tokens
    (F32, 3, 3, 40, 16, True, "q", 8, 2, 3, [0, 1, 4]),
    (F16, 5, 1, 256, 256, False, "qk", 128, 2, 2, [0, 2, 3]),
    (BF16, 0, 2, 64, 0, False, "", 16, 3, 2, None),                  # keys and values alone, nothing done to them
    (F32, 2, 1, 512, 512, False, "qk", 8, 1, 3, None),
    (BF16, 1, 1, 8, 0, False, "k", 8, 70, 2, None),                  # one lane per head
    (F32, 70, 9, 64, 48, False, "qk", 16, 2, 1, None),               # more heads than one pass requests
]


@pytest.mark.parametrize("case", APPEND, ids=lambda c: "%s-%dx%dx%d-p%d-%s" % (str(c[0])[6:], c[1], c[2], c[3], c[7], c[10]))
@pytest.mark.parametrize("prefix", [0, 131071])
def test_append(cuda, case, prefix):
    from paella_amd import decode
    dtype, heads, kv_heads, dim, rotary, interleaved, norms, size, sequences, new, starts = case
    g = gen(dim + heads)
    past = [(11 * i + 5) % (3 * size) for i in range(sequences)]
    tokens = (starts[-1] if starts else sequences * new) + (2 if starts else 0)   # ragged: two rows behind the last sequence
    tables, _, _, total = tables_for(g, sequences, 4, 0)
    k, v = paged(g, total, kv_heads, size, dim, dtype)
    tables[0, past[0] // size] = total if sequences > 1 else tables[0, past[0] // size]   # a page outside the cache: not written
    qkv = randn(g, tokens, heads + 2 * kv_heads, dim, dtype=dtype)
    wq, wk = (randn(g, dim) * 0.3 + 1 if n in norms else None for n in "qk")
    freq = torch.tensor([10000.0 ** (-2 * i / rotary) for i in range(rotary // 2)]) if rotary else None
    dev = qkv.to(cuda)
    q = dev[:, :heads] if heads else None
    cache = decode.KVCache(k.to(cuda), v.to(cuda))
    batch = decode.KVBatch(torch.tensor(past, dtype=torch.int32, device=cuda), tables.to(cuda), max_new=new,
                           starts=None if starts is None else torch.tensor(starts, dtype=torch.int32, device=cuda), tokens=tokens, prefix_len=prefix,
                           prefix_table=torch.zeros(1, dtype=torch.int32, device=cuda))
    out = torch.full((tokens, heads, dim), 7.0, dtype=dtype, device=cuda) if heads else None
    res = decode.kv_append(cache, batch, dev[:, heads:heads + kv_heads], dev[:, heads + kv_heads:], q=q, q_norm=None if wq is None else wq.to(cuda),
                           k_norm=None if wk is None else wk.to(cuda), eps=1e-5, inv_freq=None if freq is None else freq.to(cuda), interleaved=interleaved, out=out)
    torch.cuda.synchronize()
    assert res is out
    want_q = torch.full((tokens, heads, dim), 7.0, dtype=torch.float64)
    want_k, want_v = k.double(), v.double()
    touched = torch.zeros(k.shape, dtype=torch.bool)
    for t, owner in enumerate(ref.owners(starts, past, new, tokens)):
        if owner is None:
            continue
        b, own = owner
        f = None if freq is None else freq.double().tolist()
        x = qkv[t].double()
        want_q[t] = ref.norm_rotate(x[:heads], None if wq is None else wq.double(), 1e-5, f, interleaved, prefix + own)
        page = int(tables[b, own // size]) if own // size < tables.shape[1] else -1
        if 0 <= page < total:
            want_k[page, :, own % size] = ref.norm_rotate(x[heads:heads + kv_heads], None if wk is None else wk.double(), 1e-5, f, interleaved, prefix + own)
            want_v[page, :, own % size] = x[heads + kv_heads:]
            touched[page, :, own % size] = True
    # one rounding to the type; in 32 bits before it: a norm's sum of dim squares over 8 values a lane and 6 exchanges, its root and two products (under 20 roundings),
    # the angle (half a step of up to half a turn, 2^-25 * 2 pi), sine and cosine (an ulp) and the turn (3): under 64 roundings of the larger of the pair, which the head's bounds
    def bound(want):
        return ref.HALF_STEP[dtype] * want.abs() + 64 * 2.0 ** -24 * want.abs().amax(-1, keepdim=True) + (2.0 ** -25 if dtype == F16 else 0)
    if heads:
        within(out, want_q, bound(want_q))
    got_k = cache.k.cpu()
    within(got_k, want_k, torch.where(touched, bound(want_k), torch.zeros(())))
    assert torch.equal(cache.v.cpu().double(), want_v)


def test_append_in_place_and_into_pages_behind_32_bits(cuda):
    """q may be its own output; a page whose offset passes 2^32 bytes is reached."""
    from paella_amd import decode
    heads, dim, size = 4, 128, 128
    pages = (1 << 32) // (heads * size * dim * 2) + 40
    cache = decode.KVCache(torch.zeros((pages, heads, size, dim), dtype=BF16, device=cuda), torch.zeros((pages, heads, size, dim), dtype=BF16, device=cuda))
    g = gen(5)
    q, k, v = (randn(g, 2, heads, dim, dtype=BF16).to(cuda) for _ in range(3))
    table = torch.tensor([[pages - 1], [pages - 3]], dtype=torch.int32, device=cuda)
    batch = decode.KVBatch(torch.tensor([17, 3], dtype=torch.int32, device=cuda), table)
    freq = torch.ones(dim // 2, device=cuda)
    want = decode.kv_append(cache, batch, k, v, q=q, inv_freq=freq)
    got = decode.kv_append(cache, batch, k, v, q=q, inv_freq=freq, out=q)
    torch.cuda.synchronize()
    assert got is q and torch.equal(got, want)
    assert torch.equal(cache.v[pages - 1, :, 17], v[0]) and torch.equal(cache.v[pages - 3, :, 3], v[1])
    assert int((cache.v[:pages - 4] != 0).any()) == 0
    attend = decode.PrefixAttention(heads, cache, batch, scale=0.0)
    out = attend(q, cache, batch)   # past 17 and 3 zero keys and values, then the token's own
    torch.cuda.synchronize()
    for b, n in ((0, 17), (1, 3)):
        page = int(table[b, 0])
        x = (q[b].double() * cache.k[page, :, n].double()).sum(-1) / math.sqrt(dim)
        p = (x.exp() / (x.exp() + n))[:, None]
        within(out[b], (p * v[b].double()).cpu(), (2.0 ** -7 * v[b].double().abs()).cpu() + 1e-6)


# ------------------------------------------------------------------ attention

# dtype, heads, kv heads, dim, page, past of each sequence, new, starts, prefix
ATTEND = [
    (F32, 8, 2, 64, 16, [40, 0, 17], 1, None, 333),
    (F32, 4, 4, 128, 8, [5, 31], 1, None, 15),
    (F32, 6, 2, 256, 24, [70], 3, None, 49),
    (F16, 16, 16, 64, 32, [100, 3, 64, 7, 0, 31, 32, 33], 1, None, 70),
    (BF16, 8, 2, 128, 64, [200, 1, 63], 5, [0, 5, 6, 9], 130),
    (BF16, 8, 2, 128, 8, [9], 1, None, 0),                        # no prefix
    (BF16, 32, 8, 128, 64, [0, 0], 1, None, 1),                   # one key of the prefix, one of its own
    (F16, 3, 1, 128, 24, [50, 24], 4, [0, 0, 4], 65),             # three heads per key head; a sequence without new tokens
    (BF16, 48, 1, 64, 16, [20, 90], 1, None, 40),                 # more heads per key head than a tile has rows
    (BF16, 4, 1, 256, 16, [33, 15, 70], 2, None, 97),
    (F16, 8, 1, 256, 128, [300], 1, None, 513),
    (F16, 2, 2, 64, 8, [0], 70, None, 9),                         # a prompt: more new tokens than a tile has rows
    (BF16, 4, 2, 128, 16, [37], 45, [0, 40], 33),
    (F32, 4, 1, 64, 8, [25, 0], 21, [0, 21, 30], 5),
    (BF16, 8, 8, 64, 64, list(range(0, 200, 5)), 1, None, 1000),  # forty rows per key head
    (F32, 16, 2, 128, 32, [130] * 9, 1, None, 260),
    (BF16, 8, 2, 128, 64, [1500, 700], 1, None, 3000),
    (BF16, 32, 2, 128, 16, [50, 3, 200, 0] * 3, 1, None, 300),    # 192 rows per key head
    (F16, 16, 1, 256, 24, [20, 70, 11], 1, None, 130),
    (F32, 8, 2, 256, 8, [9] * 6, 3, [0, 3, 4, 4, 7, 9, 12], 77),
    (BF16, 32, 2, 128, 16, [50, 3, 200, 0] * 3, 1, None, 4007),   # the same over many keys
]


def attend_case(case, cuda, holes=False, offset=0.0):
    from paella_amd import decode
    dtype, heads, kv_heads, dim, size, past, new, starts, prefix = case
    g = gen(dim + heads + prefix)
    n = len(past)
    tokens = (starts[-1] + 1) if starts else n * new     # ragged: a row behind the last sequence
    each, shared = -(-(max(past) + new) // size) + 1, -(-prefix // size)
    tables, prefix_table, _, total = tables_for(g, n, each, shared, 2)
    k, v = paged(g, total, kv_heads, size, dim, dtype)
    if offset:
        k = (k.float() + offset).to(dtype)
    q = randn(g, tokens, heads, dim, dtype=dtype, scale=1.5)
    if holes:  # pages outside the cache: one of each sequence's, one of the prefix's, one whole sequence and more
        tables[:, 0] = torch.tensor([-1, total, 1 << 30, -(1 << 31)] * n)[:n].to(torch.int32)
        tables[0] = -5
        if shared:
            prefix_table[shared // 2] = total + 3
    rows = ref.owners(starts, past, new, tokens)
    # places behind what the sequences hold: anything
    seen = torch.zeros((total, size), dtype=torch.bool)
    for table, count in [(prefix_table, prefix)] + [(tables[b], max([o[1] + 1 for o in rows if o is not None and o[0] == b], default=0)) for b in range(n)]:
        for i in range(count):
            if 0 <= table[i // size] < total:
                seen[table[i // size], i % size] = True
    bad = torch.tensor([math.nan, math.inf, -math.inf, 1e4]).repeat(total * size // 4 + 1)[:total * size].view(total, size)
    k, v = (torch.where(seen[:, None, :, None], x, bad[:, None, :, None].to(dtype)) for x in (k, v))
    cache = decode.KVCache(k.to(cuda), v.to(cuda))
    batch = decode.KVBatch(torch.tensor(past, dtype=torch.int32, device=cuda), tables.to(cuda), max_new=new, tokens=tokens,
                           starts=None if starts is None else torch.tensor(starts, dtype=torch.int32, device=cuda), prefix_table=prefix_table.to(cuda), prefix_len=prefix)
    return q, k, v, rows, tables, prefix_table, cache, batch


@pytest.mark.parametrize("holes", [False, True], ids=["", "holes"])
@pytest.mark.parametrize("case", ATTEND, ids=lambda c: "%s-%dx%dx%d-p%d-%d+%d" % (str(c[0])[6:], c[1], c[2], c[3], c[4], c[8], max(c[5])))
def test_attention(cuda, case, holes):
    from paella_amd import decode
    dtype, heads, kv_heads, dim, size, past, new, starts, prefix = case
    q, k, v, rows, tables, prefix_table, cache, batch = attend_case(case, cuda, holes)
    attend = decode.PrefixAttention(heads, cache, batch)
    out = torch.full(q.shape, 7.0, dtype=dtype, device=cuda)
    for _ in range(2):  # the counters are left at zero by every launch
        attend(q.to(cuda), cache, batch, out=out)
    torch.cuda.synchronize()
    want, weight, products = ref.attention(q, k, v, rows, tables, prefix_table, prefix, 1 / math.sqrt(dim))
    bound = ref.attention_bound(want, weight, products, dtype, prefix + max(past) + new)
    for t, owner in enumerate(rows):
        if owner is None:
            want[t] = 7.0    # left as it was
            bound[t] = 0.0
    within(out, want, bound)


@pytest.mark.parametrize("form", [(16, 16), (64, 16), (128, 16), (64, 64), (128, 128)], ids=str)
@pytest.mark.parametrize("case", [0, 1, 2, 4, 7, 8, 9, 12, 14, 15, 17, 18])
def test_attention_in_every_form(cuda, case, form):
    """A plan's rows per workgroup are a choice of speed: any form that there is gives the same."""
    from paella_amd import decode
    dtype, heads, kv_heads, dim, size, past, new, starts, prefix = ATTEND[case]
    q, k, v, rows, tables, prefix_table, cache, batch = attend_case(ATTEND[case], cuda, True)
    attend = decode.PrefixAttention(heads, cache, batch)
    attend.plan.prefix_rows, attend.plan.own_rows = form
    if form[0] == 128 and dim * (4 if dtype == F32 else 2) > 256:
        with pytest.raises(RuntimeError):   # no such kernel
            attend(q.to(cuda), cache, batch)
        return
    out = torch.full(q.shape, 7.0, dtype=dtype, device=cuda)
    for _ in range(2):
        attend(q.to(cuda), cache, batch, out=out)
    torch.cuda.synchronize()
    want, weight, products = ref.attention(q, k, v, rows, tables, prefix_table, prefix, 1 / math.sqrt(dim))
    bound = ref.attention_bound(want, weight, products, dtype, prefix + max(past) + new)
    for t, owner in enumerate(rows):
        if owner is None:
            want[t] = 7.0    # left as it was
            bound[t] = 0.0
    within(out, want, bound)


LONG_WALKS = [
    (BF16, 32, 2, 64, 8, [700, 3, 0, 1300], 4, None, 2603),       # 128 rows and one workgroup's each, a page per block of 8 keys
    (F16, 16, 2, 128, 24, [1100, 40], 9, [0, 9, 15], 1537),
    (F32, 16, 2, 128, 8, [590, 8], 5, None, 1100),
    (BF16, 16, 1, 256, 16, [530, 1029], 4, None, 1041),
]


@pytest.mark.parametrize("holes", [False, True], ids=["", "holes"])
@pytest.mark.parametrize("splits", [(1, 1), (2, 3)], ids=str)
@pytest.mark.parametrize("case", LONG_WALKS, ids=lambda c: "%s-%dx%dx%d-p%d-%d+%d" % (str(c[0])[6:], c[1], c[2], c[3], c[4], c[8], max(c[5])))
def test_attention_of_many_rows_over_many_pages_by_one_workgroup(cuda, case, splits, holes):
    """Walks of many rows over more pages than a workgroup looks up at once, which short inputs get only where the keys are hardly split."""
    from paella_amd import decode
    dtype, heads, kv_heads, dim, size, past, new, starts, prefix = case
    q, k, v, rows, tables, prefix_table, cache, batch = attend_case(case, cuda, holes)
    attend = decode.PrefixAttention(heads, cache, batch)
    assert min(attend.plan.prefix_rows, attend.plan.own_rows) > 16 and attend.plan.prefix_splits >= splits[0] and attend.plan.own_splits >= splits[1]
    attend.plan.prefix_splits, attend.plan.own_splits = splits
    out = torch.full(q.shape, 7.0, dtype=dtype, device=cuda)
    for _ in range(2):
        attend(q.to(cuda), cache, batch, out=out)
    torch.cuda.synchronize()
    want, weight, products = ref.attention(q, k, v, rows, tables, prefix_table, prefix, 1 / math.sqrt(dim))
    bound = ref.attention_bound(want, weight, products, dtype, prefix + max(past) + new)
    for t, owner in enumerate(rows):
        if owner is None:
            want[t] = 7.0    # left as it was
            bound[t] = 0.0
    within(out, want, bound)


def test_attention_of_large_scores_and_a_strided_query(cuda):
    """Scores of hundreds, all of one sign: the running maximum has to carry them.  q is a view of a packed projection; a scale of its own."""
    from paella_amd import decode
    case = (BF16, 8, 2, 128, 16, [61, 5], 1, None, 100)
    q, k, v, rows, tables, prefix_table, cache, batch = attend_case(case, cuda, offset=3.0)
    q = (q.float() * 0.3 + 1.0).to(BF16)
    packed = torch.zeros((2, 12, 128), dtype=BF16, device=cuda)
    packed[:, :8] = q.to(cuda)
    out = decode.PrefixAttention(8, cache, batch, scale=0.7)(packed[:, :8], cache, batch)
    torch.cuda.synchronize()
    want, weight, products = ref.attention(q, k, v, rows, tables, prefix_table, 100, 0.7)
    within(out, want, ref.attention_bound(want, weight, products, BF16, 170))


@pytest.mark.parametrize("case", [0, 4, 14, 17, 19])
def test_attention_passes_nan_and_infinity_on(cuda, case):
    """What a row sees of them reaches that row and no other: a query, keys of one sequence, values of another."""
    from paella_amd import decode
    case = ATTEND[case]
    q, k, v, rows, tables, prefix_table, cache, batch = attend_case(case, cuda)
    attend = decode.PrefixAttention(case[1], cache, batch)
    want = attend(q.to(cuda), cache, batch)
    sequences, size = len(case[5]), case[4]
    bad = torch.zeros(q.shape[:2], dtype=torch.bool)
    q = q.clone()
    q[0, 1] = math.nan
    bad[0, 1] = True
    last = [t for t, o in enumerate(rows) if o is not None and o[0] == sequences - 1]
    own = rows[last[0]][1]      # the first new token of the last sequence: all of its rows see it
    cache.k[int(tables[-1, own // size]), 0, own % size] = math.inf if case[0] != F32 else math.nan
    bad[last[0]:last[-1] + 1, :case[1] // case[2]] = True   # the heads of key head 0; scores of infinities of both signs, or NaN
    got = attend(q.to(cuda), cache, batch)
    torch.cuda.synchronize()
    owned = torch.tensor([o is not None for o in rows])
    bad &= owned[:, None]
    gone = torch.isnan(got.cpu()).any(-1)
    assert torch.equal(gone[owned], bad[owned])
    assert torch.equal(got.cpu()[owned][~bad[owned]], want.cpu()[owned][~bad[owned]])


@pytest.mark.parametrize("case,stages", [(0, 1), (3, 1), (16, 2), (20, 2)])
def test_attention_is_the_same_every_time_in_graphs_on_streams_and_direct_queues(cuda, case, stages):
    """Which workgroup joins a row changes from run to run, the bits do not: eager, replayed (two graphs of one plan side by side, lengths changed between replays), on another
    stream and on a direct-dispatch queue."""
    from paella_amd import decode, ops
    case = ATTEND[case]
    q, k, v, rows, tables, prefix_table, cache, batch = attend_case(case, cuda)
    q = q.to(cuda)
    attend = decode.PrefixAttention(case[1], cache, batch)
    assert attend.plan.workspace_bytes and attend.plan.stages == stages
    want = attend(q, cache, batch)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = attend(q, cache, batch)
    torch.cuda.synchronize()
    assert torch.equal(other, want)
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(attend(q, cache, batch))
        graphs.append(graph)
    shorter = (batch.past - 100).clamp(min=0)
    longer = batch.past.clone()
    for past in (longer, shorter, longer):
        batch.past.copy_(past)
        now = attend(q, cache, batch)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], now) and torch.equal(outs[1], now)
    assert torch.equal(now, want)
    with ops.DirectQueue() as queue:
        for _ in range(2):
            out = torch.zeros_like(want)
            for stage in range(attend.plan.stages):
                attend(q, cache, batch, out=out, stream=queue.handle, stage=stage)
                queue.wait()
            assert torch.equal(out, want)
        if attend.plan.stages > 1:
            with pytest.raises(RuntimeError, match="-2"):
                attend(q, cache, batch, out=out, stream=queue.handle)
    with ops.DirectQueue(ordered=True) as queue:
        out = torch.zeros_like(want)
        attend(q, cache, batch, out=out, stream=queue.handle)
        queue.wait()
        assert torch.equal(out, want)


# ------------------------------------------------------------------ beam search

# dtype, groups, beams, vocab, count
SELECT = [(F32, 1, 4, 32000, 4), (BF16, 3, 4, 40001, 8), (F16, 2, 16, 5003, 32), (F32, 5, 1, 1, 1), (F32, 2, 3, 7, 9), (BF16, 2, 2, 513, 64), (F32, 200, 3, 9001, 3),
          (F16, 1, 32, 300, 64), (F32, 1, 1, 140000, 5), (BF16, 90, 8, 2049, 16)]


def check_selection(got, logits, scores, finished, pad, count):
    want = ref.select(logits.cpu(), scores.cpu(), None if finished is None else finished.cpu(), pad, count)
    values, parents, tokens = (t.cpu() for t in got)
    for g, rows in enumerate(want):
        assert [(int(p), int(t)) for p, t in zip(parents[g], tokens[g])] == [r[1:] for r in rows], g
        for c, r in enumerate(rows):
            # the sum of exponentials in 32 bits: under 64 roundings each of its terms (whose arguments are rounded, up to 64 in magnitude) and of the sum; then one rounding
            assert float(values[g, c]) == r[0] or abs(float(values[g, c]) - r[0]) <= 2.0 ** -24 * (128 + abs(r[0])), (g, c)


@pytest.mark.parametrize("ended", [False, True], ids=["", "ended"])
@pytest.mark.parametrize("case", SELECT, ids=lambda c: "%s-%dx%dx%d-%d" % ((str(c[0])[6:],) + c[1:]))
def test_select(cuda, case, ended):
    from paella_amd import decode
    dtype, groups, beams, vocab, count = case
    g = gen(vocab)
    logits = randn(g, groups, beams, vocab, dtype=dtype, scale=3.0).to(cuda)
    scores = randn(g, groups, beams).to(cuda)
    finished = (torch.rand((groups, beams), generator=g) < 0.4).to(cuda) if ended else None
    pick = decode.BeamSelect(groups, beams, vocab, count, dtype)
    for _ in range(2):
        got = pick(logits, scores, finished=finished, pad_token=vocab - 1)
    torch.cuda.synchronize()
    check_selection(got, logits, scores, finished, vocab - 1, count)


def test_select_of_equals_infinities_and_nan(cuda):
    """Equal logits go by index, within a thread's, a wave's and a beam's and, with equal scores, between beams; masked ones (-inf, the type's lowest) never come first; NaN
    counts as masked; a beam without any continuation, or with +inf, has none."""
    from paella_amd import decode
    g = gen(3)
    for dtype in (F32, BF16, F16):
        for vocab in (9, 3000, 20001):
            x = torch.zeros((8, 4, vocab))                             # all equal
            x[1] = torch.randint(0, 3, (4, vocab), generator=g).float()   # few values
            x[2] = -math.inf
            x[2, 1, vocab // 2:vocab // 2 + 3] = 1.0                   # three continuations in all
            x[3] = torch.finfo(dtype).min
            x[3, 2, 5] = 0.0
            x[4] = torch.arange(vocab).float() / vocab                 # the best side by side, in few lanes
            x[5] = -0.0
            x[5, :, 1::2] = 0.0
            x[6, 0] = math.nan
            x[6, 1, ::2] = math.nan
            x[6, 2, 3] = math.inf
            x[7] = torch.randn((4, vocab), generator=g)
            logits = x.to(dtype).to(cuda)
            scores = torch.zeros((8, 4))
            scores[7] = torch.tensor([-math.inf, 0.5, math.nan, -2.0])
            scores = scores.to(cuda)
            for count in (1, 4, 40):
                got = decode.BeamSelect(8, 4, vocab, count, dtype)(logits, scores)
                torch.cuda.synchronize()
                check_selection(got, logits, scores, None, 0, count)


def test_select_reads_rows_of_any_stride_in_graphs_and_direct_queues(cuda):
    from paella_amd import decode, ops
    g = gen(8)
    wide = randn(g, 2, 3, 5001, dtype=F16).to(cuda)
    logits, scores = wide[:, :, 1:4100], randn(g, 2, 3).to(cuda)
    pick = decode.BeamSelect(2, 3, 4099, 6, F16)
    want = pick(logits, scores)
    torch.cuda.synchronize()
    check_selection(want, logits, scores, None, 0, 6)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = pick(logits, scores)
    for _ in range(3):
        graph.replay()
        again = pick(logits, scores)
        torch.cuda.synchronize()
        for a, b, c in zip(got, want, again):
            assert torch.equal(a, b) and torch.equal(c, b)
        for t in got:
            t.zero_()
    with ops.DirectQueue() as queue:
        got = pick(logits, scores, stream=queue.handle)
        queue.wait()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


# dtype, kv heads, dim, page, groups, beams, count, past
REORDER = [(F32, 2, 64, 16, 1, 4, 4, [90]), (BF16, 8, 128, 64, 3, 8, 8, [100, 64, 7]), (F16, 1, 40, 8, 2, 3, 7, [0, 15]), (BF16, 3, 64, 24, 2, 70, 70, [47, 48]),
           (F32, 1, 8, 8, 4, 2, 1, [1, 8, 9, 23])]


@pytest.mark.parametrize("case", REORDER, ids=lambda c: "%s-%dx%d-p%d-%dx%d" % ((str(c[0])[6:],) + c[1:6]))
def test_reorder(cuda, case):
    from paella_amd import decode
    dtype, heads, dim, size, groups, beams, count, past = case
    g = gen(dim)
    each = max(past) // size + 2
    tables, _, spare, total = tables_for(g, groups * beams, each, 0, groups * count)
    k, v = paged(g, total, heads, size, dim, dtype)
    parents = torch.randint(0, beams, (groups, count), generator=g, dtype=torch.int32)
    parents[0, count - 1] = -1            # a child of nobody
    past_of = torch.tensor([p for p in past for _ in range(beams)], dtype=torch.int32)
    tables_out = torch.full((groups * count, each), -9, dtype=torch.int32)
    want_k, want_v, want_tables = k.clone(), v.clone(), tables_out.clone()
    want_past = ref.reorder(want_k, want_v, parents, past_of, tables, spare, want_tables)
    cache = decode.KVCache(k.to(cuda), v.to(cuda))
    dev = tables_out.to(cuda)
    got = decode.beam_reorder(cache, parents.to(cuda), past_of.to(cuda), tables.to(cuda), dev, spare.to(cuda))
    torch.cuda.synchronize()
    assert got.tolist() == want_past and torch.equal(dev.cpu(), want_tables)
    assert torch.equal(cache.k.cpu(), want_k) and torch.equal(cache.v.cpu(), want_v)


def test_reorder_with_numbers_outside_the_cache_and_the_table(cuda):
    from paella_amd import decode
    g = gen(1)
    k, v = paged(g, 4, 1, 8, 16, F32)
    tables = torch.tensor([[0, 9], [1, 2]], dtype=torch.int32)
    spare = torch.tensor([3, -1, 3, 40], dtype=torch.int32)
    for past in ([12, 12], [16, 200], [-3, 16]):
        for parents in ([[0, 0, 1, 1]], [[1, 1, 2, -7]]):
            parents = torch.tensor(parents, dtype=torch.int32)
            out = torch.full((4, 2), -9, dtype=torch.int32)
            want_k, want_v, want_out = k.clone(), v.clone(), out.clone()
            clipped = torch.tensor(past, dtype=torch.int32)
            want = ref.reorder(want_k, want_v, parents, clipped, tables, spare, want_out)
            cache, dev = decode.KVCache(k.to(cuda), v.to(cuda)), out.to(cuda)
            got = decode.beam_reorder(cache, parents.to(cuda), clipped.to(cuda), tables.to(cuda), dev, spare.to(cuda))
            torch.cuda.synchronize()
            assert got.tolist() == want and torch.equal(dev.cpu(), want_out)
            assert torch.equal(cache.k.cpu(), want_k) and torch.equal(cache.v.cpu(), want_v)


# ------------------------------------------------------------------ together

def test_a_beam_search_over_a_shared_prompt(cuda):
    """Eight steps of two requests' beams over one prompt: append, attend, logits, select, reorder; the prompt's own keys go into the prefix's pages by the same operator.  Against
    the same model without a cache, each hypothesis's tokens run through attention in 64 bits from the start."""
    from paella_amd import decode
    g = gen(21)
    groups, beams, heads, kv_heads, dim, size, vocab, prompt, steps = 2, 3, 4, 2, 64, 8, 97, 21, 10
    freq = torch.tensor([100.0 ** (-2 * i / dim) for i in range(dim // 2)])
    embed, wq, wk, wv = randn(g, vocab, 48), randn(g, 48, heads * dim, scale=0.2), randn(g, 48, kv_heads * dim, scale=0.2), randn(g, 48, kv_heads * dim, scale=0.2)
    wo, nq, nk = randn(g, heads * dim, vocab, scale=0.5), randn(g, dim) * 0.1 + 1, randn(g, dim) * 0.1 + 1
    words = torch.randint(0, vocab, (prompt,), generator=g)
    d_embed, d_wq, d_wk, d_wv, d_wo, d_nq, d_nk, d_freq = (t.to(cuda) for t in (embed, wq, wk, wv, wo, nq, nk, freq))

    def project(tokens):
        x = d_embed[tokens.long()]
        return (x @ d_wq).view(-1, heads, dim), (x @ d_wk).view(-1, kv_heads, dim), (x @ d_wv).view(-1, kv_heads, dim)

    rows, each = groups * beams, -(-steps // size) + 1
    shared = -(-prompt // size)
    pages = shared + rows * (steps + 2)
    cache = decode.KVCache.empty(pages, kv_heads, size, dim)
    prefix_table = torch.arange(shared, dtype=torch.int32, device=cuda)
    q, k, v = project(words.to(cuda))
    whole = decode.KVBatch(torch.zeros(1, dtype=torch.int32, device=cuda), prefix_table.view(1, -1), max_new=prompt)
    q = decode.kv_append(cache, whole, k, v, q=q, q_norm=d_nq, k_norm=d_nk, inv_freq=d_freq)
    last = decode.PrefixAttention(heads, cache, whole)(q, cache, whole)[-1:]
    first = torch.log_softmax((last.reshape(1, -1) @ d_wo).double(), -1)[0].topk(rows).indices.to(torch.int32)
    tokens, scores = first.clone(), torch.zeros((groups, beams), device=cuda)
    tables = torch.full((rows, each), -1, dtype=torch.int32, device=cuda)
    free = shared + rows
    tables[:, 0] = torch.arange(shared, shared + rows, dtype=torch.int32, device=cuda)
    past = torch.zeros(rows, dtype=torch.int32, device=cuda)
    pick = decode.BeamSelect(groups, beams, vocab, beams)
    history = [[int(t)] for t in first]

    def reference(said):
        """log-probabilities of the word after the prompt and `said`, in 64 bits."""
        text = torch.cat((words, torch.tensor(said)))
        x = embed[text].double()
        qs, ks, vs = (x[-1:] @ wq.double()).view(1, heads, dim), (x @ wk.double()).view(-1, kv_heads, dim), (x @ wv.double()).view(-1, kv_heads, dim)
        qs = ref.norm_rotate(qs[0], nq.double(), 1e-6, freq.double().tolist(), False, len(text) - 1)
        ks = torch.stack([ref.norm_rotate(ks[i], nk.double(), 1e-6, freq.double().tolist(), False, i) for i in range(len(text))])
        o = []
        for h in range(heads):
            p = torch.softmax(ks[:, h // 2] @ qs[h] / math.sqrt(dim), 0)
            o.append(p @ vs[:, h // 2])
        return torch.log_softmax(torch.cat(o) @ wo.double(), 0)

    for step in range(steps):
        batch = decode.KVBatch(past, tables, prefix_table=prefix_table, prefix_len=prompt)
        q, k, v = project(tokens)
        q = decode.kv_append(cache, batch, k, v, q=q, q_norm=d_nq, k_norm=d_nk, inv_freq=d_freq)
        out = decode.PrefixAttention(heads, cache, batch)(q, cache, batch)
        logits = (out.reshape(rows, -1) @ d_wo).view(groups, beams, vocab)
        new_scores, parents, chosen = pick(logits, scores)
        # every row's log-probabilities, and the choice made from them
        for r in range(rows):
            want = reference(history[r])
            got = torch.log_softmax(logits.view(rows, -1)[r].double().cpu(), 0)
            assert (got - want).abs().max() < 1e-4, (step, r)
        check_selection((new_scores, parents, chosen), logits, scores, None, 0, beams)
        spare = torch.arange(free, free + rows, dtype=torch.int32, device=cuda)
        free += rows
        lengths = past + 1
        tables_out = torch.full_like(tables, -1)
        past = decode.beam_reorder(cache, parents, lengths, tables, tables_out, spare)
        tables, scores, tokens = tables_out, new_scores, chosen.reshape(-1)
        history = [history[r // beams * beams + int(parents.view(-1)[r])] + [int(tokens[r])] for r in range(rows)]
    assert past.tolist() == [steps] * rows


def test_a_step_reports_to_its_notifier(cuda):
    """Every operator's launch sends end messages that add up to the grid that its dims announce."""
    import ctypes
    import numpy as np
    from paella_amd import _abi, decode
    from paella_amd._abi_decode import BeamReorderDesc, KvAppendDesc
    lib = _abi.ops()
    ring = ctypes.c_void_p()
    _abi.check(lib.paella_ring_create(4096, 1, ctypes.byref(ring)), "paella_ring_create")
    try:
        note = lib.paella_ring_notifier(ring, 0)
        case = ATTEND[4]
        q, k, v, rows, tables, prefix_table, cache, batch = attend_case(case, cuda)
        q, new = q.to(cuda), torch.zeros((q.shape[0], 2, 128), dtype=BF16, device=cuda)
        attend, pick = decode.PrefixAttention(8, cache, batch), decode.BeamSelect(2, 3, 5000, 4)
        logits, scores = torch.zeros((2, 3, 5000), device=cuda), torch.zeros((2, 3), device=cuda)
        parents, past = torch.zeros((2, 4), dtype=torch.int32, device=cuda), torch.ones(6, dtype=torch.int32, device=cuda)
        old, out, spare = (torch.zeros(s, dtype=torch.int32, device=cuda) for s in ((6, 2), (8, 2), (8,)))
        append_dims, reorder_dims = _abi.LaunchDims(), _abi.LaunchDims()
        assert lib.paella_kv_append_dims(ctypes.byref(KvAppendDesc(8, 0, 0, 1e-6, 1024, 256, 256)), cache.ref, batch.ref, ctypes.byref(append_dims)) == 0
        assert lib.paella_beam_reorder_dims(ctypes.byref(BeamReorderDesc(2, 3, 4, 2)), cache.ref, ctypes.byref(reorder_dims)) == 0
        calls = [(append_dims, lambda i: decode.kv_append(cache, batch, new, new, q=q, job_id=i, notifier=note)),
                 (attend.dims(attend.plan.stages - 1), lambda i: attend(q, cache, batch, job_id=i, notifier=note)),
                 (pick.dims(), lambda i: pick(logits, scores, job_id=i, notifier=note)),
                 (reorder_dims, lambda i: decode.beam_reorder(cache, parents, past, old, out, spare, job_id=i, notifier=note))]
        for i, (dims, call) in enumerate(calls):
            assert dims.block == 256 and 0 < dims.vgprs <= 512 and dims.lds_bytes <= 160 * 1024
            call(11 + i)
            torch.cuda.synchronize()
            messages = 2 * -(-dims.grid // lib.paella_ring_batch_size())
            bits = np.zeros(messages, np.uint64)
            assert lib.paella_ring_drain(ring, bits.ctypes.data, messages, 20.0) == messages and not lib.paella_ring_can_read(ring)
            num, start, job = (bits >> np.uint64(16)) & np.uint64(0xFF), bits & np.uint64(0xFF), bits >> np.uint64(32)
            assert int(num[start == 0].sum()) == dims.grid == int(num[start == 1].sum()) and set(job.tolist()) == {11 + i}
    finally:
        lib.paella_ring_destroy(ring)


def test_the_front_end_refuses_what_does_not_fit(cuda):
    """Nothing of these calls is launched: the cache stays as it was."""
    from paella_amd import decode
    cache = decode.KVCache.empty(6, 2, 8, 64, BF16)
    ints = lambda *shape: torch.zeros(shape, dtype=torch.int32, device=cuda)  # noqa: E731
    past, tables = ints(3), ints(3, 2)
    batch = decode.KVBatch(past, tables, prefix_table=ints(2), prefix_len=16)
    k = torch.ones((3, 2, 64), dtype=BF16, device=cuda)
    q = torch.ones((3, 4, 64), dtype=BF16, device=cuda)
    attend, pick = decode.PrefixAttention(4, cache, batch), decode.BeamSelect(2, 3, 100, 4)
    logits, scores = torch.zeros((2, 3, 100), device=cuda), torch.zeros((2, 3), device=cuda)
    parents, out, spare = ints(1, 3), ints(3, 2), ints(3)
    wide = torch.ones((3, 4, 128), dtype=BF16, device=cuda)
    calls = [lambda: decode.KVCache(k, k), lambda: decode.KVCache(cache.k, cache.v.float()), lambda: decode.KVCache(cache.k, cache.v[:5]),
             lambda: decode.KVBatch(past.long(), tables), lambda: decode.KVBatch(past, tables[:2]), lambda: decode.KVBatch(past, tables.t()), lambda: decode.KVBatch(past.cpu(), tables),
             lambda: decode.KVBatch(past, tables, tokens=4), lambda: decode.KVBatch(past, tables, starts=ints(4)), lambda: decode.KVBatch(past, tables, starts=ints(3), tokens=3),
             lambda: decode.KVBatch(past, tables, prefix_len=3), lambda: decode.KVBatch(past, tables, max_new=0),
             lambda: decode.kv_append(cache, batch, k[:2], k[:2]), lambda: decode.kv_append(cache, batch, k.float(), k), lambda: decode.kv_append(cache, batch, k, k.cpu()),
             lambda: decode.kv_append(cache, batch, k.transpose(0, 1).contiguous().transpose(0, 1), k), lambda: decode.kv_append(cache, batch, k, k, q=wide),
             lambda: decode.kv_append(cache, batch, k, k, q=wide[:, :, ::2]), lambda: decode.kv_append(cache, batch, k, k, k_norm=torch.ones(32, device=cuda)),
             lambda: decode.kv_append(cache, batch, k, k, k_norm=torch.ones(64, device=cuda, dtype=BF16)), lambda: decode.kv_append(cache, batch, k, k, inv_freq=torch.ones(7, device=cuda)),
             lambda: decode.kv_append(cache, batch, k, k, q=q, out=q[:2]), lambda: decode.kv_append(cache, batch, k, k, inv_freq=torch.ones(40, device=cuda)),
             lambda: attend(q[:2], cache, batch), lambda: attend(q.float(), cache, batch), lambda: attend(q, cache, batch, out=q), lambda: attend(k, cache, batch),
             lambda: attend(q, decode.KVCache.empty(6, 2, 16, 64, BF16), batch), lambda: attend(q, cache, decode.KVBatch(past, tables, prefix_table=ints(1), prefix_len=16)),
             lambda: attend(q, cache, decode.KVBatch(past, tables)), lambda: attend(q, cache, batch, stage=2), lambda: decode.PrefixAttention(3, cache, batch),
             lambda: decode.PrefixAttention(4, cache, batch, scale=-1.0), lambda: decode.PrefixAttention(4, decode.KVCache.empty(6, 2, 8, 96, BF16), batch),
             lambda: decode.BeamSelect(1, 33, 10, 1), lambda: decode.BeamSelect(1, 3, 10, 65), lambda: decode.BeamSelect(1, 3, 10, 2, torch.float64),
             lambda: pick(logits[:, :, :99], scores), lambda: pick(logits.half(), scores), lambda: pick(logits, scores[:, :2]), lambda: pick(logits, scores.double()),
             lambda: pick(logits.transpose(0, 1).contiguous().transpose(0, 1), scores), lambda: pick(logits, scores, finished=scores), lambda: pick(logits, scores, finished=scores.bool(), pad_token=100),
             lambda: decode.beam_reorder(cache, parents, past, tables, tables, spare), lambda: decode.beam_reorder(cache, parents, past, tables, out, spare[:2]),
             lambda: decode.beam_reorder(cache, parents, past, tables, out, spare, past_out=past), lambda: decode.beam_reorder(cache, parents.long(), past, tables, out, spare),
             lambda: decode.beam_reorder(cache, ints(2, 3), past, tables, out, spare)]
    for i, call in enumerate(calls):
        with pytest.raises((AssertionError, RuntimeError)):
            call()
            pytest.fail("call %d was taken" % i)
    torch.cuda.synchronize()
    assert not cache.k.any() and not cache.v.any() and not out.any()
