"""The operators over long caches against their definitions in 64 bits (_long_ref.py), at the sizes, lengths, tables and masks where they can go wrong, and a run of them together."""
import math

import pytest
import torch

import _decode_ref as ref
import _long_ref as long_ref
from test_decode_gpu import BF16, F16, F32, gen, randn, tables_for, within

pytestmark = pytest.mark.gpu


class Case:
    """A cache whose places behind the tokens hold NaN, a batch, and what the host knows of both."""

    def __init__(self, seed, dtype, kv_heads, dim, page, past, new=1, starts=None, prefix=0, bad=(), each=None, behind=0):
        g = gen(seed)
        n = len(past)
        most = [max(p, 0) + (new if starts is None else starts[b + 1] - starts[b]) for b, p in enumerate(past)]
        each = each or max(1, -(-max(most) // page))
        shared = -(-prefix // page)
        self.tables, self.prefix_table, _, total = tables_for(g, n, each, shared, 2)
        self.k, self.v = (randn(g, total, kv_heads, page, dim, dtype=dtype) for _ in range(2))
        held = torch.zeros((total, page), dtype=torch.bool)
        for b in range(n):
            for i in range(min(most[b], each * page)):
                held[self.tables[b, i // page], i % page] = True
        for i in range(prefix):
            held[self.prefix_table[i // page], i % page] = True
        for t in (self.k, self.v):
            t.masked_fill_(~held[:, None, :, None], math.nan)
        for where, value in bad:   # (sequence or -1 for the prefix, page along it): a number outside the cache
            (self.prefix_table if where[0] < 0 else self.tables[where[0]])[where[1]] = value if value < 0 else total + value
        self.tokens = (starts[-1] if starts else n * new) + behind
        self.past, self.new, self.starts, self.prefix, self.page, self.dtype, self.total = past, new, starts, prefix, page, dtype, total
        self.kv_heads, self.dim, self.gen = kv_heads, dim, g
        self.host = long_ref.Sequences(starts, past, new, self.tokens, self.tables, self.prefix_table, prefix, page, total)

    def to(self, cuda):
        from paella_amd import decode
        self.cache = decode.KVCache(self.k.to(cuda), self.v.to(cuda))
        self.batch = decode.KVBatch(torch.tensor(self.past, dtype=torch.int32, device=cuda), self.tables.to(cuda), max_new=self.new,
                                    starts=None if self.starts is None else torch.tensor(self.starts, dtype=torch.int32, device=cuda), tokens=self.tokens,
                                    prefix_table=self.prefix_table.to(cuda), prefix_len=self.prefix)
        return self.cache, self.batch

    def queries(self, heads, scale=1.5):
        return randn(self.gen, self.tokens, heads, self.dim, dtype=self.dtype, scale=scale)


def same(got, want):
    """Equal, NaN in the same places."""
    got, want = got.cpu(), want.cpu()
    ok = (got == want) | (got.isnan() & want.isnan()) if got.is_floating_point() else got == want
    assert ok.all(), "%d of %d differ, first at %s" % ((~ok).sum(), ok.numel(), (~ok).nonzero()[0].tolist())


# ------------------------------------------------------------------ bounds

BOUNDS = [
    (F32, 2, 64, 16, [0, 5, 15, 16, 31], 1, None),
    (BF16, 8, 128, 64, [0, 63, 64, 1000], 1, None),
    (F16, 3, 256, 24, [7, 0, 48], 5, None),
    (BF16, 1, 40, 8, [3, 0, 9], 30, [0, 30, 30, 47]),          # a head of no power of two, a sequence without new tokens
    (F32, 2, 512, 8, [1, 6], 9, None),                         # a row of more pieces than a wave has lanes
    (F16, 2, 8, 8, [0, 70], 3, None),                          # one lane a key
    (F32, 1, 96, 128, [100, 0], 300, [0, 1, 301]),
    (F16, 7, 64, 8, [0, 50, 7], 20, None),                     # four heads a wave, and a group of three
    (BF16, 5, 64, 16, [3, 0, 9], 30, [0, 30, 30, 47]),         # two, and one that is left over
    (F32, 1, 32, 8, [5, 20], 3, None),                         # no other head
]


@pytest.mark.parametrize("case", BOUNDS, ids=lambda c: "%s-%dx%d-p%d-%d" % (str(c[0])[6:], c[1], c[2], c[3], c[5]))
def test_bounds(cuda, case):
    from paella_amd import long_cache
    dtype, heads, dim, page, past, new, starts = case
    c = Case(dim + page, dtype, heads, dim, page, past, new, starts, behind=2 if starts else 0)
    cache, batch = c.to(cuda)
    old = randn(c.gen, c.total, heads, 2, dim, dtype=dtype)
    bounds = old.to(cuda)
    assert long_cache.page_bounds(cache, bounds, batch) is bounds
    same(bounds, long_ref.bounds(c.host, c.k, old))
    long_cache.page_bounds(cache, bounds, batch)   # what was there does not matter
    same(bounds, long_ref.bounds(c.host, c.k, old))


def test_bounds_of_bad_pages_of_long_tables_and_of_odd_numbers(cuda):
    from paella_amd import long_cache
    c = Case(3, BF16, 2, 64, 16, [20, 50, 7, 30], 4, bad=[((0, 1), -5), ((2, 0), 3)], each=3)   # sequence 1 goes past its table, pages of two others lie outside the cache
    c.k[c.tables[3, 1], 0, 0] = math.nan
    c.k[c.tables[3, 1], 0, 1, :5] = torch.tensor([math.inf, -math.inf, 0.0, -0.0, 1e38])
    cache, batch = c.to(cuda)
    old = randn(c.gen, c.total, 2, 2, 64, dtype=BF16)
    bounds = old.to(cuda)
    long_cache.page_bounds(cache, bounds, batch)
    same(bounds, long_ref.bounds(c.host, c.k, old))
    batch.past.copy_(torch.tensor([-9, 1 << 30, 2 ** 31 - 1, 0], dtype=torch.int32))   # lengths are read at the launch
    c.host.past = [0, 1 << 30, 2 ** 31 - 1, 0]
    c.host.rows = ref.owners(None, c.host.past, 4, 16)
    again = old.to(cuda)
    long_cache.page_bounds(cache, again, batch)
    same(again, long_ref.bounds(c.host, c.k, old))


# ------------------------------------------------------------------ selection

# dtype, heads, kv heads, dim, page, past, new, starts, prefix, count, first, last
PICK = [
    (F32, 8, 2, 64, 16, [900, 40, 0], 1, None, 0, 16, 1, 2),
    (BF16, 32, 8, 128, 64, [4000, 3, 700], 1, None, 0, 8, 0, 1),
    (F16, 6, 2, 64, 8, [1000, 999], 5, None, 333, 40, 4, 4),                  # three heads a key head, drafts over a prefix that ends inside a page
    (BF16, 16, 1, 256, 8, [70, 200, 1], 3, [0, 1, 1, 4], 17, 5, 1, 1),        # more heads than are taken together; a sequence without new tokens
    (F32, 5, 1, 128, 24, [500], 1, None, 100, 3, 0, 3),                       # those that are taken whatever they are worth, and no more
    (F16, 2, 2, 256, 16, [5000, 100], 1, None, 0, 400, 2, 2),                 # more than there are
    (BF16, 4, 4, 64, 8, [20000], 2, None, 0, 300, 1, 1),                      # as many heads as key heads; thousands of pages
    (F32, 2, 1, 256, 8, [600], 1, None, 9, 1, 0, 1),
    (F16, 3, 1, 64, 8, [40000, 100], 1, None, 0, 200, 4, 4),                  # more pages than one form's registers hold, and than another's
    (BF16, 2, 1, 64, 8, [150000], 1, None, 5, 77, 1, 2),
    (BF16, 4, 1, 128, 16, [16000, 9000], 1, None, 0, 50, 0, 1),               # one launch, a row's pages shared out
    (F32, 32, 2, 64, 8, [4000], 3, None, 0, 20, 0, 2),
    (F16, 8, 8, 64, 16, [1000] * 40, 1, None, 300, 30, 1, 1),                 # many rows
]


def bounds_like(c, scale=1.0):
    low = randn(c.gen, c.total, c.kv_heads, c.dim, scale=scale)
    return torch.stack((low, low + randn(c.gen, c.total, c.kv_heads, c.dim, scale=scale).abs()), 2).to(c.dtype)


@pytest.mark.parametrize("case", PICK, ids=lambda c: "%s-%dx%dx%d-p%d-%d" % (str(c[0])[6:], c[1], c[2], c[3], c[4], c[9]))
@pytest.mark.parametrize("kind", ["values", "ties"])
def test_selection(cuda, case, kind):
    from paella_amd import long_cache
    dtype, heads, kv_heads, dim, page, past, new, starts, prefix, count, first, last = case
    c = Case(heads + dim, dtype, kv_heads, dim, page, past, new, starts, prefix, behind=2 if starts else 0)
    cache, batch = c.to(cuda)
    q, bounds = c.queries(heads), bounds_like(c)
    if kind == "ties":   # small whole numbers, mostly none: equal worths by the dozen
        q, bounds = (q > 2.0).to(dtype), bounds.float().round().clamp(-1, 1).to(dtype)
    select = long_cache.PageSelect(heads, cache, batch, count, first=first, last=last)
    pages = torch.full((c.tokens, kv_heads, count), -7, dtype=torch.int32, device=cuda)
    wide = torch.zeros((c.tokens, heads + 3, dim), dtype=dtype, device=cuda)
    wide[:, :heads] = q.to(cuda)
    assert select(wide[:, :heads], bounds.to(cuda), cache, batch, out=pages) is pages
    same(pages, long_ref.pick(c.host, q, bounds, count, first, last))


def test_selection_of_bad_pages_of_no_numbers_and_of_infinite_ones(cuda):
    from paella_amd import long_cache
    c = Case(8, F32, 1, 64, 8, [200, 100, 30], 1, prefix=50, bad=[((0, 3), -1), ((0, 25), 0), ((-1, 2), 4), ((2, 3), 1)], each=27)
    cache, batch = c.to(cuda)
    q, bounds = c.queries(3), bounds_like(c)
    bounds[c.tables[0, 7], 0, 0, 5] = -math.inf
    bounds[c.tables[0, 9], 0, 1, 6] = math.nan
    bounds[c.tables[1, 4], 0, 1, 0] = math.inf
    bounds[c.tables[1, 5], 0] = 3e38
    bounds[c.tables[1, 6], 0] = -3e38
    q[1, 0, 0] = 0.0   # nothing times infinity
    for count in (2, 6, 12):
        select = long_cache.PageSelect(3, cache, batch, count, first=1, last=1)
        same(select(q.to(cuda), bounds.to(cuda), cache, batch), long_ref.pick(c.host, q, bounds, count, 1, 1))


def test_selection_decided_in_the_last_digits(cuda):
    """Worths that 32 bits do not tell apart."""
    from paella_amd import long_cache
    c = Case(1, F32, 1, 64, 8, [797], 1)
    cache, batch = c.to(cuda)
    q = torch.ones((1, 1, 64))
    bounds = torch.zeros((c.total, 1, 2, 64))
    for e in range(99):
        bounds[c.tables[0, e], 0, :, 0] = 2.0 ** 20
        bounds[c.tables[0, e], 0, :, 63] = ((e * 37) % 99) * 2.0 ** -20
    select = long_cache.PageSelect(1, cache, batch, 20)
    got = select(q.to(cuda), bounds.to(cuda), cache, batch)
    same(got, long_ref.pick(c.host, q, bounds, 20, 0, 1))
    assert set(got.flatten().tolist()) == {e for e in range(99) if (e * 37) % 99 >= 80} | {99}


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=lambda d: str(d)[6:])
def test_selection_by_subnormal_bounds_and_by_the_largest(cuda, dtype):
    """Products of the type's least numbers count, and sums beyond 32 bits are compared like any."""
    from paella_amd import long_cache
    c = Case(2, dtype, 1, 64, 8, [1600], 1)
    cache, batch = c.to(cuda)
    info = torch.finfo(dtype)
    large = math.sqrt(info.max) if dtype == F16 else 2.0 ** 120
    least = info.smallest_normal / 2 ** (4 if dtype == BF16 else 6)
    ones = (1.0 + torch.rand((c.total, 1, 2, 64), generator=c.gen)).float()
    for q, bounds in (((torch.rand((1, 3, 64), generator=c.gen) * large).to(dtype), (ones * least).to(dtype)),
                      ((torch.rand((1, 3, 64), generator=c.gen) * info.max * 0.5).to(dtype), (ones * large).to(dtype)),
                      ((torch.rand((1, 3, 64), generator=c.gen) * least).to(dtype), (ones * least).to(dtype))):
        bounds = bounds.sort(2).values
        mixed = bounds.clone()
        mixed[::2] *= -1
        for b in (bounds, mixed.sort(2).values):
            select = long_cache.PageSelect(3, cache, batch, 30)
            same(select(q.to(cuda), b.to(cuda), cache, batch), long_ref.pick(c.host, q, b, 30, 0, 1))


# ------------------------------------------------------------------ attention over picked pages

# dtype, heads, kv heads, dim, page, past, new, starts, prefix, count
ATTEND = [
    (F32, 8, 2, 64, 16, [900, 40, 0], 1, None, 0, 16),
    (BF16, 32, 8, 128, 64, [4000, 3, 700], 1, None, 0, 8),
    (F16, 6, 2, 64, 8, [1000, 999], 5, None, 333, 40),
    (BF16, 16, 1, 256, 8, [70, 200, 1], 3, [0, 1, 1, 4], 17, 5),
    (F32, 5, 1, 128, 24, [500], 1, None, 100, 3),
    (F32, 2, 1, 256, 8, [600], 1, None, 9, 1),
    (BF16, 20, 1, 128, 32, [700, 64], 2, None, 64, 9),          # more heads a key head than a tile has rows
    (F16, 4, 4, 128, 16, [20000], 1, None, 0, 700),             # a long list, shared out
    (F32, 4, 1, 64, 8, [9000], 1, None, 1000, 1100),
    (F16, 3, 1, 256, 128, [5000], 2, None, 0, 30),
    (BF16, 8, 8, 64, 40, [400] * 40, 1, None, 77, 6),           # many rows: one workgroup each
]


def lists(c, count, order):
    """Pages that a row sees, in any number up to count; its own one among them."""
    out = torch.full((c.tokens, c.kv_heads, count), -1, dtype=torch.int32)
    for t, owner in enumerate(c.host.rows):
        if owner is None:
            continue
        n = c.host.pages_seen(owner[1], owner[0])
        for h in range(c.kv_heads):
            some = torch.randperm(n, generator=c.gen)[:count - (t + h) % 3 if count > 3 else count]
            if order == "picked":
                some = some.sort().values
                if not (some == n - 1).any():
                    some[-1] = n - 1
            out[t, h, :len(some)] = some.to(torch.int32)
    return out


@pytest.mark.parametrize("case", ATTEND, ids=lambda c: "%s-%dx%dx%d-p%d-%d" % (str(c[0])[6:], c[1], c[2], c[3], c[4], c[9]))
@pytest.mark.parametrize("order", ["picked", "any"])
def test_attention(cuda, case, order):
    from paella_amd import long_cache
    dtype, heads, kv_heads, dim, page, past, new, starts, prefix, count = case
    c = Case(heads * 3 + dim, dtype, kv_heads, dim, page, past, new, starts, prefix, behind=2 if starts else 0)
    cache, batch = c.to(cuda)
    q, pages = c.queries(heads), lists(c, count, order)
    attend = long_cache.PageAttention(heads, cache, batch, count)
    out = torch.full(q.shape, 7.0, dtype=dtype, device=cuda)
    assert attend(q.to(cuda), cache, batch, pages.to(cuda), out=out) is out
    want, weight, products, most = long_ref.attend(c.host, q, c.k, c.v, pages, 1 / math.sqrt(dim))
    live = torch.tensor([o is not None for o in c.host.rows])
    within(out[live.to(cuda)], want[live], ref.attention_bound(want, weight, products, dtype, most)[live])
    assert (out[~live.to(cuda)] == 7.0).all()
    first = out.clone()
    for _ in range(2):   # the same in every run, whatever the last call left in the workspace
        attend(q.to(cuda), cache, batch, pages.to(cuda), out=out)
        assert torch.equal(out, first)


def test_attention_over_odd_lists(cuda):
    """Entries that name nothing wherever they stand, pages outside the cache, pages a row does not see yet, a page twice, and a row that sees nothing."""
    from paella_amd import long_cache
    c = Case(5, BF16, 2, 64, 8, [100, 30, 11], 2, prefix=21, bad=[((0, 4), -1), ((-1, 1), 0)], each=14)
    cache, batch = c.to(cuda)
    q = c.queries(6)
    pages = torch.full((c.tokens, 2, 12), -1, dtype=torch.int32)
    pages[0, 0] = torch.tensor([-1, 3, 99, 7, 16, -5, 2, 1, 2 ** 31 - 1, -2 ** 31, 5, 0])
    pages[0, 1] = torch.tensor([15, 14, 13, 12, 11, 10, 9, 8, 7, 6, 5, 4])
    pages[1, 0] = torch.tensor([1, 7, -1, -1, -1, -1, -1, -1, -1, -1, -1, -1])           # both outside the cache
    pages[2] = torch.tensor([3, 3, 4, 4, 4, 0, 2, 16, 15, 14, 17, 18])                   # some twice, some behind the sequence
    pages[3, 1, 11] = 6
    pages[4] = 4
    attend = long_cache.PageAttention(6, cache, batch, 12, scale=0.3)
    out = attend(q.to(cuda), cache, batch, pages.to(cuda))
    want, weight, products, most = long_ref.attend(c.host, q, c.k, c.v, pages, 0.3)
    within(out, want, ref.attention_bound(want, weight, products, BF16, most))
    assert (out[1, :3] == 0).all() and (out[3, :3] == 0).all() and (out[5] == 0).all()


def test_attention_over_all_pages_is_attention(cuda):
    """Lists of every page give what the decoding step's attention gives."""
    from paella_amd import decode, long_cache
    for dtype, dim in ((F32, 64), (BF16, 128), (F16, 256)):
        c = Case(dim, dtype, 2, dim, 16, [100, 37], 3, prefix=40)
        cache, batch = c.to(cuda)
        q = c.queries(8)
        pages = torch.arange(10, dtype=torch.int32).expand(c.tokens, 2, 10).contiguous()
        out = long_cache.PageAttention(8, cache, batch, 10)(q.to(cuda), cache, batch, pages.to(cuda))
        whole = decode.PrefixAttention(8, cache, batch)(q.to(cuda), cache, batch)
        want, weight, products, most = long_ref.attend(c.host, q, c.k, c.v, pages, 1 / math.sqrt(dim))
        bound = ref.attention_bound(want, weight, products, dtype, most)
        within(out, want, bound)
        within(whole, want, bound)


# ------------------------------------------------------------------ weights

# dtype, heads, kv heads, dim, page, past, new, starts, prefix
WEIGH = [
    (F32, 8, 2, 64, 16, [300, 40, 0], 1, None, 0),
    (BF16, 32, 8, 128, 64, [900, 3, 700], 1, None, 0),
    (F16, 6, 2, 64, 8, [100, 99], 5, None, 33),
    (BF16, 16, 1, 256, 8, [70, 200, 1], 3, [0, 1, 1, 4], 17),
    (F32, 5, 1, 128, 24, [500], 1, None, 100),
    (F32, 2, 1, 256, 8, [60], 1, None, 9),
    (BF16, 8, 2, 128, 32, [200, 64], 33, None, 64),            # two chunks of rows, the second not full
    (F16, 3, 1, 64, 16, [0, 10], 70, [0, 70, 80], 0),          # prompts
    (F32, 4, 2, 256, 40, [100], 12, None, 50),
    (F16, 2, 2, 256, 8, [0], 1, None, 0),                      # a single key
]


@pytest.mark.parametrize("case", WEIGH, ids=lambda c: "%s-%dx%dx%d-p%d-%d" % (str(c[0])[6:], c[1], c[2], c[3], c[4], c[6]))
def test_weights(cuda, case):
    from paella_amd import long_cache
    dtype, heads, kv_heads, dim, page, past, new, starts, prefix = case
    c = Case(heads * 5 + dim, dtype, kv_heads, dim, page, past, new, starts, prefix, behind=2 if starts else 0)
    cache, batch = c.to(cuda)
    q = c.queries(heads)
    plan = long_cache.KeyWeights(heads, cache, batch)
    places = c.tables.shape[1] * page
    old = torch.rand((len(past), kv_heads, places), generator=c.gen)
    for b, p in enumerate(past):
        old[b, :, p:] = math.nan   # what new tokens and places behind them hold does not matter, and stays behind them
    weights = old.to(cuda)
    assert plan(q.to(cuda), cache, batch, weights) is weights
    want, error = long_ref.weigh(c.host, q, c.k, old, 1 / math.sqrt(dim))
    kept = want.isnan()
    assert torch.equal(weights.cpu().isnan(), kept)
    within(weights.cpu().masked_fill(kept, 0), want.masked_fill(kept, 0), error.masked_fill(kept, 0))
    again = old.to(cuda)
    plan(q.to(cuda), cache, batch, again)
    same(again, weights)


def test_weights_of_bad_pages_and_of_rows_that_see_nothing(cuda):
    from paella_amd import long_cache
    c = Case(9, BF16, 1, 64, 8, [20, 50, 3], 2, prefix=20, bad=[((0, 1), -1), ((-1, 1), 7)], each=4)   # sequence 1 goes past its table
    cache, batch = c.to(cuda)
    q = c.queries(4)
    old = torch.rand((3, 1, 32), generator=c.gen)
    weights = old.to(cuda)
    plan = long_cache.KeyWeights(4, cache, batch, scale=0.2)
    plan(q.to(cuda), cache, batch, weights)
    want, error = long_ref.weigh(c.host, q, c.k, old, 0.2)
    within(weights, want, error)
    alone = Case(9, BF16, 1, 64, 8, [5, 6], 1, bad=[((0, 0), -1)])
    cache, batch = alone.to(cuda)
    weights = torch.ones((2, 1, 8), device=cuda)
    long_cache.KeyWeights(4, cache, batch)(alone.queries(4).to(cuda), cache, batch, weights)
    assert torch.equal(weights[0].cpu(), torch.tensor([[1.0, 1, 1, 1, 1, 0, 1, 1]]))


# ------------------------------------------------------------------ eviction

# dtype, kv heads, dim, page, past, keep, first, recent
EVICT = [
    (F32, 2, 64, 16, [300, 100, 101, 99, 0], 100, 4, 20),
    (BF16, 8, 128, 64, [900, 1], 64, 0, 0),
    (F16, 1, 256, 24, [700], 699, 0, 10),
    (BF16, 3, 40, 8, [50, 3000], 7, 3, 4),              # nothing is chosen
    (F32, 1, 512, 8, [200, 64], 33, 1, 0),
    (F16, 2, 8, 8, [5000], 1, 0, 1),
    (BF16, 2, 96, 128, [2000], 1500, 100, 300),
    (F32, 1, 64, 8, [40], 1000, 3, 3),                  # longer than any
    (F16, 1, 8, 8, [9000, 3000], 2100, 4, 8),           # longer than one form's registers hold, and than another's
    (BF16, 1, 8, 8, [20000], 1900, 0, 100),
]


@pytest.mark.parametrize("case", EVICT, ids=lambda c: "%s-%dx%d-p%d-%d" % (str(c[0])[6:], c[1], c[2], c[3], c[5]))
@pytest.mark.parametrize("kind", ["values", "ties"])
def test_eviction(cuda, case, kind):
    from paella_amd import long_cache
    dtype, kv_heads, dim, page, past, keep, first, recent = case
    c = Case(dim + keep, dtype, kv_heads, dim, page, past)
    cache, batch = c.to(cuda)
    old = torch.rand((len(past), kv_heads, c.tables.shape[1] * page), generator=c.gen) ** 12
    if kind == "ties":
        old = (old * 3).round()
    k, v, weights, dev = c.k.clone(), c.v.clone(), old.clone(), old.to(cuda)
    evict = long_cache.Evict(cache, len(past), c.tables.shape[1], keep, first=first, recent=recent)
    in_place = kind == "ties"
    got_past, kept = evict(cache, dev, batch.past, batch.tables, past_out=batch.past if in_place else None)
    want_kept, want_past = long_ref.evict(past, c.tables, c.total, k, v, weights, keep, first, recent)
    same(kept, want_kept)
    assert got_past.tolist() == want_past and batch.past.tolist() == (want_past if in_place else past)
    for got, want in ((cache.k, k), (cache.v, v), (dev, weights)):
        same(got, want)


def test_eviction_of_odd_weights_lengths_and_pages(cuda):
    from paella_amd import long_cache
    c = Case(4, BF16, 2, 64, 8, [100, 60, 60, 60], bad=[((0, 2), -1), ((0, 9), 5), ((3, 0), -2)])
    cache, batch = c.to(cuda)
    old = torch.randn((4, 2, c.tables.shape[1] * 8), generator=c.gen)
    old[0, 0, 3:60:5] = math.nan
    old[1, 0, 2:9] = torch.tensor([math.inf, -math.inf, 0.0, -0.0, -math.nan, 1e-40, -1e-40])
    old[1, 1] = 0.0
    old[1, 1, ::2] = -0.0
    old[2, 0] = math.nan
    old[2, 1] = -math.inf
    for keep, first, recent in ((30, 2, 5), (59, 0, 0), (1, 0, 0)):
        k, v, weights, dev = c.k.clone(), c.v.clone(), old.clone(), old.to(cuda)
        cache, batch = c.to(cuda)
        past = [100, -3, 60, 2 ** 31 - 1] if keep == 30 else c.past
        batch.past.copy_(torch.tensor(past, dtype=torch.int32))
        got_past, kept = long_cache.Evict(cache, 4, c.tables.shape[1], keep, first=first, recent=recent)(cache, dev, batch.past, batch.tables)
        want_kept, want_past = long_ref.evict(past, c.tables, c.total, k, v, weights, keep, first, recent)
        same(kept, want_kept)
        assert got_past.tolist() == want_past
        for got, want in ((cache.k, k), (cache.v, v), (dev, weights)):
            same(got, want)


# ------------------------------------------------------------------ positions

def test_append_at_positions(cuda):
    """Rotation by given positions; places in the cache as ever."""
    from paella_amd import decode
    for dtype, interleaved in ((F32, False), (BF16, True)):
        c = Case(2, dtype, 2, 64, 16, [5, 30, 0], 3, prefix=20)
        cache, batch = c.to(cuda)
        heads = 4
        q, k, v = (randn(c.gen, c.tokens, n, 64, dtype=dtype) for n in (heads, 2, 2))
        freq = torch.tensor([10000.0 ** (-2 * i / 64) for i in range(32)])
        positions = [100000, 7, 2 ** 30]
        dev = [t.to(cuda) for t in (q, k, v)]
        out = decode.kv_append(cache, batch, dev[1], dev[2], q=dev[0], inv_freq=freq.to(cuda), interleaved=interleaved, positions=torch.tensor(positions, dtype=torch.int32, device=cuda))
        for t, (b, own) in enumerate(c.host.rows):
            at = positions[b] + own - c.past[b]
            p = c.host.physical(b, c.host.shared + own // 16)
            for got, x in ((out[t], q[t]), (cache.k[p, :, own % 16], k[t])):
                want = ref.norm_rotate(x.double(), None, 0.0, freq.double().tolist(), interleaved, at)
                # the angle of position 2^30 in 64 bits is off by 2^-53 * 2^30 turns; for the rest as in test_append
                within(got, want, ref.HALF_STEP[dtype] * want.abs() + 64 * 2.0 ** -24 * want.abs().amax(-1, keepdim=True))
            assert torch.equal(cache.v[p, :, own % 16].cpu(), v[t])


# ------------------------------------------------------------------ together

@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=lambda d: str(d)[6:])
def test_a_long_cache_is_read_and_kept_in_part(cuda, dtype):
    """Steps of two sequences behind a prefix: append, bounds, selection, attention over the picked pages, weights; then an eviction, bounds anew, and steps at later positions.  Every step against the
    definitions on what the cache holds."""
    from paella_amd import decode, long_cache
    heads, kv_heads, dim, page, count = 8, 2, 64, 8, 5
    c = Case(6, dtype, kv_heads, dim, page, [61, 40], 1, prefix=19, each=12)
    cache, batch = c.to(cuda)
    past = batch.past
    positions = past + 19
    bounds, weights = long_cache.new_bounds(cache), long_cache.new_weights(cache, batch)
    everything = decode.KVBatch(torch.zeros(2, dtype=torch.int32, device=cuda), batch.tables, max_new=61, starts=torch.tensor([0, 61, 101], dtype=torch.int32, device=cuda), tokens=101)
    shared = decode.KVBatch(torch.zeros(1, dtype=torch.int32, device=cuda), batch.prefix_table[None], max_new=19)
    for b in (everything, shared):
        long_cache.page_bounds(cache, bounds, b)
    freq = torch.tensor([10000.0 ** (-2 * i / dim) for i in range(dim // 2)], device=cuda)
    select, attend = long_cache.PageSelect(heads, cache, batch, count, first=1, last=2), long_cache.PageAttention(heads, cache, batch, count)
    weigh, evict = long_cache.KeyWeights(heads, cache, batch), long_cache.Evict(cache, 2, 12, 33, first=2, recent=6)
    lengths = [61, 40]

    def step():
        q, k, v = (randn(c.gen, 2, n, dim, dtype=dtype, scale=1.5).to(cuda) for n in (heads, kv_heads, kv_heads))
        q = decode.kv_append(cache, batch, k, v, q=q, inv_freq=freq, positions=positions)
        long_cache.page_bounds(cache, bounds, batch)
        pages = select(q, bounds, cache, batch)
        out = attend(q, cache, batch, pages)
        before = weights.cpu()
        weigh(q, cache, batch, weights)
        host = long_ref.Sequences(None, lengths, 1, 2, c.tables, c.prefix_table, 19, page, c.total)
        keys, values = cache.k.cpu(), cache.v.cpu()
        for b in range(2):   # bounds are those of the keys, of all pages
            for e in range(host.pages_seen(lengths[b], b)):
                p, n = host.physical(b, e), host.seen_in(b, lengths[b], e)
                same(bounds[p], torch.stack((keys[p, :, :n].amin(1), keys[p, :, :n].amax(1)), 1))
        same(pages, long_ref.pick(host, q.cpu(), bounds.cpu(), count, 1, 2))
        want, weight, products, most = long_ref.attend(host, q.cpu(), keys, values, pages.cpu(), 1 / math.sqrt(dim))
        within(out, want, ref.attention_bound(want, weight, products, dtype, most))
        want, error = long_ref.weigh(host, q.cpu(), keys, before, 1 / math.sqrt(dim))
        within(weights, want, error)
        past.add_(1)
        positions.add_(1)
        for b in range(2):
            lengths[b] += 1

    for _ in range(4):
        step()
    k, v, w = cache.k.cpu(), cache.v.cpu(), weights.cpu()
    want_kept, want_past = long_ref.evict(lengths, c.tables, c.total, k, v, w, 33, 2, 6)
    _, kept = evict(cache, weights, past, batch.tables, past_out=past)
    same(kept, want_kept)
    assert past.tolist() == want_past == [33, 33]
    for got, want in ((cache.k, k), (cache.v, v), (weights, w)):
        same(got, want)
    lengths[:] = want_past
    kept_batch = decode.KVBatch(torch.zeros(2, dtype=torch.int32, device=cuda), batch.tables, max_new=33)
    long_cache.page_bounds(cache, bounds, kept_batch)
    for _ in range(9):   # into the next page
        step()
