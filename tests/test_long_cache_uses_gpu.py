"""The operators over long caches as programs use them: in graphs, on other streams and direct-dispatch queues, stage by stage, by several threads, over strided rows and pages behind 32 bits, with a
notifier.  What they compute is tested in test_long_cache_gpu.py; here every use gives the bits of an eager call."""
import ctypes
import threading

import pytest
import torch

from test_decode_gpu import BF16, F16, F32, randn
from test_long_cache_gpu import Case, bounds_like, lists, same

pytestmark = pytest.mark.gpu


class Use:
    """An operator with inputs, and outputs made for a call: fresh() gives memory for them, begin(state) fills it as it is before a call, call(state) issues the call, results(state) are what it wrote."""

    def __init__(self, name, cuda):
        from paella_amd import long_cache
        dtype, heads, kv_heads, dim, page, past, new, prefix, count, stages = USES[name]
        c = self.case = Case(len(name) + dim, dtype, kv_heads, dim, page, past, new, prefix=prefix)
        self.cache, self.batch = c.to(cuda)
        self.kind, self.stages, places = name.split()[0], stages, c.tables.shape[1] * page
        self.q = c.queries(heads).to(cuda)
        self.bounds = bounds_like(c).to(cuda)
        self.pages = lists(c, count, "any").to(cuda)
        self.old = torch.rand((len(past), kv_heads, places), generator=c.gen).to(cuda)
        self.plan = {"bounds": lambda: None, "select": lambda: long_cache.PageSelect(heads, self.cache, self.batch, count, first=1, last=2),
                     "attend": lambda: long_cache.PageAttention(heads, self.cache, self.batch, count), "weigh": lambda: long_cache.KeyWeights(heads, self.cache, self.batch),
                     "evict": lambda: long_cache.Evict(self.cache, len(past), c.tables.shape[1], count, first=3, recent=4)}[self.kind]()
        assert self.plan is None or (self.plan.stages if self.kind == "evict" else self.plan.plan.stages) == stages
        self.spaces = self.kind in ("select", "attend", "weigh") and self.plan.plan.workspace_bytes > 0

    def fresh(self):
        from paella_amd import decode
        s = {"bounds": dict(out=torch.empty_like(self.bounds)), "select": dict(out=torch.empty_like(self.pages)), "attend": dict(out=torch.empty_like(self.q)), "weigh": dict(out=torch.empty_like(self.old)),
             "evict": dict(k=torch.empty_like(self.cache.k), v=torch.empty_like(self.cache.v), weights=torch.empty_like(self.old), past=torch.empty_like(self.batch.past),
                           kept=self.batch.past.new_empty((len(self.case.past), self.case.kv_heads, self.plan.desc.keep if self.kind == "evict" else 1)))}[self.kind]
        if self.kind == "evict":
            s["cache"] = decode.KVCache(s["k"], s["v"])
        return self.begin(s)

    def begin(self, s):
        if self.kind in ("bounds", "weigh"):
            s["out"].copy_(self.bounds if self.kind == "bounds" else self.old)
        elif self.kind == "evict":
            for name, t in (("k", self.cache.k), ("v", self.cache.v), ("weights", self.old), ("past", self.batch.past)):
                s[name].copy_(t)
            s["kept"].fill_(-9)
        else:
            s["out"].fill_(-9)
        return s

    def call(self, s, q=None, **kw):
        from paella_amd import long_cache
        if self.kind == "bounds":
            long_cache.page_bounds(self.cache, s["out"], self.batch, **kw)
        elif self.kind == "evict":
            self.plan(s["cache"], s["weights"], s["past"], self.batch.tables, past_out=s["past"], kept=s["kept"], **kw)
        else:
            q = self.q if q is None else q
            args = {"select": (q, self.bounds, self.cache, self.batch), "attend": (q, self.cache, self.batch, self.pages), "weigh": (q, self.cache, self.batch, s["out"])}[self.kind]
            self.plan(*args, **kw, **({} if self.kind == "weigh" else dict(out=s["out"])))
        return s

    def results(self, s):
        return [s[n] for n in (("k", "v", "weights", "past", "kept") if self.kind == "evict" else ("out",))]

    def check(self, s, want):
        for got, w in zip(self.results(s), want):
            same(got, w)

    def eager(self, q=None):
        s = self.call(self.fresh(), q)
        torch.cuda.synchronize()
        return [t.clone() for t in self.results(s)]


# dtype, heads, kv heads, dim, page, past, new, prefix, count (or what an eviction keeps), launches of a call
USES = {
    "bounds": (BF16, 4, 2, 128, 16, [700, 31, 100], 5, 0, 4, 1),
    "select at once": (F32, 4, 2, 64, 8, [900, 40, 300], 1, 21, 9, 1),
    "select in two": (BF16, 16, 8, 128, 16, [9000, 40, 3000, 5000], 3, 40, 30, 2),
    "attend alone": (BF16, 4, 4, 64, 16, [300] * 200, 1, 0, 4, 1),
    "attend joined": (F16, 8, 2, 128, 16, [9000, 500], 1, 100, 200, 1),
    "attend in many": (F16, 8, 2, 128, 16, [9000, 500], 1, 100, 300, 2),
    "attend in two": (BF16, 16, 1, 256, 16, [4000, 500], 1, 0, 200, 2),
    "weigh few": (BF16, 8, 2, 128, 16, [3000, 100], 2, 70, 4, 2),
    "weigh many": (F16, 8, 2, 64, 16, [3000, 100], 9, 0, 4, 2),
    "evict": (BF16, 2, 2, 128, 16, [3000, 200, 90], 1, 0, 100, 2),
}
every = pytest.mark.parametrize("name", USES)


@every
def test_graphs_and_streams(cuda, name):
    """Another stream; two graphs of one plan replayed side by side, lengths changed between replays, eager calls between."""
    use = Use(name, cuda)
    want = use.eager()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        s = use.call(use.fresh())
    torch.cuda.synchronize()
    use.check(s, want)
    states, graphs = [use.fresh() for _ in range(2)], []
    torch.cuda.synchronize()
    for s in states:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            use.call(use.begin(s))
        graphs.append(graph)
    longer, shorter = use.batch.past.clone(), (use.batch.past - 100).clamp(min=0)
    for past in (longer, shorter, longer, shorter, longer):
        use.batch.past.copy_(past)
        now = use.eager()
        with torch.cuda.stream(side):
            graphs[0].replay()
        graphs[1].replay()
        busy = use.eager()
        torch.cuda.synchronize()
        for s in states:
            use.check(s, now)
        for got, w in zip(busy, now):
            same(got, w)
    for got, w in zip(now, want):
        same(got, w)


@every
def test_direct_queues(cuda, name):
    from paella_amd import ops
    use = Use(name, cuda)
    want = use.eager()
    staged = name.split()[0] in ("select", "attend", "weigh", "evict")
    with ops.DirectQueue() as queue:
        for _ in range(2):
            s = use.fresh()
            torch.cuda.synchronize()
            for stage in range(use.stages):
                use.call(s, stream=queue.handle, **(dict(stage=stage) if staged else {}))
                queue.wait()
            use.check(s, want)
        if use.stages > 1:
            with pytest.raises(RuntimeError, match="-2"):
                use.call(s, stream=queue.handle)
    with ops.DirectQueue(ordered=True) as queue:
        states = [use.fresh() for _ in range(2)]
        torch.cuda.synchronize()
        for s in states:
            use.call(s, stream=queue.handle)
        queue.wait()
        for s in states:
            use.check(s, want)


@pytest.mark.parametrize("name", [n for n in USES if n.split()[0] in ("select", "attend", "weigh") and n != "attend alone"])
def test_calls_captured_on_a_side_stream_need_a_workspace(cuda, name):
    use = Use(name, cuda)
    assert use.spaces
    want, space, s = use.eager(), use.plan.new_workspace(), use.fresh()
    home, side, graph = torch.cuda.Stream(), torch.cuda.Stream(), torch.cuda.CUDAGraph()   # (one after the other: two of torch's streams)
    assert home.cuda_stream != side.cuda_stream
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=home):
        use.begin(s)
        side.wait_stream(home)
        with pytest.raises(AssertionError):
            use.call(s, stream=side.cuda_stream)
        use.call(s, stream=side.cuda_stream, workspace=space)
        home.wait_stream(side)
    for _ in range(3):
        graph.replay()
        again = use.eager()
        use.check(s, want)
        for got, w in zip(again, want):
            same(got, w)


@pytest.mark.parametrize("name", [n for n in USES if n not in ("bounds", "evict")])
def test_threads_that_share_a_plan_and_a_stream(cuda, name):
    use = Use(name, cuda)
    queries = [(use.q.float() * f).to(use.q.dtype) for f in (1.0, 0.5, -0.75, 0.25)]
    want = [use.eager(q) for q in queries]
    made, start = [[] for _ in queries], threading.Barrier(len(queries))

    def calls(i):
        torch.cuda.set_device(cuda)
        start.wait()
        for _ in range(10):
            made[i].append(use.call(use.fresh(), queries[i]))

    threads = [threading.Thread(target=calls, args=(i,)) for i in range(len(queries))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for i, mine in enumerate(made):
        assert len(mine) == 10
        for s in mine:
            use.check(s, want[i])


@pytest.mark.parametrize("name", [n for n in USES if n not in ("bounds", "evict")])
def test_queries_that_lie_apart(cuda, name):
    use = Use(name, cuda)
    want = use.eager()
    t, h, d = use.q.shape
    wide = torch.full((t, h + 1, d), float("nan"), dtype=use.q.dtype, device=cuda)
    wide[:, :h] = use.q
    use.check(use.call(use.fresh(), wide[:, :h]), want)
    for first in (wide[:, 0].clone()[:, None].expand(t, h, d), wide.transpose(0, 1).contiguous().transpose(0, 1)[:, :h]):   # heads that do not lie side by side
        if h > 1 and t > 1:
            with pytest.raises(AssertionError):
                use.call(use.fresh(), first)


@every
def test_a_call_reports_to_its_notifier(cuda, name):
    """A call's last launch sends end messages that add up to the grid that its dims announce."""
    import numpy as np
    from paella_amd import _abi
    lib, use = _abi.ops(), Use(name, cuda)
    dims = _abi.LaunchDims()
    if name == "bounds":
        assert lib.paella_page_bounds_dims(use.cache.ref, use.batch.ref, ctypes.byref(dims)) == 0
    else:
        dims = use.plan.dims(use.cache, 1) if name == "evict" else use.plan.dims(use.stages - 1)
    ring = ctypes.c_void_p()
    _abi.check(lib.paella_ring_create(4096, 1, ctypes.byref(ring)), "paella_ring_create")
    try:
        assert dims.block % 64 == 0 and 0 < dims.vgprs <= 512 and dims.lds_bytes <= 160 * 1024
        s = use.call(use.fresh(), job_id=17, notifier=lib.paella_ring_notifier(ring, 0))
        torch.cuda.synchronize()
        messages = 2 * -(-dims.grid // lib.paella_ring_batch_size())
        bits = np.zeros(messages, np.uint64)
        assert lib.paella_ring_drain(ring, bits.ctypes.data, messages, 20.0) == messages and not lib.paella_ring_can_read(ring)
        num, start, job = (bits >> np.uint64(16)) & np.uint64(0xFF), bits & np.uint64(0xFF), bits >> np.uint64(32)
        assert int(num[start == 0].sum()) == dims.grid == int(num[start == 1].sum()) and set(job.tolist()) == {17}
        use.check(s, use.eager())
    finally:
        lib.paella_ring_destroy(ring)


def test_pages_behind_32_bits(cuda):
    """Keys, values and bounds of pages whose offsets pass 2^32 bytes: the bits of the same pages in a small cache."""
    from paella_amd import decode, long_cache
    heads, kv_heads, dim, page, count, each = 8, 4, 128, 8, 11, 40
    c = Case(3, BF16, kv_heads, dim, page, [311, 150], 1, prefix=20, each=each)
    small, batch = c.to(cuda)
    extra = (1 << 32) // (2 * kv_heads * dim * 2) + 5      # pages ahead of the small cache's in the large one
    large = decode.KVCache(*(torch.empty((extra + c.total, kv_heads, page, dim), dtype=BF16, device=cuda) for _ in range(2)))
    large.k[extra:] = small.k
    large.v[extra:] = small.v
    far = decode.KVBatch(batch.past, batch.tables + extra, prefix_table=batch.prefix_table + extra, prefix_len=20)
    bounds = [torch.empty((n, kv_heads, 2, dim), dtype=BF16, device=cuda) for n in (c.total, extra + c.total)]
    bounds[0].copy_(bounds_like(c))
    bounds[1][extra:] = bounds[0]
    q, old = c.queries(heads).to(cuda), torch.rand((2, kv_heads, each * page), generator=c.gen).to(cuda)
    made = []
    for cache, b, low in ((small, batch, bounds[0]), (large, far, bounds[1])):
        long_cache.page_bounds(cache, low, b)
        pages = long_cache.PageSelect(heads, cache, b, count)(q, low, cache, b)
        out = long_cache.PageAttention(heads, cache, b, count)(q, cache, b, pages)
        weights = old.clone()
        long_cache.KeyWeights(heads, cache, b)(q, cache, b, weights)
        past, kept = long_cache.Evict(cache, 2, each, 100, first=2, recent=9)(cache, weights, b.past, b.tables)
        made.append((low[-c.total:], pages, out, weights, past, kept, cache.k[-c.total:], cache.v[-c.total:]))
    torch.cuda.synchronize()
    for got, want in zip(*made):
        same(got, want)
    assert made[0][4].tolist() == [100, 100]


def test_second_stages_over_what_no_first_stage_left(cuda):
    """A workspace or a list that is not this call's: results are of no use, but nothing beside the outputs is written."""
    for name in ("select in two", "evict"):
        use = Use(name, cuda)
        s = use.fresh()
        torch.cuda.synchronize()
        if use.kind == "select":
            for poison in (-1, 0x7F7F7F7F, 1):
                space = use.plan.new_workspace()
                space.fill_(poison)
                wide = torch.full((3,) + s["out"].shape, -9, dtype=torch.int32, device=cuda)
                use.plan(use.q, use.bounds, use.cache, use.batch, out=wide[1], stage=1, workspace=space)
                torch.cuda.synchronize()
                assert (wide[0] == -9).all() and (wide[2] == -9).all()
        else:
            from paella_amd import long_cache
            places = use.old.shape[2]
            for keep, poison in ((100, 2 ** 31 - 1), (places + 50, 2 ** 31 - 1), (places + 50, -5)):
                plan = long_cache.Evict(use.cache, len(use.case.past), use.case.tables.shape[1], keep)
                kept = torch.full((len(use.case.past), use.case.kv_heads, keep), poison, dtype=torch.int32, device=cuda)
                wide = torch.full((3,) + use.old.shape, 0.5, device=cuda)
                plan(s["cache"], wide[1], s["past"], use.batch.tables, past_out=s["past"], kept=kept, stage=1)
                torch.cuda.synchronize()
                assert (wide[0] == 0.5).all() and (wide[2] == 0.5).all()
                same(s["k"], use.cache.k)
                same(s["v"], use.cache.v)


@pytest.mark.parametrize("pages", [100, 1500, 3000, 10000, 20000])
def test_every_form_of_picking_on_direct_queues(cuda, pages):
    from paella_amd import decode, long_cache, ops
    c = Case(pages, BF16, 1, 64, 8, [8 * pages - 5, 100], 3)
    cache, batch = c.to(cuda)
    q, bounds = c.queries(2).to(cuda), bounds_like(c).to(cuda)
    select = long_cache.PageSelect(2, cache, batch, 50)
    weights = torch.rand((2, 1, pages), generator=c.gen).to(cuda)   # an eviction from as many tokens
    tokens = decode.KVCache(*(torch.rand((2 * pages // 4, 1, 8, 8), generator=c.gen).to(cuda) for _ in range(2))) if pages % 8 == 0 else None
    want = select(q, bounds, cache, batch)
    with ops.DirectQueue() as queue:
        out = torch.zeros_like(want)
        torch.cuda.synchronize()
        assert select.plan.stages == 2
        for stage in range(2):
            select(q, bounds, cache, batch, out=out, stage=stage, stream=queue.handle)
            queue.wait()
        same(out, want)
        if tokens is not None:
            evict = long_cache.Evict(tokens, 2, pages // 8, pages // 3, first=2, recent=3)
            past = torch.tensor([pages, pages // 4], dtype=torch.int32, device=cuda)
            tables = torch.randperm(2 * pages // 8, generator=c.gen).to(torch.int32).view(2, pages // 8).to(cuda)
            made = []
            for direct in (False, True):
                k, v, w = tokens.k.clone(), tokens.v.clone(), weights.clone()
                lengths, kept = torch.zeros_like(past), torch.zeros((2, 1, pages // 3), dtype=torch.int32, device=cuda)
                torch.cuda.synchronize()
                for stage in range(2):
                    evict(decode.KVCache(k, v), w, past, tables, past_out=lengths, kept=kept, stage=stage, stream=queue.handle if direct else None)
                    if direct:
                        queue.wait()
                torch.cuda.synchronize()
                made.append((k, v, w, lengths, kept))
            for got, expected in zip(*made):
                same(got, expected)


def test_append_at_positions_on_direct_queues(cuda):
    from paella_amd import decode, ops
    c = Case(12, BF16, 2, 64, 16, [5, 30, 0], 3)
    k, v = (randn(c.gen, c.tokens, 2, 64, dtype=BF16).to(cuda) for _ in range(2))
    q, freq = c.queries(4).to(cuda), torch.rand(32, generator=c.gen).to(cuda)
    positions = torch.tensor([77, 3, 1000], dtype=torch.int32, device=cuda)
    made = []
    with ops.DirectQueue() as queue:
        for direct in (False, True):
            cache, batch = c.to(cuda)
            out = torch.zeros_like(q)
            torch.cuda.synchronize()
            decode.kv_append(cache, batch, k, v, q=q, inv_freq=freq, positions=positions, out=out, stream=queue.handle if direct else None)
            queue.wait()
            torch.cuda.synchronize()
            made.append((out, cache.k, cache.v))
    for got, want in zip(*made):
        same(got, want)
