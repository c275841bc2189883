"""The C-ABI of the operators over long caches without a device: every declared symbol, what the plans plan, and what each entry point refuses before anything is launched."""
import ctypes
import math
import os
import re
import types

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
EINVAL, ENOSUP = -1, -2
AT = 1 << 32   # an address on a boundary of every kind, far from its multiples; none of the calls here gets as far as using it
K, V, PAST, TABLES, STARTS, PREFIX, Q, BOUNDS, PAGES, OUT, SPACE, WEIGHTS, KEPT, LENGTHS = (i * AT for i in range(1, 15))


@pytest.fixture(scope="module")
def lib():
    from paella_amd import _abi
    return _abi.ops()


def cache(dtype=1, pages=10, heads=2, size=16, dim=64, k=K, v=V):
    from paella_amd._abi_decode import KvCache
    return KvCache(k, v, dtype, pages, heads, size, dim)


def batch(sequences=3, max_new=1, tokens=None, max_pages=4, prefix=0, starts=None, past=PAST, tables=TABLES, prefix_table=None):
    from paella_amd._abi_decode import KvBatch
    return KvBatch(sequences, max_new, sequences * max_new if tokens is None else tokens, max_pages, prefix, starts, past, tables, PREFIX if prefix and prefix_table is None else prefix_table)


CACHE_BYTES = 10 * 2 * 16 * 64 * 2
BAD_CACHES = [dict(dtype=3), dict(dtype=-1), dict(pages=0), dict(heads=0), dict(size=12), dict(size=0), dict(dim=60), dict(dim=520)]
BAD_BATCHES = [dict(sequences=0), dict(max_new=0), dict(tokens=0, starts=STARTS), dict(max_pages=0), dict(prefix=-1), dict(prefix=1 << 30)]


def refs(*xs):
    return [ctypes.byref(x) for x in xs]


def test_header_and_table_and_library_agree(lib):
    from paella_amd import _abi_long
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "paella_long_cache.h")).read(), flags=re.S)
    declared = sorted(set(re.findall(r"\b(paella_[a-z0-9_]+)\s*\(", text)))
    assert declared == sorted(_abi_long.LONG_SYMBOLS) and all(hasattr(lib, n) for n in declared)


def test_no_kernel_needs_scratch_memory(lib):
    """Direct-dispatch queues have none to give: by what the library's code objects say of their kernels."""
    built = open(lib._name, "rb").read()
    said = re.findall(rb"\.name[\xa0-\xbf\xd9\xda]..?.?([\w$.]{8,200}?)\xbb\.private_segment_fixed_size(.)", built, flags=re.S)
    kernels = {name.decode(): size for name, size in said if re.search(rb"page_(bounds|screen|pick|select|attention)_kernel|evict_\w+_kernel|key_(sums|weights)_kernel|stored_weights_kernel", name)}
    assert len(kernels) == 12 + 9 + 9 + 5 + 9 + 4 + 1 + 18 + 9 + 1, sorted(kernels)
    assert [name for name, size in kernels.items() if size != b"\0"] == []


# ------------------------------------------------------------------ bounds

def bounds(lib, c=None, b=None, at=BOUNDS):
    return lib.paella_page_bounds_launch(*refs(c or cache(), b or batch()), at, None, 0, None)


def test_bounds_refuse(lib):
    from paella_amd import _abi
    assert [bounds(lib, c=cache(**kw)) for kw in BAD_CACHES + [dict(k=None), dict(v=None), dict(k=K + 8)]] == [EINVAL] * (len(BAD_CACHES) + 3)
    bad = BAD_BATCHES + [dict(past=None), dict(tables=None), dict(tokens=4)]
    assert [bounds(lib, b=batch(**kw)) for kw in bad] == [EINVAL] * len(bad)
    size = 10 * 2 * 2 * 64 * 2
    for at in (None, BOUNDS + 8, K, K + CACHE_BYTES - 16, V - size + 16, PAST, TABLES + 32):
        assert bounds(lib, at=at) == EINVAL, at
    assert bounds(lib, b=batch(starts=STARTS, tokens=3), at=STARTS) == EINVAL
    d = _abi.LaunchDims()
    assert lib.paella_page_bounds_dims(*refs(cache(), batch(sequences=5)), ctypes.byref(d)) == 0 and (d.grid, d.block) == (2, 256)   # a wave for both key heads of a small page
    assert lib.paella_page_bounds_dims(*refs(cache(size=64), batch(sequences=5)), ctypes.byref(d)) == 0 and (d.grid, d.block) == (3, 256)   # a wave per page and key head
    assert lib.paella_page_bounds_dims(*refs(cache(), batch()), None) == EINVAL and lib.paella_page_bounds_dims(None, ctypes.byref(batch()), ctypes.byref(d)) == EINVAL


# ------------------------------------------------------------------ plans

def select_plan(lib, c, b, heads=8, count=3, first=1, last=1):
    from paella_amd._abi_long import PageSelectPlan
    p = PageSelectPlan()
    return lib.paella_page_select_plan_make(*refs(c, b), heads, count, first, last, ctypes.byref(p)), p


def attend_plan(lib, c, b, heads=8, count=3, scale=0.0):
    from paella_amd._abi_long import PageAttentionPlan
    p = PageAttentionPlan()
    return lib.paella_page_attention_plan_make(*refs(c, b), heads, count, scale, ctypes.byref(p)), p


def weigh_plan(lib, c, b, heads=8, scale=0.0):
    from paella_amd._abi_long import KeyWeightsPlan
    p = KeyWeightsPlan()
    return lib.paella_key_weights_plan_make(*refs(c, b), heads, scale, ctypes.byref(p)), p


@pytest.mark.parametrize("make", [select_plan, attend_plan, weigh_plan], ids=["select", "attend", "weigh"])
def test_plans_refuse(lib, make):
    for kw in BAD_CACHES:
        assert make(lib, cache(**kw), batch())[0] == EINVAL, kw
    for kw in BAD_BATCHES:
        assert make(lib, cache(), batch(**kw))[0] == EINVAL, kw
    assert make(lib, cache(), batch(), heads=0)[0] == EINVAL and make(lib, cache(), batch(), heads=7)[0] == EINVAL
    assert make(lib, cache(dim=96), batch())[0] == ENOSUP and make(lib, cache(dim=512), batch())[0] == ENOSUP
    assert make(lib, cache(), batch(sequences=1 << 22), heads=8)[0] == ENOSUP                        # queries beyond 32-bit offsets
    assert make(lib, cache(), batch(sequences=1, max_pages=1 << 26))[0] == ENOSUP                     # a table of 2^30 tokens
    if make is not weigh_plan:
        for bad in (0, -1):
            assert make(lib, cache(), batch(), count=bad)[0] == EINVAL
    if make is select_plan:
        for first, last in ((-1, 1), (0, 0), (3, 1), (2 ** 31 - 1, 2 ** 31 - 1)):
            assert make(lib, cache(), batch(), first=first, last=last)[0] == EINVAL
    else:
        for scale in (-1.0, math.nan, math.inf):
            assert make(lib, cache(), batch(), scale=scale)[0] == EINVAL
        assert make(lib, cache(), batch())[1].scale == 0.125 and make(lib, cache(), batch(), scale=0.5)[1].scale == 0.5


def test_what_plans_plan(lib):
    from paella_amd import _abi
    # few rows of few pages: one launch; more workgroups than two to a compute unit, or more pages than four waves hold: two
    assert select_plan(lib, cache(), batch())[1].stages == 1
    rc, p = select_plan(lib, cache(heads=8, dim=128, size=64, pages=9000), batch(sequences=32, max_pages=1025), 32, 64, 1, 2)
    assert rc == 0 and p.stages == 1 and p.workspace_bytes >= 3 * 32 * 8 * 1025 * 4
    assert select_plan(lib, cache(heads=8, dim=128, size=64, pages=9000), batch(sequences=80, max_pages=1025), 32, 64, 1, 2)[1].stages == 2
    assert select_plan(lib, cache(pages=9000), batch(sequences=1, max_pages=5000))[1].stages == 2
    # lists that fill the device are not shared out; one of many pages is, and a wide one's parts are joined by a launch of their own
    assert attend_plan(lib, cache(heads=8, dim=128, size=64), batch(sequences=64), 32, 64)[1].workspace_bytes == 0
    rc, p = attend_plan(lib, cache(heads=1, dim=128, size=64), batch(sequences=1, max_pages=64), 4, 64)
    assert rc == 0 and (p.splits, p.stages) == (16, 1) and p.dims.grid == 16
    assert attend_plan(lib, cache(heads=1, dim=128, size=64), batch(sequences=1, max_pages=4), 4, 64)[1].splits == 1   # (there are no more pages than that)
    rc, p = attend_plan(lib, cache(heads=1, dim=256, size=64), batch(sequences=1, max_pages=64), 16, 64)
    assert rc == 0 and p.stages == 2
    join = _abi.LaunchDims()
    assert lib.paella_page_attention_dims(ctypes.byref(p), 1, ctypes.byref(join)) == 0 and join.grid >= 1
    # scores are kept for 16 rows at most
    few, many = weigh_plan(lib, cache(), batch(max_new=4), 8)[1], weigh_plan(lib, cache(), batch(max_new=5), 8)[1]
    assert few.workspace_bytes >= 3 * 2 * 16 * 64 * 4 > many.workspace_bytes and few.stages == many.stages == 2
    for n in (1, 16, 33, 500):   # every plan that is made has kernels
        for sequences in (1, 40):
            for dtype in (0, 1, 2):
                for dim in (64, 128, 256):
                    for prefix in (0, 1000):
                        args = lib, cache(dtype=dtype, dim=dim), batch(sequences=sequences, max_new=n, prefix=prefix)
                        assert select_plan(*args)[0] == attend_plan(*args)[0] == weigh_plan(*args)[0] == 0


# ------------------------------------------------------------------ launches

class Call:
    """One planned operator's launch with every operand replaceable."""

    def __init__(self, lib, name, make, operands, width=4, **kw):
        self.lib, self.name, self.operands, self.width = lib, "paella_%s_launch" % name, operands, width
        self.c, self.b = cache(), batch(prefix=40, max_pages=width)
        rc, self.plan = make(lib, self.c, self.b, **kw)
        assert rc == 0
        self.fresh = lambda: make(lib, self.c, self.b, **kw)[1]

    def __call__(self, stage=None, plan=None, c=None, b=None, stride=512, space=SPACE, **given):
        operands = dict(self.operands, **given)
        args = [ctypes.byref(plan or self.plan)] + ([] if stage is None else [stage]) + refs(c or self.c, b or self.b) + [operands.pop("q"), stride] + list(operands.values()) + [space, None, 0, None]
        return getattr(self.lib, self.name + ("" if stage is None else "_stage"))(*args)


CALLS = {
    "select": lambda lib: Call(lib, "page_select", select_plan, dict(q=Q, bounds=BOUNDS, pages=PAGES)),
    "attend": lambda lib: Call(lib, "page_attention", attend_plan, dict(q=Q, pages=PAGES, out=OUT), width=100, count=100),
    "weigh": lambda lib: Call(lib, "key_weights", weigh_plan, dict(q=Q, weights=WEIGHTS)),
}


@pytest.mark.parametrize("which", CALLS)
def test_launches_refuse(lib, which):
    call = CALLS[which](lib)
    need = call.plan.workspace_bytes
    assert need
    for name, at in call.operands.items():
        assert call(**{name: None}) == EINVAL, name
        assert call(**{name: at + (2 if name == "pages" else 8)}) == EINVAL, name
    assert call(space=None) == EINVAL and call(space=SPACE + 8) == EINVAL and call(stride=504) == EINVAL and call(stride=516) == EINVAL
    assert call(stage=call.plan.stages) == EINVAL and call(stage=-1) == EINVAL
    for kw in (dict(dtype=2), dict(heads=4), dict(size=8), dict(dim=128), dict(k=None), dict(v=V + 8)):
        assert call(c=cache(**kw)) == EINVAL, kw
    for kw in (dict(prefix=41), dict(prefix=0), dict(sequences=4), dict(max_pages=5), dict(past=None), dict(tables=None), dict(max_new=2, tokens=3)):
        assert call(b=batch(**{"prefix": 40, "max_pages": call.width, **kw})) == EINVAL, kw
    broken = batch(prefix=40, max_pages=call.width)
    broken.prefix_table = None
    assert call(b=broken) == EINVAL
    fields = [("splits", 0), ("heads", 7), ("dtype", 5), ("head_dim", 96), ("page_size", 12), ("sequences", 0), ("max_pages", 0), ("tokens", 0)]
    fields += dict(select=[("count", 0), ("first", -1), ("last", 0), ("first", 5)], attend=[("count", 0), ("splits", 65), ("scale", -1.0)], weigh=[("own_splits", 0), ("splits", 65), ("scale", math.nan)])[which]
    for field, value in fields:
        plan = call.fresh()
        setattr(plan, field, value)
        assert call(plan=plan) == EINVAL, field


@pytest.mark.parametrize("which", CALLS)
def test_outputs_over_what_is_read(lib, which):
    """Outputs and the workspace over anything that the call reads, or over one another."""
    call = CALLS[which](lib)
    need = call.plan.workspace_bytes
    result = list(call.operands)[-1]
    sizes = {"q": 3 * 512 * 2, "bounds": 10 * 2 * 2 * 64 * 2, "pages": 3 * 2 * call.plan.count * 4 if which != "weigh" else 0, "out": 3 * 512 * 2, "weights": 3 * 2 * 16 * call.width * 4}
    inputs = [(call.operands[n], sizes[n]) for n in call.operands if n != result] + [(PAST, 12), (TABLES, 12 * call.width), (PREFIX, 12)]
    if which != "select":
        inputs += [(K, CACHE_BYTES), (V, CACHE_BYTES)]
    for at, size in inputs:
        for name, extent in ((result, sizes[result]), ("space", need)):
            last = at + (size - 1) // 16 * 16   # the last boundary within it
            for over in (at, last, at - (extent + 15) // 16 * 16 + 16):
                assert call(**{name: over}) == EINVAL, (name, at // AT)
    last = call.operands[result] + (sizes[result] - 1) // 16 * 16
    assert call(space=call.operands[result]) == EINVAL and call(space=last) == EINVAL and call(space=call.operands[result] - (need + 15) // 16 * 16 + 16) == EINVAL
    assert call(stride=1 << 20, space=Q + (4 << 20) + 256) == EINVAL                       # over the last of rows that lie far apart
    ragged = batch(prefix=40, starts=STARTS, max_pages=call.width)
    assert call(b=ragged, space=STARTS) == EINVAL


# ------------------------------------------------------------------ eviction

def evict(lib, c=None, sequences=3, max_pages=4, keep=20, first=2, recent=5, weights=WEIGHTS, past=PAST, tables=TABLES, kept=KEPT, past_out=LENGTHS, stage=None):
    from paella_amd._abi_long import KvEvictDesc
    d = KvEvictDesc(sequences, max_pages, keep, first, recent)
    args = [ctypes.byref(c or cache()), weights, past, tables, kept, past_out, None, 0, None]
    if stage is None:
        return lib.paella_kv_evict_launch(ctypes.byref(d), *args)
    return lib.paella_kv_evict_launch_stage(ctypes.byref(d), stage, *args)


def test_eviction_refuses(lib):
    from paella_amd import _abi
    from paella_amd._abi_long import KvEvictDesc
    assert [evict(lib, c=cache(**kw)) for kw in BAD_CACHES + [dict(k=None), dict(v=None), dict(v=V + 8)]] == [EINVAL] * (len(BAD_CACHES) + 3)
    for kw in (dict(sequences=0), dict(max_pages=0), dict(keep=0), dict(first=-1), dict(recent=-1), dict(first=16), dict(first=2 ** 31 - 1, recent=2 ** 31 - 1), dict(stage=-1), dict(stage=2)):
        assert evict(lib, **kw) == EINVAL, kw
    assert evict(lib, max_pages=1 << 26) == ENOSUP and evict(lib, sequences=1 << 30, max_pages=1) == ENOSUP
    for name in ("weights", "past", "tables", "kept", "past_out"):
        assert evict(lib, **{name: None}) == EINVAL, name
    sizes = dict(weights=3 * 2 * 64 * 4, past=12, tables=48, kept=3 * 2 * 20 * 4, past_out=12)
    at = dict(weights=WEIGHTS, past=PAST, tables=TABLES, kept=KEPT, past_out=LENGTHS)
    for name in ("weights", "kept", "past_out"):
        for other in sizes:
            if other != name:
                for over in (at[other] + sizes[other] - 4, at[other] - sizes[name] + 4) + (() if (name, other) == ("past_out", "past") else (at[other],)):
                    assert evict(lib, **{name: over}) == EINVAL, (name, other)
        for base in (K, V):
            assert evict(lib, **{name: base}) == EINVAL and evict(lib, **{name: base + CACHE_BYTES - 4}) == EINVAL
    d, good = _abi.LaunchDims(), KvEvictDesc(3, 4, 20, 2, 5)
    assert lib.paella_kv_evict_dims(*refs(good, cache()), 0, ctypes.byref(d)) == 0 and d.grid == 6
    assert lib.paella_kv_evict_dims(*refs(good, cache()), 2, ctypes.byref(d)) == EINVAL and lib.paella_kv_evict_dims(*refs(good, cache()), 0, None) == EINVAL


# ------------------------------------------------------------------ the front-end

def test_the_front_end_refuses_what_does_not_fit(monkeypatch):
    """Shapes, types and devices, with the launches replaced."""
    from paella_amd import decode, long_cache
    monkeypatch.setattr(decode, "_current_device", lambda: -1)   # what tensors of the CPU say
    monkeypatch.setattr(long_cache, "_stream", lambda s: 0)
    ints = lambda *shape: torch.zeros(shape, dtype=torch.int32)  # noqa: E731
    c = decode.KVCache(torch.zeros((4, 2, 16, 64)), torch.zeros((4, 2, 16, 64)))
    b = decode.KVBatch(ints(3), ints(3, 2))
    launched = []
    note = lambda *a: launched.append(a) or 0  # noqa: E731
    monkeypatch.setattr(long_cache, "_library", lambda: types.SimpleNamespace(paella_page_bounds_launch=note))
    select, attend, weigh = long_cache.PageSelect(4, c, b, 2), long_cache.PageAttention(4, c, b, 2), long_cache.KeyWeights(4, c, b)
    evict = long_cache.Evict(c, 3, 2, keep=8)
    for planned in (select, attend, weigh):
        planned._whole = note
        monkeypatch.setattr(planned, "_issue", lambda cache, batch, operands, *a, planned=planned: launched.append(operands))
    evict.lib = types.SimpleNamespace(paella_kv_evict_launch=note, paella_kv_evict_launch_stage=note)
    low, sums, q, pages = long_cache.new_bounds(c), long_cache.new_weights(c, b), torch.zeros((3, 4, 64)), ints(3, 2, 2)
    assert low.shape == (4, 2, 2, 64) and sums.shape == (3, 2, 32) and sums.dtype is torch.float32

    def calls(c=c, b=b, low=low, sums=sums, q=q, pages=pages, past=b.past, tables=b.tables):
        return dict(bounds=lambda: long_cache.page_bounds(c, low, b), select=lambda: select(q, low, c, b), attend=lambda: attend(q, c, b, pages), weigh=lambda: weigh(q, c, b, sums),
                    evict=lambda: evict(c, sums, past, tables))

    for call in calls().values():
        call()
    assert len(launched) == 5
    elsewhere = lambda t: types.SimpleNamespace(get_device=lambda: 1, dtype=t.dtype, shape=t.shape)  # noqa: E731
    bad = [(dict(low=low[:3]), "bounds select"), (dict(low=low.half()), "bounds select"), (dict(low=low.transpose(2, 3).contiguous().transpose(2, 3)), "bounds select"),
           (dict(q=q[:2]), "select attend weigh"), (dict(q=q.half()), "select attend weigh"), (dict(q=q[:, :2]), "select attend weigh"), (dict(sums=sums[:2]), "weigh evict"),
           (dict(sums=sums.double()), "weigh evict"), (dict(sums=torch.zeros((3, 2, 64))[..., ::2]), "weigh evict"), (dict(pages=pages.long()), "attend"), (dict(pages=pages[:, :1]), "attend"),
           (dict(past=ints(2)), "evict"), (dict(tables=ints(3, 3)), "evict"), (dict(tables=ints(3, 2).long()), "evict"), (dict(low=elsewhere(low)), "bounds select"),
           (dict(sums=elsewhere(sums)), "weigh evict"), (dict(q=elsewhere(q)), "select attend weigh"), (dict(pages=elsewhere(pages)), "attend"), (dict(past=elsewhere(b.past)), "evict")]
    for kw, names in bad:
        for name in names.split():
            with pytest.raises(AssertionError):
                calls(**kw)[name]()
    for planned, args in ((select, (q, low, c, b)), ):
        with pytest.raises(AssertionError):
            planned(*args, stage=0)
    with pytest.raises(AssertionError):
        evict(c, sums, b.past, b.tables, stage=0)
    assert len(launched) == 5
    moved = decode.KVBatch(ints(3), ints(3, 2))
    moved.past = types.SimpleNamespace(get_device=lambda: 1, shape=(3,))
    for name in ("bounds", "select", "attend", "weigh"):   # a batch is made once and used for many calls
        with pytest.raises(AssertionError):
            calls(b=moved)[name]()
    assert len(launched) == 5
