"""The C-ABI of the decoding step's operators without a device: every declared symbol, what the plans plan, and what each entry point refuses before anything is launched."""
import ctypes
import os
import re

import pytest
import torch

import _decode_ref as ref

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
EINVAL, ENOSUP = -1, -2
AT = 1 << 20   # an address on a boundary of every kind; none of the calls here gets as far as using it


@pytest.fixture(scope="module")
def lib():
    from paella_amd import _abi
    return _abi.ops()


def cache(dtype=1, pages=10, heads=2, size=16, dim=64, k=AT, v=AT + (1 << 30)):
    from paella_amd._abi_decode import KvCache
    return KvCache(k, v, dtype, pages, heads, size, dim)


def batch(sequences=3, max_new=1, tokens=None, max_pages=4, prefix=0, starts=None, past=AT, tables=AT, prefix_table=None):
    from paella_amd._abi_decode import KvBatch
    return KvBatch(sequences, max_new, sequences * max_new if tokens is None else tokens, max_pages, prefix, starts, past, tables, prefix_table)


def test_header_and_table_and_library_agree(lib):
    from paella_amd import _abi_decode
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "paella_decode.h")).read(), flags=re.S)
    declared = sorted(set(re.findall(r"\b(paella_[a-z0-9_]+)\s*\(", text)))
    assert declared == sorted(_abi_decode.DECODE_SYMBOLS) and all(hasattr(lib, n) for n in declared)


def append(lib, c=None, b=None, heads=4, rotary=64, interleaved=0, eps=1e-6, strides=(512, 512, 512), q=AT, k=AT, v=AT, freq=AT, out=2 * AT):
    from paella_amd._abi_decode import KvAppendDesc
    c, b = c or cache(), b or batch()
    d = KvAppendDesc(heads, rotary, interleaved, eps, *strides)
    return lib.paella_kv_append_launch(ctypes.byref(d), ctypes.byref(c), ctypes.byref(b), q, k, v, None, None, freq, out, None, 0, None)


def test_append_refuses(lib):
    bad_caches = [cache(dtype=3), cache(dtype=-1), cache(pages=0), cache(heads=0), cache(size=12), cache(size=0), cache(dim=60), cache(dim=520), cache(k=None), cache(v=None),
                  cache(k=AT + 8), cache(heads=1 << 12, size=1 << 12, dim=64)]
    assert [append(lib, c=c) for c in bad_caches] == [EINVAL] * len(bad_caches)
    bad_batches = [batch(sequences=0), batch(max_new=0), batch(tokens=0), batch(max_pages=0), batch(prefix=-1), batch(prefix=1 << 30), batch(past=None), batch(tables=None),
                   batch(tokens=4), batch(sequences=1 << 16, max_new=1 << 16, tokens=1 << 20, starts=AT), batch(sequences=1 << 25, tokens=1 << 25)]
    assert [append(lib, b=b) for b in bad_batches] == [EINVAL] * len(bad_batches)
    assert append(lib, heads=-1) == EINVAL and append(lib, heads=0) == EINVAL          # no heads, but queries
    assert append(lib, q=None) == EINVAL and append(lib, out=None) == EINVAL and append(lib, k=None) == EINVAL and append(lib, v=None) == EINVAL
    assert append(lib, rotary=24) == EINVAL and append(lib, rotary=80) == EINVAL and append(lib, rotary=-16) == EINVAL and append(lib, freq=None) == EINVAL
    assert append(lib, eps=-1.0) == EINVAL and append(lib, eps=float("nan")) == EINVAL
    assert append(lib, strides=(512, 64, 512)) == EINVAL and append(lib, strides=(128, 512, 512)) == EINVAL and append(lib, strides=(512, 516, 512)) == EINVAL
    assert append(lib, q=AT + 4) == EINVAL and append(lib, out=AT) == EINVAL            # misaligned; over rows that do not lie side by side
    assert append(lib, out=AT + 512, strides=(256, 512, 512)) == EINVAL                 # one row further on
    from paella_amd._abi_decode import KvAppendDesc
    from paella_amd import _abi
    good, d = KvAppendDesc(4, 64, 0, 1e-6, 512, 512, 512), _abi.LaunchDims()
    assert lib.paella_kv_append_dims(ctypes.byref(good), ctypes.byref(cache()), ctypes.byref(batch(sequences=5)), ctypes.byref(d)) == 0 and (d.grid, d.block) == (5, 256)
    assert lib.paella_kv_append_dims(ctypes.byref(good), ctypes.byref(cache()), ctypes.byref(batch()), None) == EINVAL
    assert lib.paella_kv_append_dims(None, ctypes.byref(cache()), ctypes.byref(batch()), ctypes.byref(d)) == EINVAL


def plan(lib, c, b, heads, scale=0.0):
    from paella_amd._abi_decode import PrefixAttentionPlan
    p = PrefixAttentionPlan()
    return lib.paella_prefix_attention_plan_make(ctypes.byref(c), ctypes.byref(b), heads, scale, ctypes.byref(p)), p


def test_attention_plans(lib):
    from paella_amd import _abi
    # few rows: 16 of them, one part of a short own context, no prefix: no workspace
    rc, p = plan(lib, cache(), batch(), 8)
    assert rc == 0 and (p.prefix_rows, p.own_rows, p.prefix_splits, p.own_splits, p.stages, p.workspace_bytes) == (16, 16, 0, 1, 1, 0)
    assert p.dims.grid == 3 * 2 and p.scale == 0.125
    # a long own context of one sequence is shared out; a prefix over many rows takes 128 of them and a launch that joins
    assert plan(lib, cache(pages=5000), batch(sequences=1, max_pages=4096), 8)[1].own_splits == 64
    rc, p = plan(lib, cache(heads=8, dim=128, size=64, pages=3000), batch(sequences=64, max_pages=63, prefix=65536, prefix_table=AT), 32)
    assert rc == 0 and (p.prefix_rows, p.own_rows, p.stages) == (128, 16, 2) and p.prefix_splits >= 16
    items = [2 * 8 * p.prefix_splits, 64 * 8 * p.own_splits]
    assert p.dims.grid == sum(items)
    parts, rows = p.prefix_splits + p.own_splits, 64 * 32
    assert p.workspace_bytes == 8 * 1024 + parts * rows * 8 + parts * rows * 128 * 4
    join = _abi.LaunchDims()
    assert lib.paella_prefix_attention_dims(ctypes.byref(p), 1, ctypes.byref(join)) == 0 and join.grid == rows // 2
    # rows of a key head beyond 16 and 64 over many keys; head size 256 and wide fp32 heads have fewer forms
    for dtype, dim, rows, prefix, want in [(1, 64, 17, 40000, 64), (1, 64, 65, 40000, 128), (1, 64, 65, 1000, 16), (0, 64, 65, 40000, 128), (0, 128, 65, 40000, 64),
                                           (0, 128, 32, 1000, 16), (2, 256, 17, 100, 64), (0, 256, 65, 100, 64), (1, 256, 16, 40000, 16)]:
        p = plan(lib, cache(dtype=dtype, dim=dim, heads=1), batch(sequences=rows, prefix=prefix, prefix_table=AT), 1)[1]
        assert (p.prefix_rows, p.own_rows) == (want, 16), (dtype, dim, rows)
    for rows, dim, want in [(32, 128, 16), (33, 128, 64), (65, 128, 128), (17, 256, 64)]:   # of one sequence
        assert plan(lib, cache(dtype=1, dim=dim, heads=1), batch(max_new=rows), 1)[1].own_rows == want
    for n in (1, 16, 33, 70, 500):   # every planned pair of forms has a kernel
        for sequences in (1, 40):
            for dtype in (0, 1, 2):
                for dim in (64, 128, 256):
                    for prefix in (0, 1000):
                        assert plan(lib, cache(dtype=dtype, dim=dim), batch(sequences=sequences, max_new=n, prefix=prefix, prefix_table=AT), 4)[0] == 0
    assert plan(lib, cache(dim=96), batch(), 8)[0] == ENOSUP and plan(lib, cache(dim=512), batch(), 8)[0] == ENOSUP
    assert plan(lib, cache(), batch(sequences=1 << 22), 8)[0] == ENOSUP                                       # outputs beyond 32-bit offsets
    for c, b, heads, scale in [(cache(), batch(), 3, 0.0), (cache(), batch(), 0, 0.0), (cache(), batch(), 8, -1.0), (cache(), batch(), 8, float("nan")),
                               (cache(), batch(), 8, float("inf")), (cache(size=4), batch(), 8, 0.0), (cache(), batch(tokens=0), 8, 0.0)]:
        assert plan(lib, c, b, heads, scale)[0] == EINVAL


def test_attention_launch_refuses(lib):
    from paella_amd import _abi
    c, b = cache(), batch(prefix=100, prefix_table=AT)
    rc, p = plan(lib, c, b, 8)
    assert rc == 0 and p.workspace_bytes and p.stages == 1

    def launch(c=c, b=b, p=p, q=AT, stride=512, out=4 * AT, workspace=8 * AT, stage=None):
        args = [ctypes.byref(c), ctypes.byref(b), q, stride, out, workspace, None, 0, None]
        if stage is None:
            return lib.paella_prefix_attention_launch(ctypes.byref(p), *args)
        return lib.paella_prefix_attention_launch_stage(ctypes.byref(p), stage, *args)

    assert launch(q=None) == EINVAL and launch(out=None) == EINVAL and launch(workspace=None) == EINVAL and launch(workspace=8 * AT + 4) == EINVAL
    assert launch(q=AT + 8) == EINVAL and launch(stride=504) == EINVAL and launch(stride=516) == EINVAL
    assert launch(out=AT) == EINVAL and launch(out=AT + 2048) == EINVAL                   # over the queries
    assert launch(stage=1) == EINVAL and launch(stage=-1) == EINVAL
    for other in (cache(dtype=2), cache(heads=4), cache(size=8), cache(dim=128), cache(k=None)):
        assert launch(c=other) == EINVAL
    for other in (batch(prefix=101, prefix_table=AT), batch(prefix=100), batch(sequences=4, prefix=100, prefix_table=AT), batch(max_pages=5, prefix=100, prefix_table=AT),
                  batch(prefix=100, prefix_table=AT, past=None), batch(prefix=100, prefix_table=AT, max_new=2, tokens=3)):
        assert launch(b=other) == EINVAL
    for field, value in [("own_splits", 0), ("own_splits", 65), ("prefix_splits", 0), ("own_rows", 48), ("prefix_rows", 128), ("scale", -1.0), ("heads", 7), ("dtype", 5)]:
        broken = plan(lib, c, b, 8)[1]
        setattr(broken, field, value)
        if field == "prefix_rows":
            broken.own_rows = 64   # no such pair
        assert launch(p=broken) == EINVAL, field
    d = _abi.LaunchDims()
    assert lib.paella_prefix_attention_dims(ctypes.byref(p), 1, ctypes.byref(d)) == EINVAL and lib.paella_prefix_attention_dims(ctypes.byref(p), 0, None) == EINVAL


def select_plan(lib, *args):
    from paella_amd._abi_decode import BeamSelectPlan
    p = BeamSelectPlan()
    return lib.paella_beam_select_plan_make(*args, ctypes.byref(p)), p


def test_selection_plans_and_refusals(lib):
    rc, p = select_plan(lib, 0, 1, 4, 32000, 4)
    assert rc == 0 and (p.values, p.splits, p.dims.grid) == (8, 16, 64)
    rc, p = select_plan(lib, 1, 32, 4, 131072, 8)
    assert rc == 0 and (p.values, p.splits, p.dims.grid) == (32, 16, 2048)
    assert select_plan(lib, 0, 1, 32, 262144, 64)[1].splits == 32 and select_plan(lib, 0, 1, 16, 524288, 64)[0] == 0
    assert [select_plan(lib, *a)[0] for a in [(0, 1, 33, 10, 1), (0, 1, 4, 524289, 1), (0, 1, 4, 10, 65), (0, 1, 32, 524288, 1)]] == [ENOSUP] * 4
    assert [select_plan(lib, *a)[0] for a in [(3, 1, 4, 10, 1), (0, 0, 4, 10, 1), (0, 1, 0, 10, 1), (0, 1, 4, 0, 1), (0, 1, 4, 10, 0)]] == [EINVAL] * 5
    rc, p = select_plan(lib, 1, 2, 4, 1000, 4)

    def launch(p=p, logits=AT, stride=1000, scores=AT, finished=None, pad=0, scores_out=AT, parents=AT, tokens=AT, workspace=AT):
        return lib.paella_beam_select_launch(ctypes.byref(p), logits, stride, scores, finished, pad, scores_out, parents, tokens, workspace, None, 0, None)

    for name in ("logits", "scores", "scores_out", "parents", "tokens", "workspace"):
        assert launch(**{name: None}) == EINVAL, name
    assert launch(stride=999) == EINVAL and launch(logits=AT + 1) == EINVAL and launch(workspace=AT + 4) == EINVAL
    assert launch(finished=AT, pad=-1) == EINVAL and launch(finished=AT, pad=1000) == EINVAL
    for field, value in [("splits", 2), ("values", 16), ("beams", 40), ("count", 0), ("dtype", 4), ("vocab", 0)]:
        broken = select_plan(lib, 1, 2, 4, 1000, 4)[1]
        setattr(broken, field, value)
        assert launch(p=broken, stride=2000) == EINVAL, field


def test_reorder_refuses(lib):
    from paella_amd import _abi
    from paella_amd._abi_decode import BeamReorderDesc

    def launch(shape=(2, 3, 3, 5), c=None, parents=AT, past=2 * AT, tables=3 * AT, spare=4 * AT, out=5 * AT, past_out=6 * AT):
        return lib.paella_beam_reorder_launch(ctypes.byref(BeamReorderDesc(*shape)), ctypes.byref(c or cache()), parents, past, tables, spare, out, past_out, None, 0, None)

    for shape in [(0, 3, 3, 5), (2, 0, 3, 5), (2, 3, 0, 5), (2, 3, 3, 0), (1 << 24, 3, 3, 5)]:
        assert launch(shape=shape) == EINVAL
    for name in ("parents", "past", "tables", "spare", "out", "past_out"):
        assert launch(**{name: None}) == EINVAL, name
    assert launch(out=3 * AT) == EINVAL and launch(out=3 * AT + 4) == EINVAL and launch(past_out=2 * AT) == EINVAL and launch(past_out=AT) == EINVAL
    assert launch(c=cache(v=None)) == EINVAL and launch(c=cache(size=20)) == EINVAL
    d = _abi.LaunchDims()
    assert lib.paella_beam_reorder_dims(ctypes.byref(BeamReorderDesc(2, 3, 4, 5)), ctypes.byref(cache()), ctypes.byref(d)) == 0 and d.grid == 2 * 4 * 2
    assert lib.paella_beam_reorder_dims(ctypes.byref(BeamReorderDesc(2, 3, 4, 5)), ctypes.byref(cache()), None) == EINVAL


def test_the_definitions_used_as_reference():
    """_decode_ref against torch where torch has the operator, and against hand-worked cases."""
    g = torch.Generator()
    g.manual_seed(1)
    k, v = torch.randn((4, 2, 8, 64), generator=g), torch.randn((4, 2, 8, 64), generator=g)
    q = torch.randn((3, 4, 64), generator=g)
    tables, prefix = torch.tensor([[2, 0]]), torch.tensor([1, 3])
    rows = ref.owners(None, [7], 3, 3)
    assert rows == [(0, 7), (0, 8), (0, 9)] and ref.owners([0, 2, 2], [1, 5], 2, 3) == [(0, 1), (0, 2), None]
    out = ref.attention(q, k, v, rows, tables, prefix, 11, 0.125)[0]
    line = lambda t: torch.cat((t[1], t[3, :, :3], t[2], t[0, :, :2]), 1)  # noqa: E731  prefix 11, own 10
    keys, values = line(k).double().repeat_interleave(2, 0), line(v).double().repeat_interleave(2, 0)
    mask = torch.arange(21)[None] <= 11 + 7 + torch.arange(3)[:, None]
    want = torch.nn.functional.scaled_dot_product_attention(q.double().transpose(0, 1), keys, values, attn_mask=mask, scale=0.125).transpose(0, 1)
    assert (out - want).abs().max() < 1e-12
    x = torch.tensor([[3.0, 4.0, 1.0, 2.0]]).double()
    turned = ref.norm_rotate(x, None, 0.0, [0.5], False, 1)
    assert torch.allclose(turned[0, :2], torch.tensor([3 * 0.8775825618903728 - 4 * 0.479425538604203, 4 * 0.8775825618903728 + 3 * 0.479425538604203]).double())
    assert ref.select(torch.tensor([[[1.0, 1.0], [1.0, 1.0]]]), torch.tensor([[0.0, 0.0]]), None, 0, 3)[0] == [(pytest.approx(-0.6931471805599453), 0, 0),
                                                                                                   (pytest.approx(-0.6931471805599453), 0, 1),
                                                                                                   (pytest.approx(-0.6931471805599453), 1, 0)]
