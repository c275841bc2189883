"""Outputs of the decoding step's operators that lie over what the same call reads, or over one another: refused before anything is launched."""
import ctypes

import pytest

EINVAL = -1
AT = 1 << 32


@pytest.fixture(scope="module")
def lib():
    from paella_amd import _abi
    return _abi.ops()


def cache():
    from paella_amd._abi_decode import KvCache
    return KvCache(AT, 2 * AT, 1, 10, 2, 16, 64)      # 40960 bytes each


def batch(tokens=3):
    from paella_amd._abi_decode import KvBatch
    return KvBatch(tokens, 1, tokens, 4, 0, None, 3 * AT, 4 * AT, None)


CACHE_BYTES = 10 * 2 * 16 * 64 * 2


def test_append_over_its_own_inputs(lib):
    from paella_amd._abi_decode import KvAppendDesc

    def append(q=5 * AT, k=6 * AT, v=7 * AT, out=8 * AT, strides=(256, 128, 128), heads=4):
        d = KvAppendDesc(heads, 0, 0, 1e-6, *strides)
        return lib.paella_kv_append_launch(ctypes.byref(d), ctypes.byref(cache()), ctypes.byref(batch()), q if heads else None, k, v, None, None, None, out if heads else None, None, 0, None)

    k_bytes, out_bytes = 3 * 128 * 2, 3 * 256 * 2
    for base in (6 * AT, 7 * AT):                      # queries' outputs over keys or values that other tokens' workgroups still read
        assert append(out=base) == EINVAL and append(out=base + k_bytes - 16) == EINVAL and append(out=base - out_bytes + 16) == EINVAL
    for base in (AT, 2 * AT):                          # and over the cache
        assert append(out=base) == EINVAL and append(out=base + CACHE_BYTES - 16) == EINVAL
    for inside in (0, 1, 2):                            # keys' rows far apart: over any of them
        assert append(strides=(256, 1 << 20, 128), out=6 * AT + inside * (2 << 20) + 240) == EINVAL
        assert append(strides=(256, 1 << 20, 128), out=6 * AT + inside * (2 << 20) - out_bytes + 16) == EINVAL
    assert append(q=5 * AT, k=5 * AT + 512, v=5 * AT + 768, out=5 * AT, strides=(512, 512, 512)) == EINVAL   # a packed projection, its queries not side by side


def test_attention_over_the_cache_or_its_workspace(lib):
    from paella_amd._abi_decode import KvBatch, PrefixAttentionPlan
    b = KvBatch(3, 1, 3, 4, 100, None, 3 * AT, 4 * AT, 9 * AT)
    p = PrefixAttentionPlan()
    assert lib.paella_prefix_attention_plan_make(ctypes.byref(cache()), ctypes.byref(b), 8, 0.0, ctypes.byref(p)) == 0 and p.workspace_bytes

    def attend(q=5 * AT, out=6 * AT, workspace=7 * AT):
        return lib.paella_prefix_attention_launch(ctypes.byref(p), ctypes.byref(cache()), ctypes.byref(b), q, 512, out, workspace, None, 0, None)

    for base in (AT, 2 * AT):
        assert attend(out=base) == EINVAL and attend(out=base + CACHE_BYTES - 16) == EINVAL and attend(out=base - 16) == EINVAL
        assert attend(workspace=base) == EINVAL and attend(workspace=base - p.workspace_bytes + 16) == EINVAL
    assert attend(workspace=5 * AT) == EINVAL and attend(workspace=6 * AT + 16) == EINVAL and attend(out=7 * AT + p.workspace_bytes - 16) == EINVAL


def test_selection_over_its_own_inputs(lib):
    from paella_amd._abi_decode import BeamSelectPlan

    def select(count=4, groups=2, logits=AT, scores=2 * AT, finished=3 * AT, values=4 * AT, parents=5 * AT, tokens=6 * AT, workspace=7 * AT):
        p = BeamSelectPlan()
        assert lib.paella_beam_select_plan_make(0, groups, 4, 1000, count, ctypes.byref(p)) == 0
        return lib.paella_beam_select_launch(ctypes.byref(p), logits, 1000, scores, finished, 0, values, parents, tokens, workspace, None, 0, None)

    for name in ("values", "parents", "tokens"):
        for at in (AT, AT + 2 * 4 * 4000 - 4, 2 * AT + 4, 3 * AT, 3 * AT + 4, 7 * AT):
            assert select(**{name: at}) == EINVAL, (name, at)
    assert select(parents=2 * AT) == EINVAL and select(tokens=2 * AT) == EINVAL
    # scores of the next step in place of this one's: only where every group's are its own
    assert select(count=8, values=2 * AT) == EINVAL and select(count=3, values=2 * AT) == EINVAL
    assert select(values=5 * AT) == EINVAL and select(tokens=5 * AT + 16) == EINVAL and select(tokens=4 * AT + 4) == EINVAL
    assert select(workspace=AT) == EINVAL and select(workspace=2 * AT) == EINVAL


def test_reordering_over_its_own_inputs(lib):
    from paella_amd._abi_decode import BeamReorderDesc

    def reorder(parents=3 * AT, past=4 * AT, tables=5 * AT, spare=6 * AT, out=7 * AT, past_out=8 * AT):
        return lib.paella_beam_reorder_launch(ctypes.byref(BeamReorderDesc(2, 3, 4, 5)), ctypes.byref(cache()), parents, past, tables, spare, out, past_out, None, 0, None)

    for name in ("out", "past_out"):
        for base in (AT, 2 * AT, 3 * AT, 4 * AT, 5 * AT, 6 * AT):
            assert reorder(**{name: base}) == EINVAL and reorder(**{name: base + 4}) == EINVAL, (name, base)
    assert reorder(out=8 * AT) == EINVAL and reorder(past_out=7 * AT + 4 * 8 * 5 - 4) == EINVAL
