"""Plans of the decoding step's operators over batches and plans that the ordinary ones do not reach, without a device."""
import ctypes

import pytest

EINVAL, ENOSUP = -1, -2
AT = 1 << 20


@pytest.fixture(scope="module")
def lib():
    from paella_amd import _abi
    return _abi.ops()


def attention_plan(lib, dtype, heads, kv_heads, dim, size, sequences, max_new, tokens, max_pages, prefix):
    from paella_amd._abi_decode import KvBatch, KvCache, PrefixAttentionPlan
    p = PrefixAttentionPlan()
    c = KvCache(AT, AT + (1 << 40), dtype, 1000, kv_heads, size, dim)
    b = KvBatch(sequences, max_new, tokens, max_pages, prefix, AT, AT, AT, AT if prefix else None)
    return lib.paella_prefix_attention_plan_make(ctypes.byref(c), ctypes.byref(b), heads, 0.0, ctypes.byref(p)), p


def test_a_ragged_batch_with_room_for_more_new_tokens_than_it_has_is_planned(lib):
    """max_new bounds what a sequence may have: a batch of few rows with a large bound has a kernel like any other."""
    rc, p = attention_plan(lib, 1, 32, 8, 128, 64, 4, 32, 14, 20, 5000)
    assert rc == 0 and (p.prefix_rows, p.own_rows) == (64, 64)
    for dtype in (0, 1, 2):
        for dim in (64, 128, 256):
            for per_kv in (1, 4, 8):
                for sequences in (1, 4):
                    for max_new in (1, 7, 17, 33, 64, 200):
                        for tokens in {1, max(1, max_new // 3), max_new, (max_new * sequences + max_new) // 2, max_new * sequences}:
                            for prefix in (0, 9, 300, 5000):
                                rc, p = attention_plan(lib, dtype, 2 * per_kv, 2, dim, 16, sequences, max_new, tokens, 20, prefix)
                                assert rc == 0, (dtype, dim, per_kv, sequences, max_new, tokens, prefix, p.prefix_rows, p.own_rows)


def test_a_selection_of_more_lists_than_the_merge_adds_up_is_refused(lib):
    """A plan is the caller's memory: one that was not made by the library has to hold to the same bounds, or a beam's normaliser would leave part of the vocabulary out."""
    from paella_amd import _abi
    from paella_amd._abi_decode import BeamSelectPlan
    p, d = BeamSelectPlan(), _abi.LaunchDims()
    for vocab in (131073, 140000, 524288):
        assert lib.paella_beam_select_plan_make(0, 1, 1, vocab, 5, ctypes.byref(p)) == 0
        assert (p.values, p.splits) == (32, -(-vocab // 8192)) and lib.paella_beam_select_dims(ctypes.byref(p), ctypes.byref(d)) == 0
        p.values, p.splits = 8, -(-vocab // 2048)
        assert p.splits > 64 and lib.paella_beam_select_dims(ctypes.byref(p), ctypes.byref(d)) == EINVAL
        assert lib.paella_beam_select_launch(ctypes.byref(p), AT, vocab, AT, None, 0, AT, AT, AT, AT, None, 0, None) == EINVAL
    assert lib.paella_beam_select_plan_make(0, 1, 1, 131072, 5, ctypes.byref(p)) == 0 and (p.values, p.splits) == (8, 64)


def test_no_selection_needs_more_shared_memory_than_any_launch_may_have(lib):
    from paella_amd._abi_decode import BeamSelectPlan
    p, most = BeamSelectPlan(), 0
    for beams in (1, 2, 16, 31, 32):
        for vocab in (1, 2048, 2049, 50021, 131072, 131073, 262144, 524288):
            for count in (1, 15, 16, 17, 32, 63, 64):
                for groups in (1, 300):
                    if lib.paella_beam_select_plan_make(0, groups, beams, vocab, count, ctypes.byref(p)) == 0:
                        most = max(most, p.dims.lds_bytes)
    assert most == 64 * 64 * 12


@pytest.mark.parametrize("sequences,keys,rows", [(24, 1600, 16), (48, 1200, 16), (48, 2200, 64), (48, 3000, 64), (24, 3000, 64)])
def test_fp32_rows_by_sixteen_as_long_as_that_is_faster(lib, sequences, keys, rows):
    """4 key heads of 128 for 16 query heads.  By 16 rows / by 64: 15.7 / 18.7 us, 19.6 / 20.4, then 23.2 / 21.7, 32.0 / 23.1, 21.2 / 20.2."""
    rc, p = attention_plan(lib, 0, 16, 4, 128, 64, sequences, 1, sequences, 1, keys)
    assert rc == 0 and (p.prefix_rows, p.own_rows) == (rows, 16)
