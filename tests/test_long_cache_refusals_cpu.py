"""What the entry points over long caches refuse, beyond test_long_cache_cpu.py: nothing here is launched."""
import ctypes

from test_long_cache_cpu import (AT, CACHE_BYTES, CALLS, EINVAL, ENOSUP, K, KEPT, LENGTHS, OUT, PAGES, PAST, Q, TABLES, V, WEIGHTS, batch, bounds, cache, evict, lib,  # noqa: F401  (lib: a fixture)
                                 refs)


def test_selections_over_the_cache(lib):  # noqa: F811
    """A list, or what is kept between two launches, would be written over keys or values."""
    call = CALLS["select"](lib)
    sizes = dict(pages=3 * 2 * call.plan.count * 4, space=call.plan.workspace_bytes)
    for base in (K, V):
        for name, extent in sizes.items():
            for over in (base, base + CACHE_BYTES - 16, base - (extent + 15) // 16 * 16 + 16):
                assert call(**{name: over}) == EINVAL, (name, base // AT)


def test_evictions_of_more_threads_than_a_launch_has(lib):  # noqa: F811
    """Histories of thousands of tokens are picked from by 1024 threads a head, of which 2^32 are more than the runtime counts; the same heads with short ones are not."""
    from paella_amd import _abi
    from paella_amd._abi_long import KvEvictDesc
    c, d = cache(heads=8), _abi.LaunchDims()
    for tokens, most in ((1024, 16777215 // 3 // 8), (1040, 16777215 // 4 // 8), (2400, 16777215 // 4 // 8), (20000, 16777215 // 4 // 8)):
        for sequences, want in ((most, 0), (most + 1, ENOSUP), (550000, 0 if most >= 550000 else ENOSUP)):
            for stage in (0, 1):
                desc = KvEvictDesc(sequences, tokens // 16, 100, 0, 0)
                got = lib.paella_kv_evict_dims(*refs(desc, c), stage, ctypes.byref(d))
                assert got == want and (got or d.grid * d.block < 2 ** 32), (tokens, sequences, stage, d.grid, d.block)
            if want:
                assert evict(lib, c=c, sequences=sequences, max_pages=tokens // 16, keep=100) == ENOSUP


def test_bounds_of_tables_of_2_to_the_30_tokens(lib):  # noqa: F811
    """Refused as by the other operators that work on the same batch."""
    from paella_amd import _abi
    d = _abi.LaunchDims()
    for size, pages, want in ((8, (1 << 27) - 1, 0), (8, 1 << 27, ENOSUP), (8, 1 << 28, ENOSUP), (16, (1 << 26) - 1, 0), (16, 1 << 26, ENOSUP)):
        c, b = cache(size=size), batch(sequences=1, max_pages=pages)
        assert lib.paella_page_bounds_dims(*refs(c, b), ctypes.byref(d)) == want, (size, pages)
        if want:
            assert bounds(lib, c=c, b=b) == want


def test_numbers_that_begin_inside_a_word(lib):  # noqa: F811
    """Lengths, tables, lists, weights and positions are read and written by words."""
    from paella_amd._abi_decode import KvAppendDesc
    for name, at in (("weights", WEIGHTS), ("past", PAST), ("tables", TABLES), ("kept", KEPT), ("past_out", LENGTHS)):
        for off in (1, 2, 3):
            for stage in (None, 0, 1):
                assert evict(lib, **{name: at + off}, stage=stage) == EINVAL, (name, off, stage)
    d = KvAppendDesc(4, 64, 0, 1e-6, 256, 128, 128)
    for off in (1, 2, 3):
        assert lib.paella_kv_append_at_launch(ctypes.byref(d), *refs(cache(), batch()), KEPT + off, Q, OUT, OUT + AT // 2, None, None, WEIGHTS, PAGES, None, 0, None) == EINVAL, off
