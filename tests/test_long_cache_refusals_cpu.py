"""What the entry points over long caches refuse, beyond test_long_cache_cpu.py: nothing here is launched."""
from test_long_cache_cpu import CACHE_BYTES, CALLS, EINVAL, K, V, lib  # noqa: F401  (lib: a fixture)


def test_selections_over_the_cache(lib):  # noqa: F811
    """A list, or what is kept between two launches, would be written over keys or values."""
    call = CALLS["select"](lib)
    sizes = dict(pages=3 * 2 * call.plan.count * 4, space=call.plan.workspace_bytes)
    for base in (K, V):
        for name, extent in sizes.items():
            for over in (base, base + CACHE_BYTES - 16, base - (extent + 15) // 16 * 16 + 16):
                assert call(**{name: over}) == EINVAL, (name, base // AT)
