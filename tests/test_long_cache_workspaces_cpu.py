"""What of a plan's scratch memory is filled: a call under graph capture fills its own again at every replay."""
import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

from test_long_cache_cpu import attend_plan, batch, cache, lib, select_plan, weigh_plan  # noqa: F401  (lib: a fixture)


class Filled(TorchDispatchMode):
    """Bytes that operations write which are not allocations."""

    def __init__(self):
        super().__init__()
        self.bytes = 0

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        out = func(*args, **(kwargs or {}))
        if func.overloadpacket.__name__ in ("zeros", "zero_", "fill_", "full"):
            self.bytes += out.numel() * out.element_size()
        return out


def filled(nbytes, stages, *zeroed):
    from paella_amd import decode
    with Filled() as f:
        space = decode._Workspaces(nbytes, stages, *zeroed).new(torch.device("cpu"))
    assert space.numel() * 4 >= nbytes and not space[:(zeroed[0] if zeroed else nbytes) // 4].any()
    return f.bytes


def test_what_has_to_be_zero_is_filled_and_no_more():
    assert filled(4096, 1) >= 4096          # (all of it where a plan does not say)
    assert filled(1 << 20, 1, 512) == 512
    assert filled(1 << 20, 2, 0) == 0


@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_plans_say_what_has_to_be_zero(lib, dtype):  # noqa: F811
    """The counters of calls whose last workgroup puts a row together; nothing else is read before it is written."""
    c = cache(dtype=dtype, heads=2, dim=64, size=64, pages=4000)
    plans = [(select_plan(lib, c, batch(max_pages=500))[1], 1, 3 * 2 * 128), (select_plan(lib, c, batch(sequences=1, max_pages=3000))[1], 2, 0),
             (attend_plan(lib, c, batch(max_pages=500), count=40)[1], 1, None), (attend_plan(lib, c, batch(sequences=1, max_pages=3000), count=300)[1], 2, 0),
             (weigh_plan(lib, c, batch(max_pages=500))[1], 2, 0), (weigh_plan(lib, c, batch(max_new=40, max_pages=500))[1], 2, 0)]
    for p, stages, zero in plans:
        assert p.stages == stages and (p.zero_bytes == zero if zero is not None else 0 < p.zero_bytes < p.workspace_bytes // 8), (type(p).__name__, p.stages, p.zero_bytes)
        assert p.zero_bytes % 4 == 0
    whole = attend_plan(lib, c, batch(sequences=500, max_pages=4), count=4)[1]
    assert (whole.workspace_bytes, whole.zero_bytes) == (0, 0)


@pytest.mark.parametrize("dtype, dim", [(1, 64), (2, 128), (0, 256)])
def test_key_weights_of_wide_tables_keep_a_bounded_workspace(lib, dtype, dim):  # noqa: F811
    """Scores are stored for few rows up to 1 GB by the tables' width; beyond it a call keeps each row's sums alone, as with many rows."""
    c = cache(dtype=dtype, heads=8, dim=dim, size=64, pages=100)
    for sequences, rows, pages in ((32, 16, 1024), (32, 16, 2048), (32, 4, 1024), (1, 16, 1 << 15), (500, 1, 4096), (2, 8, 200000)):
        rc, p = weigh_plan(lib, c, batch(sequences=sequences, max_new=1, max_pages=pages), 8 * rows)
        scores = sequences * 8 * rows * pages * 64 * 4
        sums = p.splits * sequences * 8 * rows * 8
        assert rc == 0 and p.workspace_bytes == -(-sums // 256) * 256 + (scores if scores <= 1 << 30 else 0), (sequences, rows, pages)
