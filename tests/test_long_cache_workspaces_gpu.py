"""Scratch memory of the operators over long caches: whatever it holds beyond what a plan wants zeroed, results are the same."""
import math

import pytest
import torch

import _long_ref as long_ref
from test_decode_gpu import BF16, F16, F32, within
from test_long_cache_gpu import Case
from test_long_cache_uses_gpu import USES, Use

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", [n for n in USES if n.split()[0] in ("select", "attend", "weigh") and n != "attend alone"])
@pytest.mark.parametrize("poison", [0x7FC00000, -1, 0x3F800000])
def test_workspaces_that_hold_anything(cuda, name, poison):
    use = Use(name, cuda)
    want, space = use.eager(), use.plan.new_workspace()
    assert space.numel() * 4 >= use.plan.plan.workspace_bytes
    space.fill_(poison)
    space[:use.plan.plan.zero_bytes // 4] = 0
    for _ in range(3):
        use.check(use.call(use.fresh(), workspace=space), want)


@pytest.mark.parametrize("case", [(BF16, 16, 64, 1), (F16, 5, 256, 1), (F32, 2, 128, 3)], ids=lambda c: str(c[0])[6:])
def test_few_rows_over_tables_too_wide_for_their_scores(cuda, case):
    """Weights are those of the definition where scores are not stored, and what lies behind a sequence stays as it was."""
    from paella_amd import decode, long_cache
    dtype, heads, dim, new = case
    c = Case(dim + 3, dtype, 1, dim, 8, [300, 20, 0], new, prefix=30)
    cache, batch = c.to(cuda)
    tables = torch.full((3, (1 << 28) // (3 * 8 * heads * new) + 8), -1, dtype=torch.int32, device=cuda)
    tables[:, :c.tables.shape[1]] = batch.tables
    wide = decode.KVBatch(batch.past, tables, max_new=new, prefix_table=batch.prefix_table, prefix_len=30)
    plan = long_cache.KeyWeights(heads, cache, wide)
    assert plan.plan.workspace_bytes < 1 << 20
    old = torch.rand((3, 1, c.tables.shape[1] * 8), generator=c.gen)
    weights = torch.full((3, 1, tables.shape[1] * 8), 0.25, device=cuda)
    weights[..., :old.shape[2]] = old.to(cuda)
    q = c.queries(heads)
    plan(q.to(cuda), cache, wide, weights)
    want, error = long_ref.weigh(c.host, q, c.k, old, 1 / math.sqrt(dim))
    within(weights[..., :old.shape[2]], want, error)
    assert (weights[..., old.shape[2]:] == 0.25).all()
