"""Key weights where the number of a call's rows decides how they are taken through: on both sides of what is stored, and of what a workgroup has in LDS."""
import math

import pytest
import torch

import _long_ref as long_ref
from test_decode_gpu import BF16, F16, F32, within
from test_long_cache_gpu import Case

pytestmark = pytest.mark.gpu

ROWS = [(BF16, 64, 4, 4), (F16, 64, 1, 16), (F32, 256, 16, 1), (BF16, 64, 1, 17), (F16, 256, 17, 1), (F32, 64, 1, 17),   # a tile of scores, and one row more
        (BF16, 128, 4, 32), (BF16, 128, 1, 129), (F16, 64, 8, 16), (F32, 128, 8, 8), (F32, 128, 5, 13), (F32, 256, 4, 8), (F32, 256, 3, 11), (F16, 256, 8, 8), (F16, 256, 13, 5)]


@pytest.mark.parametrize("case", ROWS, ids=lambda c: "%s-%d-%dx%d" % (str(c[0])[6:], *c[1:]))
def test_weights_by_the_number_of_rows(cuda, case):
    from paella_amd import long_cache
    dtype, dim, per, new = case
    starts = [0, new, new + 1, new + 1 + (new + 1) // 2]   # sequences of all, of one and of half as many new tokens
    c = Case(dim + per, dtype, 2, dim, 16, [150, 0, 37], new, starts, prefix=21, behind=1)
    cache, batch = c.to(cuda)
    q = c.queries(2 * per)
    plan = long_cache.KeyWeights(2 * per, cache, batch)
    places = c.tables.shape[1] * 16
    stored = 3 * 2 * per * new * places * 4
    assert (plan.plan.workspace_bytes > stored) == (per * new <= 16)
    old = torch.rand((3, 2, places), generator=c.gen)
    weights = old.to(cuda)
    plan(q.to(cuda), cache, batch, weights)
    want, error = long_ref.weigh(c.host, q, c.k, old, 1 / math.sqrt(dim))
    within(weights, want, error)
    again = old.to(cuda)
    plan(q.to(cuda), cache, batch, again)
    assert torch.equal(weights, again)
