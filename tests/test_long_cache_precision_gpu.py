"""How many bits the operators over long caches keep, where a call of a few tokens shows it."""
import math

import pytest
import torch

import _decode_ref as ref
import _long_ref as long_ref
from test_decode_gpu import BF16, F16, F32, within
from test_long_cache_gpu import Case, lists

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("dtype", [BF16, F16], ids=lambda d: str(d)[6:])
def test_attention_over_pages_is_off_by_its_own_rounding(cuda, dtype, dim):
    """Weighted values that cancel: where a sum is small beside what it adds up, weights of the type's few bits would show.  A weight is held as the sum of two numbers of the type, the second of which has what
    the first leaves, so what is lost is half a step of half a step of it, once in the sum of the values and once in that of the weights; to that come the output's own rounding and what 32-bit sums add, as in
    attention_bound.  fp16 has no steps below 2^-24: an output is off by half of that, and a weight, whose largest is 2^11 at least, by 2^-36 of the largest."""
    from paella_amd import long_cache
    c = Case(dim, dtype, 2, dim, 16, [70, 40, 3], 2, prefix=19)
    cache, batch = c.to(cuda)
    q, pages = c.queries(8, scale=0.05), lists(c, 7, "any")
    out = long_cache.PageAttention(8, cache, batch, 7)(q.to(cuda), cache, batch, pages.to(cuda))
    want, weight, products, most = long_ref.attend(c.host, q, c.k, c.v, pages, 1 / math.sqrt(dim))
    half = ref.HALF_STEP[dtype]
    largest = c.v[~c.v.isnan()].abs().max().item()
    tiny = 2.0 ** -25 + 2.0 ** -36 * most * largest if dtype == F16 else 0.0
    within(out, want, half * want.abs() + (2 * half ** 2 + 2.0 ** -24 * (2 * dim * products[..., None] + 2 * most + 64)) * weight * 1.01 + tiny)


@pytest.mark.parametrize("case", [(F32, 4, 256, 64), (BF16, 8, 128, 70), (F16, 8, 64, 40)], ids=lambda c: str(c[0])[6:])
def test_a_heavy_old_weight_is_rounded_once(cuda, case):
    """Many rows, which are taken through in several chunks, each of which gives a token less than half a step of what it weighs already: half a step of the result, and the error of the call's own sum."""
    from paella_amd import long_cache
    dtype, heads, dim, new = case
    c = Case(dim + 1, dtype, 1, dim, 16, [100, 70], new, prefix=20)
    cache, batch = c.to(cuda)
    q = c.queries(heads, scale=0.3)
    places = c.tables.shape[1] * 16
    nothing = torch.zeros((2, 1, places))
    old = nothing + 2.0 ** 24
    weights = old.to(cuda)
    long_cache.KeyWeights(heads, cache, batch)(q.to(cuda), cache, batch, weights)
    want, error = long_ref.weigh(c.host, q, c.k, nothing, 1 / math.sqrt(dim))
    for b, past in enumerate(c.past):
        assert want[b, :, :past].min() > 1.0   # half a step of the old weight
        want[b, :, :past] += old[b, :, :past]
        want[b, :, past + new:] = old[b, :, past + new:]
    within(weights, want, error + 2.0 ** -24 * want.abs())
