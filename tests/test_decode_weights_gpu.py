"""Attention where one key has nearly all of the weight and very many others share the rest: against the closed form in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
HALF_STEP = {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11}


def weighted(scores, values):
    """softmax(scores) @ values in 64 bits, by numerator and denominator."""
    p = (scores.double() - scores.double().max()).exp()
    return p @ values.double() / p.sum()


@pytest.mark.parametrize("place", ["first", "middle", "last"])
@pytest.mark.parametrize("dtype,dim,heads,keys,gap,splits", [(F16, 64, 1, 32768, 12, 64), (F16, 64, 1, 32768, 16, 8), (F16, 128, 40, 32768, 16, 8), (F16, 128, 70, 131072, 17, 64),
                                                             (F16, 256, 20, 32768, 17, 8), (BF16, 128, 1, 32768, 16, 8), (BF16, 128, 70, 32768, 16, 8), (F32, 64, 1, 32768, 16, 8),
                                                             (F32, 64, 70, 32768, 16, 8)],
                         ids=lambda x: str(x)[6:] if isinstance(x, torch.dtype) else str(x))
def test_attention_beside_one_dominating_key(cuda, dtype, dim, heads, keys, gap, splits, place):
    """One key of value 0 whose score is `gap` above the others', whose scores spread over one more; the others make up all of the output.  By few rows and by many (the heads all
    share one key head), wherever the walk over the keys meets the one."""
    from paella_amd import decode
    g = torch.Generator()
    g.manual_seed(keys + gap)
    size, own = 64, 20
    q = torch.zeros((1, heads, dim))
    q[..., 0] = 16.0
    k, v = torch.zeros((keys + size, dim)), torch.zeros((keys + size, dim))
    k[:, 0] = torch.randint(-128, 1, (keys + size,), generator=g) / 2048.0    # exact in every type; scores from -1 to 0
    v[:] = torch.rand((dim,), generator=g) + 0.5
    v[:, 1::2] += torch.rand((keys + size, dim // 2), generator=g)
    one = {"first": 0, "middle": keys // 2 + 5, "last": keys + own - 1}[place]
    k[one, 0], v[one] = gap / 16.0, 0.0
    k, v = k.to(dtype), v.to(dtype)
    pages = (keys + size) // size
    cache = decode.KVCache(*(t.view(pages, 1, size, dim).to(cuda) for t in (k, v)))
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    # the prefix in all pages but the last, own tokens in that
    batch = decode.KVBatch(ints(own - 1), ints(pages - 1).view(1, 1), prefix_table=torch.arange(pages - 1, dtype=torch.int32, device=cuda), prefix_len=keys)
    attend = decode.PrefixAttention(heads, cache, batch, scale=1.0)
    assert attend.plan.prefix_splits >= splits
    attend.plan.prefix_splits = splits
    out = attend(q.to(dtype).to(cuda), cache, batch)
    torch.cuda.synchronize()
    seen = keys + own
    want = weighted(k[:seen, 0].float() * 16.0, v[:seen])
    # Relative to the output: its own rounding, and that of the weights above and below the line (fp32: none of these two), whose products are of second order.  In 32 bits, above and
    # below as well: sums of n terms one after the other, those of a part of the keys and then those of the parts; exponentials of arguments up to 32 whose factor and sum are
    # rounded (the products of queries and keys here are exact).  fp16, beside that: weights under 2^-14 by half a step of 2^-24, where the largest is 2^11 at least.
    half = HALF_STEP[dtype]
    n = keys // splits + 32 + splits + 1 + 8
    bound = want * ((half if dtype == F32 else 3.05 * half) + 2.0 ** -24 * (2 * n + 100)) + (seen * 2.0 ** -36 * 1.01 * v.double().max() if dtype == F16 else 0.0)
    err = (out[0].double().cpu() - want).abs()
    assert (err <= bound).all(), "off by %g of its bound, %g of the output" % ((err / bound).max(), (err / want).max())
    assert math.isfinite(float(want.sum())) and want.min() > 0


@pytest.mark.parametrize("heads", [1, 40, 70])
@pytest.mark.parametrize("dtype,dim", [(F16, 64), (F16, 128), (F16, 256), (BF16, 128), (F32, 64)], ids=lambda x: str(x)[6:] if isinstance(x, torch.dtype) else str(x))
def test_attention_of_scores_of_tens_of_millions(cuda, dtype, dim, heads):
    """Scores so far from 0 that a step of 32 bits is several units: one key is thousands above the others, and its value is the output; where many are within a few steps of
    one another their weights are anybody's, but they are weights."""
    from paella_amd import decode
    g = torch.Generator()
    g.manual_seed(dim + heads)
    size, pages = 64, 40
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    for near in (False, True):
        for top in (300.0, 600.0, 1000.0, 2000.0):
            k = torch.zeros((pages * size, dim))
            if near:
                k[:, 0] = top
                k[:, 1] = torch.rand((pages * size,), generator=g) * 40.0
            else:
                k[:, 0] = top * (0.25 + 0.5 * torch.rand((pages * size,), generator=g))   # below it in every type
                one = int(torch.randint(0, pages * size - 40, (1,), generator=g))
                k[one, 0] = top
            q = torch.zeros((1, heads, dim))
            q[..., 0], q[..., 1] = 32768.0, 1.0
            v = torch.rand((pages * size, dim), generator=g) + 0.5
            k, v, q = k.to(dtype), v.to(dtype), q.to(dtype)
            cache = decode.KVCache(*(t.view(pages, 1, size, dim).to(cuda) for t in (k, v)))
            batch = decode.KVBatch(ints(20), ints(pages - 1).view(1, 1), prefix_table=torch.arange(pages - 1, dtype=torch.int32, device=cuda), prefix_len=(pages - 1) * size)
            for sign in (1.0, -1.0):
                if sign < 0 and not near:
                    continue
                out = decode.PrefixAttention(heads, cache, batch, scale=1.0)((q * sign).to(cuda), cache, batch)[0].cpu()
                torch.cuda.synchronize()
                if near:
                    assert bool(((out >= v.min() * 0.98) & (out <= v.max() * 1.02)).all()), (top, sign)
                else:
                    # the sum and the weight that divides it, and the output: a rounding each
                    assert ((out.double() - v[one].double()).abs() <= v[one].double() * (HALF_STEP[dtype] * 1.01 + 2.0 ** -22)).all(), top
