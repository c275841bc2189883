"""Norms of an append at the ends of what head's values can be, against the definition in 64 bits."""
import pytest
import torch

from test_decode_gpu import gen, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("size", [1e-21, 3e-20, 1e-19, 1e18])
def test_norms_of_tiny_and_huge_heads(cuda, dtype, size):
    """No epsilon, and mean squares under the smallest normal number or near the largest: the norm is the head's direction all the same."""
    from paella_amd import decode
    g = gen(3)
    cache = decode.KVCache.empty(2, 2, 8, 64, dtype)
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    batch = decode.KVBatch(ints(0, 3), ints(0, 1).view(2, 1))
    q, k = (randn(g, 2, h, 64, dtype=torch.float32) * size for h in (4, 2))
    q, k = q.to(dtype), k.to(dtype)
    weight = torch.rand((64,), generator=g) + 0.5
    out = decode.kv_append(cache, batch, k.to(cuda), k.to(cuda), q=q.to(cuda), q_norm=weight.to(cuda), k_norm=weight.to(cuda), eps=0.0)
    torch.cuda.synchronize()
    half = torch.finfo(dtype).eps / 2
    for got, x in ((out, q), (torch.stack((cache.k[0, :, 0], cache.k[1, :, 3])), k)):
        x = x.double()
        want = x / x.pow(2).mean(-1, keepdim=True).sqrt() * weight.double()
        # squares under 2^-126 are off by half a step of 2^-149 each, and so is each of their sums and the mean; half of that reaches the root
        mean = x.pow(2).mean(-1, keepdim=True)
        bound = want.abs() * (half + 2.0 ** -24 * 80 + 0.5 * 2.0 ** -150 * (2 + 1) / mean)
        assert ((got.double().cpu() - want).abs() <= bound).all(), ((got.double().cpu() - want).abs() / want.abs()).max()
