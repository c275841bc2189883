"""Append at given positions, in every type and form, against its definition in 64 bits."""
import pytest
import torch

import _decode_ref as ref
from test_decode_gpu import BF16, F16, F32, randn, within
from test_long_cache_gpu import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("norms", [False, True], ids=["plain", "normed"])
@pytest.mark.parametrize("rotary", [64, 32])
@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "pairs"])
@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=lambda d: str(d)[6:])
def test_rotation_at_positions(cuda, dtype, interleaved, rotary, norms):
    """A ragged batch with rows behind it and a page outside the cache, at positions from below 0 to the largest.  Tolerances as in test_append (an angle of position 2^31 in 64 bits is off by 2^-22 radians, 4 of the
    64 roundings)."""
    from paella_amd import decode
    starts, past, heads, kv_heads, page = [0, 3, 3, 5, 6], [14, 7, 0, 21], 4, 2, 16
    c = Case(rotary + norms, dtype, kv_heads, 64, page, past, 3, starts, prefix=20, bad=[((3, 1), -4)], behind=2)
    cache, batch = c.to(cuda)
    q, k, v = (randn(c.gen, c.tokens, n, 64, dtype=dtype) for n in (heads, kv_heads, kv_heads))
    wq, wk = ((randn(c.gen, 64) * 0.3 + 1 for _ in range(2)) if norms else (None, None))
    freq = torch.tensor([10000.0 ** (-2 * i / rotary) for i in range(rotary // 2)])
    positions = [100000, 5, -3, 2 ** 31 - 1]
    dev = [t if t is None else t.to(cuda) for t in (q, k, v, wq, wk, freq)]
    out = torch.full(q.shape, 7.0, dtype=dtype, device=cuda)
    before = cache.k.cpu(), cache.v.cpu()
    decode.kv_append(cache, batch, dev[1], dev[2], q=dev[0], q_norm=dev[3], k_norm=dev[4], eps=1e-5, inv_freq=dev[5], interleaved=interleaved, out=out,
                     positions=torch.tensor(positions, dtype=torch.int32, device=cuda))

    def bound(want):
        return ref.HALF_STEP[dtype] * want.abs() + 64 * 2.0 ** -24 * want.abs().amax(-1, keepdim=True) + (2.0 ** -25 if dtype == F16 else 0)

    untouched = torch.ones(cache.k.shape[:1] + cache.k.shape[2:3], dtype=torch.bool)
    for t, owner in enumerate(c.host.rows):
        if owner is None:
            assert (out[t] == 7.0).all()
            continue
        b, own = owner
        at = positions[b] + own - past[b]
        want = ref.norm_rotate(q[t].double(), None if wq is None else wq.double(), 1e-5, freq.double().tolist(), interleaved, at)
        within(out[t], want, bound(want))
        p = c.host.physical(b, c.host.shared + own // page)
        if p is None:
            continue
        want = ref.norm_rotate(k[t].double(), None if wk is None else wk.double(), 1e-5, freq.double().tolist(), interleaved, at)
        within(cache.k[p, :, own % page], want, bound(want))
        assert torch.equal(cache.v[p, :, own % page].cpu(), v[t])
        untouched[p, own % page] = False
    for got, was in zip((cache.k.cpu(), cache.v.cpu()), before):
        assert torch.equal(got.transpose(1, 2)[untouched].nan_to_num(9.0), was.transpose(1, 2)[untouched].nan_to_num(9.0))
