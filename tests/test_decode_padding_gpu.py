"""Rows behind the last sequence of a ragged batch, as a captured step of fixed size has them: what lies there is nobody's business."""
import math

import pytest
import torch

from test_decode_gpu import BF16, F16, F32, attend_case

pytestmark = pytest.mark.gpu

# dtype, heads, kv heads, head size, page size, past, most new, starts, prefix, rows behind
PADDED = [(BF16, 8, 2, 128, 64, [200, 1, 63], 5, [0, 5, 6, 9], 1300, 7), (F16, 32, 2, 64, 16, [20, 300, 11], 4, [0, 4, 5, 9], 4000, 20), (F32, 16, 1, 128, 16, [25, 0, 300], 3, [0, 3, 4, 5], 2100, 9),
          (BF16, 16, 1, 256, 16, [70, 9], 2, [0, 2, 3], 900, 5)]


@pytest.mark.parametrize("case", PADDED, ids=lambda c: "%s-%dx%dx%d-%d" % ((str(c[0])[6:],) + c[1:4] + (c[8],)))
def test_padding_leaves_every_bit_of_the_others(cuda, case):
    from paella_amd import decode
    dtype, heads, kv_heads, dim = case[:4]
    q, k, v, rows, tables, prefix_table, cache, batch = attend_case(case[:9], cuda)
    used, more = case[7][-1], case[9]
    g = torch.Generator()
    g.manual_seed(1)
    longer = decode.KVBatch(batch.past, batch.tables, max_new=case[6], starts=batch.starts, tokens=used + more, prefix_table=prefix_table.to(cuda), prefix_len=case[8])
    attend = decode.PrefixAttention(heads, cache, longer)
    outs = []
    for fill in (torch.zeros((more, heads, dim)), torch.randn((more, heads, dim), generator=g) * 40.0, torch.full((more, heads, dim), math.nan), torch.full((more, heads, dim), 1e4)):
        queries = torch.cat((q[:used], fill.to(dtype))).to(cuda)
        out = torch.full(queries.shape, 7.0, dtype=dtype, device=cuda)
        attend(queries, cache, longer, out=out)
        torch.cuda.synchronize()
        assert bool((out[used:] == 7.0).all()) and not bool((out[:used] == 7.0).all(-1).any())
        outs.append(out[:used])
    for out in outs[1:]:
        assert torch.equal(out, outs[0])
