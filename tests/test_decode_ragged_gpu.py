"""Attention over ragged batches whose bound on the new tokens of a sequence is far above what they have, against the definition in 64 bits."""
import math

import pytest
import torch

import _decode_ref as ref
from test_decode_gpu import attend_case, within

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16

# dtype, heads, kv heads, head size, page size, past, most new, starts, prefix; a row behind the last sequence in each
RAGGED = [(BF16, 32, 8, 128, 64, [100, 5, 0, 300], 32, [0, 3, 3, 10, 13], 5000), (F16, 16, 1, 64, 16, [40, 333], 200, [0, 1, 3], 700), (F32, 8, 1, 128, 8, [3, 90, 12], 40, [0, 2, 4, 7], 900),
          (BF16, 12, 2, 256, 16, [70], 64, [0, 5], 0)]


@pytest.mark.parametrize("case", RAGGED, ids=lambda c: "%s-%dx%dx%d-%d" % ((str(c[0])[6:],) + c[1:4] + (c[6],)))
def test_attention_of_few_rows_with_room_for_many(cuda, case):
    from paella_amd import decode
    dtype, heads, kv_heads, dim, size, past, new, starts, prefix = case
    q, k, v, rows, tables, prefix_table, cache, batch = attend_case(case, cuda, True)
    out = torch.full(q.shape, 7.0, dtype=dtype, device=cuda)
    attend = decode.PrefixAttention(heads, cache, batch)
    for _ in range(2):
        attend(q.to(cuda), cache, batch, out=out)
    torch.cuda.synchronize()
    want, weight, products = ref.attention(q, k, v, rows, tables, prefix_table, prefix, 1 / math.sqrt(dim))
    bound = ref.attention_bound(want, weight, products, dtype, prefix + max(past) + new)
    for t, owner in enumerate(rows):
        if owner is None:
            want[t] = 7.0    # left as it was
            bound[t] = 0.0
    within(out, want, bound)
