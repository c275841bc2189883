"""Beam selection at the ends of what logits can be, against its definition in 64 bits."""
import math

import pytest
import torch

import _decode_ref as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("vocab", [9, 3000, 20001])
@pytest.mark.parametrize("count", [1, 4, 40])
def test_select_of_logits_near_the_largest_numbers(cuda, dtype, vocab, count):
    """Logits whose product with log2 e is beyond 32 bits: spread between 1e38 and 3.3e38, all equal there, and as far below 0, beside ordinary ones and beside masked ones."""
    from paella_amd import decode
    g = torch.Generator()
    g.manual_seed(vocab)
    x = torch.randn((3, 4, vocab), generator=g) * 3.0
    x[0, 0] = (1.0 + 2.3 * torch.rand((vocab,), generator=g)) * 1e38
    x[0, 1] = 3.3e38
    x[0, 2] = (2.0 + torch.rand((vocab,), generator=g)) * -1e38
    x[1] = -math.inf
    x[1, :, vocab // 2] = 3.2e38
    x[1, 1, 0] = 3.0e38
    x[2, 0] = -math.inf
    x[2, 0, 3:5] = 2.5e38
    logits = x.to(dtype).to(cuda)
    scores = torch.randn((3, 4), generator=g).to(cuda)
    values, parents, tokens = (t.cpu() for t in decode.BeamSelect(3, 4, vocab, count, dtype)(logits, scores))
    for i, rows in enumerate(ref.select(logits.cpu(), scores.cpu(), None, 0, count)):
        assert [(int(p), int(t)) for p, t in zip(parents[i], tokens[i])] == [r[1:] for r in rows], i
        for c, r in enumerate(rows):   # 32-bit sums of exponentials (of arguments up to 64) and one rounding
            assert float(values[i, c]) == r[0] or abs(float(values[i, c]) - r[0]) <= 2.0 ** -24 * (128 + abs(r[0])), (i, c)
