"""The overlaps of inputs and outputs that the decoding step's operators allow: a selection's scores in place, queries in place, queries of a packed projection."""
import ctypes

import pytest
import torch

from test_decode_gpu import BF16, F32, gen, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("groups,beams,vocab,count,dtype", [(40, 4, 9001, 4, F32), (60, 8, 2500, 8, BF16), (1, 4, 32000, 9, F32), (1, 16, 3000, 3, BF16)])
def test_scores_in_place(cuda, groups, beams, vocab, count, dtype):
    from paella_amd import _abi, decode
    lib, g = _abi.ops(), gen(vocab)
    pick = decode.BeamSelect(groups, beams, vocab, count, dtype)
    logits, scores = randn(g, groups, beams, vocab, dtype=dtype, scale=3.0).to(cuda), randn(g, groups, beams).to(cuda)
    want = pick(logits, scores)
    space = pick.new_workspace()
    for _ in range(3):
        own = torch.zeros(groups * max(beams, count), device=cuda)
        own[:groups * beams] = scores.flatten()
        parents, tokens = (torch.empty((groups, count), dtype=torch.int32, device=cuda) for _ in range(2))
        rc = lib.paella_beam_select_launch(ctypes.byref(pick.plan), logits.data_ptr(), vocab, own.data_ptr(), None, 0, own.data_ptr(), parents.data_ptr(), tokens.data_ptr(),
                                           space.data_ptr(), torch.cuda.current_stream().cuda_stream, 0, None)
        assert rc == 0
        torch.cuda.synchronize()
        assert torch.equal(own[:groups * count].view(groups, count), want[0]) and torch.equal(parents, want[1]) and torch.equal(tokens, want[2])


def test_queries_in_place_and_beside_keys_and_values(cuda):
    """One token of a packed projection, and several side by side: the queries' place ends where the keys' begins."""
    from paella_amd import decode
    g = gen(4)
    for tokens in (1, 5):
        cache, other = decode.KVCache.empty(tokens, 2, 8, 64, BF16), decode.KVCache.empty(tokens, 2, 8, 64, BF16)
        ints = lambda *x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
        batch = decode.KVBatch(ints(*range(tokens)), torch.arange(tokens, dtype=torch.int32, device=cuda).view(tokens, 1), prefix_len=0)
        freq = torch.rand((32,), generator=g).to(cuda)
        store = randn(g, tokens * 8 * 64, dtype=BF16).to(cuda)
        q, k, v = (store[i * tokens * 64:j * tokens * 64].view(tokens, j - i, 64) for i, j in ((0, 4), (4, 6), (6, 8)))
        want = decode.kv_append(other, batch, k, v, q=q, inv_freq=freq)
        got = decode.kv_append(cache, batch, k, v, q=q, inv_freq=freq, out=q)
        torch.cuda.synchronize()
        assert got is q and torch.equal(got, want) and torch.equal(cache.k, other.k) and torch.equal(cache.v, other.v) and bool(cache.k.any())
