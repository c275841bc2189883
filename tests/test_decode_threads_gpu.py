"""Several threads that call one plan at once, all on torch's default stream."""
import threading

import pytest
import torch

from test_decode_gpu import ATTEND, attend_case, gen, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("case", [0, 16])
def test_threads_that_share_a_plan_and_a_stream(cuda, case):
    from paella_amd import decode
    case = ATTEND[case]
    q, k, v, rows, tables, prefix_table, cache, batch = attend_case(case, cuda)
    queries = [(q.float() * f).to(q.dtype).to(cuda) for f in (1.0, 0.5, -0.75, 0.25)]
    logits, scores = [randn(gen(i), 2, 3, 5001).to(cuda) for i in range(4)], randn(gen(9), 2, 3).to(cuda)
    first, pick = decode.PrefixAttention(case[1], cache, batch), decode.BeamSelect(2, 3, 5001, 6)
    want, chosen = [first(x, cache, batch) for x in queries], [pick(x, scores) for x in logits]
    torch.cuda.synchronize()
    attend, pick = decode.PrefixAttention(case[1], cache, batch), decode.BeamSelect(2, 3, 5001, 6)
    outs, start = [[] for _ in queries], threading.Barrier(len(queries))

    def calls(i):
        torch.cuda.set_device(cuda)
        start.wait()
        for _ in range(20):
            outs[i].append((attend(queries[i], cache, batch), pick(logits[i], scores)))

    threads = [threading.Thread(target=calls, args=(i,)) for i in range(len(queries))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for i, mine in enumerate(outs):
        assert len(mine) == 20
        for out, got in mine:
            assert torch.equal(out, want[i]) and all(torch.equal(a, b) for a, b in zip(got, chosen[i]))
