"""Plans that are dropped while another stream still runs their calls."""
import pytest
import torch

from test_decode_gpu import ATTEND, attend_case, gen, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("case", [0, 16])
def test_dropped_plans_keep_their_memory_while_another_stream_runs(cuda, case):
    from paella_amd import decode
    case = ATTEND[case]
    q, k, v, rows, tables, prefix_table, cache, batch = attend_case(case, cuda)
    q = q.to(cuda)
    logits, scores = randn(gen(1), 2, 3, 5001).to(cuda), randn(gen(2), 2, 3).to(cuda)
    want, chosen = decode.PrefixAttention(case[1], cache, batch)(q, cache, batch), decode.BeamSelect(2, 3, 5001, 6)(logits, scores)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for _ in range(4):
        out = torch.zeros_like(want)
        attend, pick = decode.PrefixAttention(case[1], cache, batch), decode.BeamSelect(2, 3, 5001, 6)
        sizes = attend.plan.workspace_bytes // 4 + 1, pick.plan.workspace_bytes // 4 + 1
        attend(q, cache, batch, out=out, stream=side.cuda_stream)   # (the first call on a stream waits for torch's)
        pick(logits, scores, stream=side.cuda_stream)
        out.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            torch.cuda._sleep(20_000_000)
        attend(q, cache, batch, out=out, stream=side.cuda_stream)
        got = pick(logits, scores, stream=side.cuda_stream)
        del attend, pick
        others = [torch.full((n,), -1, dtype=torch.int32, device=cuda) for n in sizes for _ in range(4)]   # where their memory would be
        torch.cuda.synchronize()
        assert torch.equal(out, want) and all(torch.equal(a, b) for a, b in zip(got, chosen))
        del others
