"""Calls captured on a stream that is not torch's current one."""
import pytest
import torch

from test_decode_gpu import ATTEND, attend_case, gen, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("case", [0, 16])
def test_calls_captured_on_a_side_stream_need_a_workspace(cuda, case):
    from paella_amd import decode
    case = ATTEND[case]
    q, k, v, rows, tables, prefix_table, cache, batch = attend_case(case, cuda)
    q = q.to(cuda)
    attend, pick = decode.PrefixAttention(case[1], cache, batch), decode.BeamSelect(2, 3, 5001, 6)
    logits, scores = randn(gen(1), 2, 3, 5001).to(cuda), randn(gen(2), 2, 3).to(cuda)
    want, chosen = attend(q, cache, batch), pick(logits, scores)
    spaces = attend.new_workspace(), pick.new_workspace()
    out, side, graph = torch.empty_like(want), torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        home = torch.cuda.current_stream()
        side.wait_stream(home)
        with pytest.raises(AssertionError):
            attend(q, cache, batch, out=out, stream=side.cuda_stream)
        with pytest.raises(AssertionError):
            pick(logits, scores, stream=side.cuda_stream)
        attend(q, cache, batch, out=out, stream=side.cuda_stream, workspace=spaces[0])
        got = pick(logits, scores, stream=side.cuda_stream, workspace=spaces[1])
        home.wait_stream(side)
    for _ in range(3):
        out.zero_()
        for t in got:
            t.zero_()
        graph.replay()
        eager = attend(q, cache, batch)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(eager, want) and all(torch.equal(a, b) for a, b in zip(got, chosen))


def test_a_stream_captured_beside_torchs_needs_a_workspace(cuda):
    """torch's current stream is not the one under capture: what the eager calls of that stream use stays out of the graph."""
    from paella_amd import decode
    pick = decode.BeamSelect(2, 3, 5001, 6)
    logits, scores = randn(gen(1), 2, 3, 5001).to(cuda), randn(gen(2), 2, 3).to(cuda)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    want = pick(logits, scores)
    pick(logits, scores, stream=side.cuda_stream)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        graph.capture_begin(capture_error_mode="thread_local")
        kept = logits + 1.0
        with torch.cuda.stream(torch.cuda.default_stream()):
            with pytest.raises(AssertionError):
                pick(logits, scores, stream=side.cuda_stream)
        graph.capture_end()
    graph.replay()
    got = pick(logits, scores, stream=side.cuda_stream)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(kept, logits + 1.0)
