"""Calls of one plan that follow each other on a queue that keeps no order, without the caller waiting between them."""
import pytest
import torch

from test_decode_gpu import ATTEND, BF16, F32, attend_case, gen, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("given", [False, True], ids=["", "workspaces"])
def test_selections_one_after_another_on_a_queue_without_order(cuda, given):
    from paella_amd import decode, ops
    g = gen(5)
    for dtype, groups, beams, vocab, count in [(F32, 2, 4, 32000, 8), (BF16, 40, 4, 20001, 16)]:
        pick = decode.BeamSelect(groups, beams, vocab, count, dtype)
        inputs = [(randn(g, groups, beams, vocab, dtype=dtype, scale=3.0).to(cuda), randn(g, groups, beams).to(cuda)) for _ in range(4)]
        want = [pick(*x) for x in inputs]
        spaces = [pick.new_workspace() if given else None for _ in inputs]
        torch.cuda.synchronize()
        with ops.DirectQueue() as queue:
            for _ in range(3):
                got = [pick(*x, stream=queue.handle, workspace=w) for x, w in zip(inputs, spaces)]
                queue.wait()
                assert all(torch.equal(a, b) for x, y in zip(got, want) for a, b in zip(x, y))
        again = pick(*inputs[1])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(again, want[1]))


@pytest.mark.parametrize("given", [False, True], ids=["", "workspaces"])
def test_attention_one_after_another_on_a_queue_without_order(cuda, given):
    from paella_amd import decode, ops
    case = ATTEND[3]
    q, k, v, rows, tables, prefix_table, cache, batch = attend_case(case, cuda)
    attend = decode.PrefixAttention(case[1], cache, batch)
    assert attend.plan.stages == 1 and attend.plan.workspace_bytes
    queries = [(q.float() * f).to(q.dtype).to(cuda) for f in (1.0, 0.5, -0.75, 0.25)]
    want = [attend(x, cache, batch, out=torch.zeros_like(x)) for x in queries]   # (rows behind the last sequence stay zero)
    spaces = [attend.new_workspace() if given else None for _ in queries]
    torch.cuda.synchronize()
    with ops.DirectQueue() as queue:
        for _ in range(3):
            outs = [torch.zeros_like(x) for x in queries]
            for x, o, w in zip(queries, outs, spaces):
                attend(x, cache, batch, out=o, stream=queue.handle, workspace=w)
            queue.wait()
            assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_what_a_handle_is(cuda):
    from paella_amd import _abi, ops
    lib = _abi.ops()
    side = torch.cuda.Stream()
    with ops.DirectQueue() as one, ops.DirectQueue(ordered=True) as other:
        assert [lib.paella_stream_kind_of(h) for h in (None, side.cuda_stream, one.handle, other.handle)] == [0, 0, 2, 3]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            assert [lib.paella_stream_kind_of(h) for h in (None, side.cuda_stream, one.handle)] == [0, 1, 2]
            torch.zeros(4, device=cuda)
    graph.replay()
    torch.cuda.synchronize()
