"""Attention issued stage by stage: both stages of a call have to meet in one workspace, whatever else is issued, captured or replayed meanwhile."""
import pytest
import torch

from test_decode_gpu import ATTEND, attend_case

pytestmark = pytest.mark.gpu


def two_stages(cuda):
    from paella_amd import decode
    case = ATTEND[20]
    q, k, v, rows, tables, prefix_table, cache, batch = attend_case(case, cuda)
    attend = decode.PrefixAttention(case[1], cache, batch)
    assert attend.plan.stages == 2
    queries = [q.to(cuda), (q.float() * 0.5 + 0.25).to(q.dtype).to(cuda), q.flip(0).to(cuda)]
    return attend, queries, [attend(x, cache, batch) for x in queries], cache, batch


def test_captured_stages_are_refused_without_a_common_workspace_and_right_with_one(cuda):
    attend, queries, want, cache, batch = two_stages(cuda)
    out, outs = torch.empty_like(want[0]), [torch.empty_like(w) for w in want]
    graph = torch.cuda.CUDAGraph()
    refused = 0
    with torch.cuda.graph(graph):
        for stage in range(2):
            try:
                attend(queries[0], cache, batch, out=out, stage=stage)
            except AssertionError:
                refused += 1
        # two calls whose stages alternate, each in memory of its own
        spaces = [attend.new_workspace(cuda) for _ in range(2)]
        for stage in range(2):
            for i in range(2):
                attend(queries[i], cache, batch, out=outs[i], stage=stage, workspace=spaces[i])
    for _ in range(3):
        for o in outs:
            o.zero_()
        graph.replay()
        again = attend(queries[2], cache, batch)
        torch.cuda.synchronize()
        assert refused == 2 or torch.equal(out, want[0])
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1]) and torch.equal(again, want[2])


def test_stages_on_different_streams_and_queues(cuda):
    from paella_amd import ops
    attend, queries, want, cache, batch = two_stages(cuda)
    torch.cuda.synchronize()
    with ops.DirectQueue() as one, ops.DirectQueue() as other:
        # the second queue's workspace has the parts of another call: they must not be taken for this one's
        for _ in range(2):
            got = attend(queries[2], cache, batch, stage=0, stream=other.handle)
            other.wait()
            attend(queries[2], cache, batch, out=got, stage=1, stream=other.handle)
            other.wait()
            assert torch.equal(got, want[2])
        out = torch.zeros_like(want[0])
        attend(queries[0], cache, batch, out=out, stage=0, stream=one.handle)
        one.wait()
        with pytest.raises(AssertionError):
            attend(queries[0], cache, batch, out=out, stage=1, stream=other.handle)
        with pytest.raises(AssertionError):
            attend(queries[1], cache, batch, out=out, stage=0, stream=one.handle)   # over the parts that the second stage has yet to read
        attend(queries[0], cache, batch, out=out, stage=1, stream=one.handle)
        one.wait()
        assert torch.equal(out, want[0])
        space = attend.new_workspace(cuda)
        for i in (1, 0):
            out.zero_()
            attend(queries[i], cache, batch, out=out, stage=0, stream=one.handle, workspace=space)
            one.wait()
            attend(queries[i], cache, batch, out=out, stage=1, stream=other.handle, workspace=space)
            other.wait()
            assert torch.equal(out, want[i])
    with pytest.raises(AssertionError):
        attend(queries[0], cache, batch, stage=1)      # nothing to join
    out = attend(queries[1], cache, batch, stage=0)
    with pytest.raises(AssertionError):
        attend(queries[0], cache, batch)               # a whole call between the stages of another
    attend(queries[1], cache, batch, out=out, stage=1)
    whole = attend(queries[0], cache, batch)
    torch.cuda.synchronize()
    assert torch.equal(out, want[1]) and torch.equal(whole, want[0])


def test_workspaces_that_do_not_fit_are_refused(cuda):
    attend, queries, want, cache, batch = two_stages(cuda)
    space = attend.new_workspace(cuda)
    for bad in (space[:8], space[:-2], space.cpu(), torch.zeros(2 * space.numel(), dtype=torch.int32, device=cuda)[::2], space[1:]):
        with pytest.raises((AssertionError, RuntimeError)):
            attend(queries[0], cache, batch, workspace=bad)
    got = attend(queries[0], cache, batch, workspace=space)
    torch.cuda.synchronize()
    assert torch.equal(got, want[0])
