"""Which scratch memory a plan's calls get, and what they wait for, with streams and queues that are only numbers and memory of the CPU."""
import pytest
import torch

STREAM, CAPTURING, UNORDERED, ORDERED = range(4)
HOME = 100   # torch's stream


class World:
    """What the front-end asks the library and torch about streams."""

    def __init__(self):
        self.kinds = {7: UNORDERED, 8: UNORDERED, 9: ORDERED, 20: STREAM, 21: CAPTURING}
        self.capturing = False
        self.log = []

    def paella_stream_kind_of(self, stream):
        return self.kinds.get(stream, STREAM)

    def paella_direct_queue_wait(self, stream):
        assert self.kinds[stream] in (UNORDERED, ORDERED)
        self.log.append(("wait", stream))
        return 0

    def synchronize(self, *device):
        assert not self.capturing
        self.log.append(("synchronize",) + device)


@pytest.fixture
def world(monkeypatch):
    from paella_amd import decode
    w = World()
    monkeypatch.setattr(decode, "_library", lambda: w)
    monkeypatch.setattr(decode, "_torch_stream", lambda: HOME)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: w.capturing)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: w)
    monkeypatch.setattr(torch.cuda, "synchronize", w.synchronize)
    yield w
    del decode._parked[:]


def spaces(nbytes=64, stages=1):
    from paella_amd import decode
    return decode._Workspaces(nbytes, stages)


CPU = torch.device("cpu")


def test_calls_on_a_queue_without_order_wait_for_one_another(world):
    from paella_amd import ops
    own = spaces()
    first = own.find(7, CPU, None, True)
    waits = lambda: [e for e in world.log if e[0] == "wait"]  # noqa: E731
    assert waits() == []                                   # nothing has used it
    assert own.find(7, CPU, None, True) is first and waits() == [("wait", 7)]
    assert own.find(7, CPU, None, True) is first and len(waits()) == 2
    ops._waits[7] = ops._waits.get(7, 0) + 1               # the caller has waited
    assert own.find(7, CPU, None, True) is first and len(waits()) == 2
    assert own.find(7, CPU, None, True) is first and len(waits()) == 3
    assert own.find(8, CPU, None, True) is not first and len(waits()) == 3
    for stream in (9, 20, HOME):                            # these keep an order themselves
        for _ in range(2):
            own.find(stream, CPU, None, True)
    assert own.find(HOME, CPU) is own.find(HOME, CPU) and len(waits()) == 3
    assert spaces(0).find(7, CPU, None, True) is None and len(waits()) == 3
    del ops._waits[7]


def test_captured_calls_find_no_workspace_that_is_not_the_graphs(world):
    """The graph's own memory is filled on torch's stream, ahead of what is captured there: a call on another stream of the capture would run beside the fill.  A stream that is
    captured while torch's is not would put its eager calls' workspace into the graph."""
    own = spaces()
    kept = own.find(HOME, CPU)
    for explicit in (False, True):
        world.capturing, world.kinds[HOME] = True, CAPTURING
        held = own.find(HOME, CPU, None, explicit)
        assert held is not kept and held is not own.find(HOME, CPU, None, explicit)
        world.capturing, world.kinds[HOME] = False, STREAM
        assert own.find(HOME, CPU, None, explicit) is kept
    world.capturing = True
    for stream in (20, 21, 7, 9):
        with pytest.raises(AssertionError):
            own.find(stream, CPU, None, True)
    assert spaces(0).find(21, CPU, None, True) is None
    world.capturing = False
    with pytest.raises(AssertionError):
        own.find(21, CPU, None, True)
    assert own.find(20, CPU, None, True) is own.find(20, CPU, None, True)


def test_memory_of_a_dropped_plan_stays_until_its_streams_are_done(world):
    """torch knows of no use of it but on its own stream, and would give it out again at once."""
    import gc
    import weakref
    from paella_amd import ops

    def used_and_dropped(*streams):
        own = spaces()
        refs = [weakref.ref(own.find(s, CPU, None, s != HOME)) for s in streams]
        del own
        gc.collect()
        return refs

    assert used_and_dropped(HOME)[0]() is None             # that one torch knows of
    stream, = used_and_dropped(20)
    assert stream() is not None
    queue, = used_and_dropped(7)                            # (whose first call waits for the device)
    assert stream() is None and ("synchronize", CPU) in world.log and queue() is not None
    other, = used_and_dropped(8)
    assert queue() is not None and other() is not None and ("wait", 7) not in world.log
    again, = used_and_dropped(7)
    assert ("wait", 7) in world.log and queue() is None and again() is not None and other() is not None
    ops._waits[8] = ops._waits.get(8, 0) + 1                # now a queue of ops.DirectQueue that has been closed, and so been waited for
    used_and_dropped(20)
    assert other() is None and again() is not None and ("wait", 8) not in world.log
    del ops._waits[8]


def test_a_whole_call_is_captured_whatever_the_streams_eager_calls_are_at(world):
    """It has memory of its own: only eager calls come between the stages of another."""
    own = spaces(64, 2)
    kept = own.find(HOME, CPU, 0)
    own.issued(HOME, CPU, 0)
    with pytest.raises(AssertionError):
        own.find(HOME, CPU)
    world.capturing = True
    assert own.find(HOME, CPU) is not kept
    for stage in (0, 1):
        with pytest.raises(AssertionError):
            own.find(HOME, CPU, stage)
    world.capturing = False
    assert own.find(HOME, CPU, 1) is kept
    own.issued(HOME, CPU, 1)
    with pytest.raises(AssertionError):
        own.find(HOME, CPU, 1)
    assert own.find(HOME, CPU) is kept


def test_a_queue_counts_as_closed_once_it_has_been_waited_for(world):
    """Closing waits for the queue's kernels: until then, memory that they may use is not let go of."""
    import types
    from paella_amd import ops
    seen = []
    queue = ops.DirectQueue.__new__(ops.DirectQueue)
    queue.handle = 8
    queue.lib = types.SimpleNamespace(paella_direct_queue_wait=lambda h: seen.append(("wait", 8 in ops._direct_queues)) or 0,
                                      paella_direct_queue_destroy=lambda h: seen.append(("destroy", 8 in ops._direct_queues)) or 0)
    ops._direct_queues.add(8)
    queue.close()
    assert seen == [("wait", True), ("destroy", False)] and queue.handle is None   # (another thread's new queue may have the handle from then on)
