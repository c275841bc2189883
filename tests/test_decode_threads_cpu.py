"""Two threads that call one plan on one stream, with the library's launches replaced by ones that take their time."""
import threading
import time

import torch

from test_decode_workspaces_cpu import HOME, world  # noqa: F401


def test_two_stages_of_a_call_stay_together(world, monkeypatch):  # noqa: F811
    """A call of two stages is two launches: another thread's between them would leave its parts where the second one looks for this call's."""
    from paella_amd import decode
    monkeypatch.setattr(decode, "_on_device", lambda *tensors: None)
    monkeypatch.setattr(decode, "_stream", lambda stream: HOME)
    ints = lambda *shape: torch.zeros(shape, dtype=torch.int32)  # noqa: E731
    cache = decode.KVCache(torch.zeros((4, 2, 16, 64)), torch.zeros((4, 2, 16, 64)))
    batch = decode.KVBatch(ints(40), ints(40, 2), prefix_table=ints(300), prefix_len=4800)
    attend = decode.PrefixAttention(32, cache, batch)
    assert attend.plan.stages == 2 and attend.plan.workspace_bytes
    q, log = torch.zeros((40, 32, 64)), []

    def launch(plan, cache, batch, q, stride, out, workspace, *rest):
        for stage in range(2):
            log.append((threading.get_ident(), stage, workspace))
            time.sleep(0.002)
        return 0

    attend._launch = launch
    start = threading.Barrier(4)

    def calls():
        start.wait()
        for _ in range(5):
            attend(q, cache, batch)

    threads = [threading.Thread(target=calls) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(log) == 40 and len({w for _, _, w in log}) == 1     # one workspace, whoever asked first
    assert all(log[i][0] == log[i + 1][0] and (log[i][1], log[i + 1][1]) == (0, 1) for i in range(0, 40, 2))
