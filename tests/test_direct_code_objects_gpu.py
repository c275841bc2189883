"""What the first direct-dispatch queue of a process loads, in a process of its own."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CHILD = """
import torch
from paella_amd import _abi, decode, ops
loaded = _abi.ops().paella_direct_code_objects
cuda = torch.device("cuda:0")
counts = [loaded()]
with ops.DirectQueue() as queue:
    counts.append(loaded())
    x = torch.rand((1, 3, 8, 8), device=cuda)
    ops.softmax(x.view(1, -1), stream=queue.handle)
    queue.wait()
    counts.append(loaded())
    logits, scores = torch.randn((2, 3, 500), device=cuda), torch.zeros((2, 3), device=cuda)
    pick = decode.BeamSelect(2, 3, 500, 4)
    want = pick(logits, scores)
    got = pick(logits, scores, stream=queue.handle)
    queue.wait()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    counts.append(loaded())
    cache = decode.KVCache.empty(4, 2, 8, 64, torch.bfloat16)
    batch = decode.KVBatch(torch.zeros(3, dtype=torch.int32, device=cuda), torch.arange(3, dtype=torch.int32, device=cuda).view(3, 1))
    q = torch.randn((3, 4, 64), device=cuda).bfloat16()
    k = torch.randn((3, 2, 64), device=cuda).bfloat16()
    decode.kv_append(cache, batch, k, k, stream=queue.handle)
    queue.wait()
    attend = decode.PrefixAttention(4, cache, batch)
    want = attend(q, cache, batch)
    got = attend(q, cache, batch, stream=queue.handle)
    queue.wait()
    assert torch.equal(got, want) and torch.equal(got, k.repeat_interleave(2, 1))
    counts.append(loaded())
print("loaded", *counts)
"""


def test_a_process_loads_the_kernels_that_it_uses(cuda):
    """A server of the models' operators does not load those of a decoding step; a decoding step loads the attention of its type."""
    run = subprocess.run([sys.executable, "-c", CHILD], cwd=ROOT, capture_output=True, text=True, timeout=100)
    assert run.returncode == 0, run.stderr[-2000:]
    assert run.stdout.split()[-6:] == ["loaded", "0", "2", "2", "3", "4"], run.stdout
