"""Calls whose tensors do not all live on the current device, with the numbers of devices replaced."""
import types

import pytest
import torch


def test_a_batch_of_another_device_is_refused(monkeypatch):
    """A batch is made once and used for many calls: the device that is current by then may be another."""
    from paella_amd import decode
    monkeypatch.setattr(decode, "_current_device", lambda: -1)   # what tensors of the CPU say
    ints = lambda *shape: torch.zeros(shape, dtype=torch.int32)  # noqa: E731
    cache = decode.KVCache(torch.zeros((4, 2, 16, 64)), torch.zeros((4, 2, 16, 64)))
    batch = decode.KVBatch(ints(3), ints(3, 2))
    attend = decode.PrefixAttention(4, cache, batch)
    launched = []
    lib = types.SimpleNamespace(paella_kv_append_launch=lambda *a: launched.append(a) or 0)
    monkeypatch.setattr(decode, "_library", lambda: lib)
    monkeypatch.setattr(decode, "_stream", lambda s: 0)
    attend._launch = lambda *a: launched.append(a) or 0
    attend.workspaces.nbytes = 0
    k, q = torch.zeros((3, 2, 64)), torch.zeros((3, 4, 64))
    decode.kv_append(cache, batch, k, k, q=q)
    attend(q, cache, batch)
    assert len(launched) == 2
    batch.past = types.SimpleNamespace(get_device=lambda: 1)
    for call in (lambda: decode.kv_append(cache, batch, k, k, q=q), lambda: attend(q, cache, batch)):
        with pytest.raises(AssertionError):
            call()
    assert len(launched) == 2
