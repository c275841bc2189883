"""Functional front-end over the operators of a decoding step (include/paella_decode.h): a paged cache of keys and values, attention for
sequences that share a prefix, beam search.

As in `ops`: tensors are torch CUDA tensors, everything runs on the calling thread's current torch stream unless a stream handle is
given, arguments that do not fit raise AssertionError here and RuntimeError from the library.  One step of a batch:

    cache = KVCache.empty(num_pages, kv_heads, page_size, head_dim, torch.bfloat16)      # one per layer
    batch = KVBatch(past, tables, prefix_table=shared, prefix_len=len_of_prefix)         # past, tables: int32 device tensors
    attend = PrefixAttention(heads, cache, batch)
    q = kv_append(cache, batch, k, v, q=q, q_norm=wq, k_norm=wk, inv_freq=freq)          # per layer
    out = attend(q, cache, batch)
    past += 1

Lengths and tables are read on the device at every launch, so a captured step may be replayed while they change.
"""
import ctypes
import threading

import torch

from . import _abi
from ._abi import LaunchDims, check
from ._abi_decode import BeamReorderDesc, BeamSelectPlan, KvAppendDesc, KvBatch, KvCache, PrefixAttentionPlan
from .ops import _direct_queues, _stream, _torch_stream, _waits

_STREAM, _STREAM_CAPTURING, _QUEUE_UNORDERED, _QUEUE_ORDERED = range(4)  # enum paella_stream_kind
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}

try:
    from torch._C import _cuda_getDevice as _current_device
except ImportError:
    _current_device = torch.cuda.current_device


_lib = None


def _library():
    global _lib
    if _lib is None:
        _lib = _abi.ops()
    return _lib


# As in `ops`, a small call's time is what it costs the calling thread: the checks below look at each tensor once and are kept to under half a microsecond each.

def _on_device(*tensors):
    """Launches go to the current device: every tensor has to live there."""
    device = _current_device()
    for t in tensors:
        if t is not None and t.get_device() != device:
            raise AssertionError("tensors of the current device are needed")


def _ints(t, *shape):
    assert t.dtype is torch.int32 and t.shape == shape and t.is_contiguous(), ("contiguous int32 of shape %s" % (shape,), t.dtype, tuple(t.shape))
    return t.data_ptr()


def _floats(t, n):
    if t is None:
        return None
    assert t.dtype is torch.float32 and t.numel() == n and t.is_contiguous(), ("%d contiguous float32" % n, t.dtype, tuple(t.shape))
    return t.data_ptr()


def _rows(t, tokens, heads, cache):
    """Address and row stride of [tokens, heads, head_dim] whose heads lie side by side."""
    dim = cache.head_dim
    assert t.dtype is cache.dtype and t.shape == (tokens, heads, dim), (t.dtype, tuple(t.shape), "wanted", cache.dtype, (tokens, heads, dim))
    row, head, value = t.stride()
    assert value == 1 and (head == dim or heads == 1), "heads have to lie side by side: strides %s" % ((row, head, value),)
    return t.data_ptr(), row if tokens > 1 else heads * dim


_parked = []  # (memory, stream, what it is) of dropped plans that calls on streams which torch knows nothing of may still be using


_unparking = threading.Lock()


def _unpark(stream):
    """Lets go of parked memory ahead of a call on `stream` that waits for the device anyway."""
    with _unparking:
        synchronized = set()
        for i in reversed(range(len(_parked))):  # (more may be parked at the end meanwhile)
            memory, where, kind = _parked[i]
            if kind in (_QUEUE_UNORDERED, _QUEUE_ORDERED):
                if where == stream:  # only its own thread may wait for a queue
                    check(_library().paella_direct_queue_wait(stream), "paella_direct_queue_wait")
                elif where not in _waits or where in _direct_queues:  # (closing a queue waits for it)
                    continue
            elif memory.device not in synchronized:
                torch.cuda.synchronize(memory.device)
                synchronized.add(memory.device)
            del _parked[i]


class _Workspaces:
    """Scratch memory of a plan that starts out zeroed, one per stream, so that calls on different streams do not meet in it.  On a queue that keeps no order, a call that
    finds it in use waits for the queue first.  A call under graph capture gets one of its own in the graph's memory: graphs that were captured from one plan may run at once.
    The stages of a call that is issued stage by stage meet in the workspace of their stream.  Where there is none that both would find, or none that a captured call may have,
    calls are refused without one of the caller's."""

    def __init__(self, nbytes, stages=1):
        self.nbytes = nbytes
        self.stages = stages
        self.of_stream = {}
        self.foreign = {}   # what those streams are that torch did not allocate the workspace for
        self.used = {}      # on queues: how often the queue had been waited for when the workspace was last given out
        self.begun = set()  # where a first stage has been issued and its second has not
        self.lock = threading.RLock()  # held over a call of two launches: another thread's on the same stream would come between them

    def new(self, device):
        return torch.zeros(self.nbytes // 4 + 1, dtype=torch.int32, device=device)

    def given(self, workspace):
        """Address of a caller's workspace."""
        assert workspace.is_contiguous() and workspace.numel() * workspace.element_size() >= self.nbytes, "a workspace of %d bytes is needed, from new_workspace()" % self.nbytes
        _on_device(workspace)
        return workspace.data_ptr()

    def find(self, stream, device, stage=None, explicit=False):
        """The workspace of a call on `stream`, which its caller named (explicit) or not."""
        if not self.nbytes:
            return None
        capturing = torch.cuda.is_current_stream_capturing()
        if not (explicit or capturing) and self.stages == 1 and (device.index, stream) in self.of_stream:
            return self.of_stream[device.index, stream]
        kind = _library().paella_stream_kind_of(stream) if explicit else _STREAM
        # a captured workspace is filled on torch's stream; one that eager calls use must not get into a graph
        if (explicit and stream != _torch_stream()) if capturing else kind == _STREAM_CAPTURING:
            raise AssertionError("a call captured on another stream than torch's has to be given a workspace")
        if capturing:
            if self.stages > 1 and stage is not None:
                raise AssertionError("stages of their own under graph capture have to be given one workspace")
            return self.new(device)
        if self.stages > 1 and ((device.index, stream) in self.begun) != (stage == 1):
            raise AssertionError("a second stage before its first, or a call between the stages of another, on this stream: give each call a workspace of its own")
        w = self.of_stream.get((device.index, stream))
        if w is None:
            with self.lock:
                w = self.of_stream.get((device.index, stream))
                if w is None:
                    w = self.new(device)
                    if stream != _torch_stream():  # the fill ran on torch's stream
                        torch.cuda.current_stream().synchronize()
                        self.foreign[device.index, stream] = kind
                        _unpark(stream)
                    self.of_stream[device.index, stream] = w
        if kind == _QUEUE_UNORDERED:
            if self.used.get((device.index, stream)) == _waits.get(stream, 0):
                check(_library().paella_direct_queue_wait(stream), "paella_direct_queue_wait")
            self.used[device.index, stream] = _waits.get(stream, 0)
        return w

    def __del__(self, park=_parked.append):
        for key, kind in self.foreign.items():
            if key in self.of_stream:
                park((self.of_stream[key], key[1], kind))

    def issued(self, stream, device, stage):
        if stage == 0:
            self.begun.add((device.index, stream))
        elif stage == 1:
            self.begun.discard((device.index, stream))


class KVCache:
    """Keys and values of one layer: two tensors [num_pages, kv_heads, page_size, head_dim] of one type (float32, bfloat16, float16)."""

    def __init__(self, k, v):
        assert k.dtype in _DTYPES and k.dim() == 4 and k.is_contiguous() and k.shape == v.shape and v.dtype == k.dtype and v.is_contiguous() and v.device == k.device
        self.k, self.v = k, v
        self.dtype = k.dtype
        self.num_pages, self.kv_heads, self.page_size, self.head_dim = k.shape
        self.desc = KvCache(k.data_ptr(), v.data_ptr(), _DTYPES[k.dtype], *k.shape)
        self.ref = ctypes.byref(self.desc)
        self.append_descs = {}  # of the calls so far: a model makes a few kinds

    @classmethod
    def empty(cls, num_pages, kv_heads, page_size, head_dim, dtype=torch.float32, device="cuda:0"):
        return cls(*(torch.zeros((num_pages, kv_heads, page_size, head_dim), dtype=dtype, device=device) for _ in range(2)))


class KVBatch:
    """The new tokens of a step.  past: int32 [sequences], own tokens in the cache so far; tables: int32 [sequences, max_pages]; prefix_table: int32, the pages of
    the prefix that all sequences share, prefix_len its tokens.  Every sequence has max_new new tokens, or, with starts (int32 [sequences + 1]), rows starts[b] to
    starts[b + 1] of the `tokens` rows.  The tensors are read at every launch, not here: change them in place."""

    def __init__(self, past, tables, max_new=1, starts=None, tokens=None, prefix_table=None, prefix_len=0):
        assert past.dim() == 1 and tables.dim() == 2 and max_new >= 1
        n = past.shape[0]
        _on_device(past, tables, starts, prefix_table)
        if starts is None:
            assert tokens is None or tokens == n * max_new, "without starts every sequence has max_new tokens"
            tokens = n * max_new
        else:
            assert tokens is not None and tokens >= 1, "the number of rows, which starts alone does not tell the host"
        assert prefix_len >= 0 and (prefix_len == 0 or prefix_table is not None)
        self.past, self.tables, self.starts, self.prefix_table = past, tables, starts, prefix_table
        self.tokens, self.prefix_len = tokens, prefix_len
        self.desc = KvBatch(n, max_new, tokens, tables.shape[1], prefix_len, None if starts is None else _ints(starts, n + 1), _ints(past, n), _ints(tables, n, tables.shape[1]),
                            _ints(prefix_table, prefix_table.numel()) if prefix_len else None)
        self.prefix_pages = prefix_table.numel() if prefix_len else 0
        self.ref = ctypes.byref(self.desc)


def kv_append(cache, batch, k, v, q=None, q_norm=None, k_norm=None, eps=1e-6, inv_freq=None, interleaved=False, out=None, stream=None, job_id=0, notifier=None):
    """Stores the new tokens' k and v ([tokens, kv_heads, head_dim]) in the cache, k normed per head (k_norm: float32 [head_dim]) and rotated (inv_freq: float32, one
    per rotated pair) on the way; returns q ([tokens, heads, head_dim]) normed and rotated likewise, in `out` where given (which may be q)."""
    _on_device(cache.k, k, v, q, q_norm, k_norm, inv_freq, out, batch.past)
    tokens, dim = batch.tokens, cache.head_dim
    kp, ks = _rows(k, tokens, cache.kv_heads, cache)
    vp, vs = _rows(v, tokens, cache.kv_heads, cache)
    heads, qs, qp, op = 0, 0, None, None
    if q is not None:
        heads = q.shape[1]
        qp, qs = _rows(q, tokens, heads, cache)
        if out is None:
            out = q.new_empty((tokens, heads, dim))
        else:
            assert out.shape == (tokens, heads, dim) and out.dtype is q.dtype and out.is_contiguous()
        op = out.data_ptr()
    rotary = 0 if inv_freq is None else 2 * inv_freq.numel()
    desc = cache.append_descs.get((heads, rotary, interleaved, eps, qs, ks, vs))
    if desc is None:
        desc = cache.append_descs[heads, rotary, interleaved, eps, qs, ks, vs] = ctypes.byref(KvAppendDesc(heads, rotary, int(interleaved), eps, qs, ks, vs))
    rc = _library().paella_kv_append_launch(desc, cache.ref, batch.ref, qp, kp, vp, _floats(q_norm, dim), _floats(k_norm, dim), _floats(inv_freq, rotary // 2), op,
                                            _stream(stream), job_id, notifier)
    if rc:
        check(rc, "paella_kv_append_launch")
    return out


class PrefixAttention:
    """Planned attention of a batch: every new token over the shared prefix and its own sequence's tokens up to itself.  The plan holds for every cache and batch of these
    extents (layers, steps); scale: 1 / sqrt(head_dim) unless given.  A call captured on a stream that is not torch's current one has to be given a workspace."""

    def __init__(self, heads, cache, batch, scale=0.0):
        self.lib = _abi.ops()
        self.plan = PrefixAttentionPlan()
        check(self.lib.paella_prefix_attention_plan_make(cache.ref, batch.ref, heads, scale, ctypes.byref(self.plan)), "paella_prefix_attention_plan_make")
        self._ref = ctypes.byref(self.plan)
        self._launch = self.lib.paella_prefix_attention_launch
        self.heads = heads
        self.workspaces = _Workspaces(self.plan.workspace_bytes, self.plan.stages)

    def new_workspace(self, device="cuda"):
        """Scratch memory for one call at a time, zero-filled on the current torch stream; a call leaves it ready for the next."""
        return self.workspaces.new(device)

    def dims(self, stage=0):
        d = LaunchDims()
        check(self.lib.paella_prefix_attention_dims(self._ref, stage, ctypes.byref(d)), "paella_prefix_attention_dims")
        return d

    def __call__(self, q, cache, batch, out=None, stream=None, job_id=0, notifier=None, stage=None, workspace=None):
        """stage: one of the plan's launches (plan.stages) alone, for queues that keep no order.  workspace: one of new_workspace() in place of the stream's own, for calls of one
        plan that may run at once on such a queue.  The stages of a call share it; under graph capture, on different streams, or with other calls of this plan between them
        they have to be given it."""
        _on_device(q, cache.k, out, batch.past)
        assert batch.prefix_pages * cache.page_size >= batch.prefix_len, "the prefix's table has too few pages"
        qp, qs = _rows(q, batch.tokens, self.heads, cache)
        if out is None:
            out = q.new_empty(q.shape)
        else:
            assert out.shape == q.shape and out.dtype is q.dtype and out.is_contiguous()
        explicit, stream = stream is not None, _stream(stream)
        spaces = self.workspaces
        if workspace is not None:
            rc = self._issue(stage, cache, batch, qp, qs, out, spaces.given(workspace), stream, job_id, notifier)
        elif spaces.stages == 1:
            workspace = spaces.find(stream, q.device, stage, explicit)
            rc = self._issue(stage, cache, batch, qp, qs, out, None if workspace is None else workspace.data_ptr(), stream, job_id, notifier)
        else:
            with spaces.lock:
                workspace = spaces.find(stream, q.device, stage, explicit)
                rc = self._issue(stage, cache, batch, qp, qs, out, workspace.data_ptr(), stream, job_id, notifier)
                if stage is not None and not rc:
                    spaces.issued(stream, q.device, stage)
        if rc:
            check(rc, "paella_prefix_attention_launch")
        return out

    def _issue(self, stage, cache, batch, qp, qs, out, workspace, stream, job_id, notifier):
        if stage is None:
            return self._launch(self._ref, cache.ref, batch.ref, qp, qs, out.data_ptr(), workspace, stream, job_id, notifier)
        return self.lib.paella_prefix_attention_launch_stage(self._ref, stage, cache.ref, batch.ref, qp, qs, out.data_ptr(), workspace, stream, job_id, notifier)


class BeamSelect:
    """Planned selection: per group of `beams` beams the `count` best continuations over the vocabulary."""

    def __init__(self, groups, beams, vocab, count, dtype=torch.float32):
        self.lib = _abi.ops()
        self.plan = BeamSelectPlan()
        assert dtype in _DTYPES, dtype
        check(self.lib.paella_beam_select_plan_make(_DTYPES[dtype], groups, beams, vocab, count, ctypes.byref(self.plan)), "paella_beam_select_plan_make")
        self._ref = ctypes.byref(self.plan)
        self._launch = self.lib.paella_beam_select_launch
        self.dtype, self.shape, self.count = dtype, (groups, beams, vocab), count
        self.workspaces = _Workspaces(self.plan.workspace_bytes)

    def dims(self):
        d = LaunchDims()
        check(self.lib.paella_beam_select_dims(self._ref, ctypes.byref(d)), "paella_beam_select_dims")
        return d

    def new_workspace(self, device="cuda"):
        """As PrefixAttention.new_workspace."""
        return self.workspaces.new(device)

    def __call__(self, logits, scores, finished=None, pad_token=0, stream=None, job_id=0, notifier=None, workspace=None):
        """logits [groups, beams, vocab] (beams one after the other, rows of any stride), scores float32 [groups, beams], finished uint8 or bool [groups, beams].  Returns scores
        (float32), parents and tokens (int32), each [groups, count], best first.  workspace: one of new_workspace() in place of the stream's own, for calls of one plan that may run
        at once on a queue that keeps no order."""
        _on_device(logits, scores, finished)
        groups, beams, vocab = self.shape
        assert logits.dtype == self.dtype and tuple(logits.shape) == self.shape, (logits.dtype, tuple(logits.shape))
        row = logits.stride(1) if beams > 1 else logits.stride(0) if groups > 1 else vocab
        assert (vocab == 1 or logits.stride(2) == 1) and (groups == 1 or beams == 1 or logits.stride(0) == beams * row), "rows have to be one stride apart: %s" % (logits.stride(),)
        if finished is not None:
            assert finished.dtype in (torch.uint8, torch.bool) and finished.is_contiguous() and finished.numel() == groups * beams
            finished = finished.data_ptr()
        shape = (groups, self.count)
        out, parents, tokens = scores.new_empty(shape), scores.new_empty(shape, dtype=torch.int32), scores.new_empty(shape, dtype=torch.int32)
        explicit, stream = stream is not None, _stream(stream)
        if workspace is None:
            workspace = self.workspaces.find(stream, logits.device, None, explicit)
            address = workspace.data_ptr()
        else:
            address = self.workspaces.given(workspace)
        rc = self._launch(self._ref, logits.data_ptr(), row, _floats(scores, groups * beams), finished, pad_token, out.data_ptr(), parents.data_ptr(), tokens.data_ptr(),
                          address, stream, job_id, notifier)
        if rc:
            check(rc, "paella_beam_select_launch")
        return out, parents, tokens


def beam_reorder(cache, parents, past, tables, tables_out, spare, past_out=None, stream=None, job_id=0, notifier=None):
    """Gives each child beam (parents: int32 [groups, count]) its parent's tokens: rows of tables_out name the parent's full pages and the page of the next token, copied to a
    spare page (spare: int32, one per child) for every child of a parent but its first.  Returns the children's lengths (past_out).  tables: int32 [groups * beams, max_pages]."""
    _on_device(cache.k, parents, past, tables, tables_out, spare, past_out)
    assert parents.dim() == 2 and tables.dim() == 2
    groups, count = parents.shape
    rows, pages = tables.shape
    assert rows % groups == 0 and spare.numel() == groups * count, (rows, groups, spare.numel())
    if past_out is None:
        past_out = past.new_empty(groups * count)
    desc = BeamReorderDesc(groups, rows // groups, count, pages)
    rc = _library().paella_beam_reorder_launch(ctypes.byref(desc), cache.ref, _ints(parents, groups, count), _ints(past, rows), _ints(tables, rows, pages),
                                        _ints(spare, *spare.shape), _ints(tables_out, groups * count, pages), _ints(past_out, groups * count), _stream(stream), job_id,
                                        notifier)
    if rc:
        check(rc, "paella_beam_reorder_launch")
    return past_out
