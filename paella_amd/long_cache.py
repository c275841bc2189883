"""Functional front-end over the operators that keep a long paged cache from being read whole and from being kept whole (include/paella_long_cache.h).

Conventions as in `decode`, whose caches and batches these work on.  A step that reads the pages that matter:

    bounds = new_bounds(cache)                                       # one per layer
    select = PageSelect(heads, cache, batch, count=64, first=1, last=2)
    attend = PageAttention(heads, cache, batch, count=64)
    q = decode.kv_append(cache, batch, k, v, q=q, inv_freq=freq)     # per layer
    page_bounds(cache, bounds, batch)
    out = attend(q, cache, batch, select(q, bounds, cache, batch))

And a cache that keeps the tokens that attention went to:

    weights = new_weights(cache, batch)
    weigh, evict = KeyWeights(heads, cache, batch), Evict(cache, sequences, max_pages, keep=4096, first=4, recent=256)
    weigh(q, cache, batch, weights)                                  # after the append of a prompt's last tokens, or of every token
    past, kept = evict(cache, weights, past, tables)                 # later tokens: kv_append(..., positions=theirs); the pages' bounds anew
"""
import ctypes

import torch

from . import _abi
from ._abi import LaunchDims, check
from ._abi_long import KeyWeightsPlan, KvEvictDesc, PageAttentionPlan, PageSelectPlan
from .decode import _Workspaces, _floats, _ints, _library, _on_device, _rows
from .ops import _stream


def new_bounds(cache):
    """Room for the bounds of all pages of a cache: [num_pages, kv_heads, 2, head_dim] of its type, least values and then largest."""
    return cache.k.new_zeros((cache.num_pages, cache.kv_heads, 2, cache.head_dim))


def new_weights(cache, batch):
    """Room for the weights of the own tokens of a batch's sequences: float32 [sequences, kv_heads, max_pages * page_size]."""
    return torch.zeros((batch.past.shape[0], cache.kv_heads, batch.tables.shape[1] * cache.page_size), dtype=torch.float32, device=cache.k.device)


def _bounds(t, cache):
    assert t.dtype is cache.dtype and t.shape == (cache.num_pages, cache.kv_heads, 2, cache.head_dim) and t.is_contiguous(), (t.dtype, tuple(t.shape))
    return t.data_ptr()


def _weights(t, cache, sequences, max_pages):
    assert t.shape == (sequences, cache.kv_heads, max_pages * cache.page_size), (tuple(t.shape), "wanted", (sequences, cache.kv_heads, max_pages * cache.page_size))
    return _floats(t, t.numel())


def page_bounds(cache, bounds, batch, stream=None, job_id=0, notifier=None):
    """Makes the bounds (of new_bounds) of every page that a new token of the batch lies in anew, from all of the page's tokens up to the last new one.  Returns them."""
    _on_device(cache.k, bounds, batch.past)
    rc = _library().paella_page_bounds_launch(cache.ref, batch.ref, _bounds(bounds, cache), _stream(stream), job_id, notifier)
    if rc:
        check(rc, "paella_page_bounds_launch")
    return bounds


class _Planned:
    """What plans over a cache and a batch have in common.  A plan holds for every cache and batch of its extents (layers, steps)."""

    def __init__(self, name, plan, cache, batch, *args):
        self.lib = _abi.ops()
        self.plan = plan
        self._ref = ctypes.byref(plan)
        self._name = "paella_%s_launch" % name
        check(getattr(self.lib, "paella_%s_plan_make" % name)(cache.ref, batch.ref, *args, self._ref), "paella_%s_plan_make" % name)
        self._dims = getattr(self.lib, "paella_%s_dims" % name)
        self._whole, self._stage = getattr(self.lib, self._name), getattr(self.lib, self._name + "_stage")
        self.workspaces = _Workspaces(plan.workspace_bytes, plan.stages, plan.zero_bytes)

    def new_workspace(self, device="cuda"):
        """Scratch memory for one call at a time of this plan, made ready (plan.zero_bytes of it zeroed) on the current torch stream; a call leaves it ready for the next."""
        return self.workspaces.new(device)

    def dims(self, stage=0):
        d = LaunchDims()
        check(self._dims(self._ref, stage, ctypes.byref(d)), self._name[:-6] + "dims")
        return d

    def _queries(self, q, cache, batch):
        assert batch.prefix_pages * cache.page_size >= batch.prefix_len, "the prefix's table has too few pages"
        return _rows(q, batch.tokens, self.plan.heads, cache)

    def _issue(self, cache, batch, operands, stream, job_id, notifier, stage, workspace):
        """One call, or one of its stages.  As in decode.PrefixAttention: the stages of a call share a workspace, a stream has one unless the caller gives one."""
        explicit, stream = stream is not None, _stream(stream)
        spaces, device = self.workspaces, cache.k.device

        def launch(space):
            if stage is None:
                return self._whole(self._ref, cache.ref, batch.ref, *operands, space, stream, job_id, notifier)
            return self._stage(self._ref, stage, cache.ref, batch.ref, *operands, space, stream, job_id, notifier)

        if workspace is not None:
            rc = launch(spaces.given(workspace))
        elif spaces.stages == 1:
            workspace = spaces.find(stream, device, stage, explicit)
            rc = launch(None if workspace is None else workspace.data_ptr())
        else:
            with spaces.lock:
                workspace = spaces.find(stream, device, stage, explicit)
                rc = launch(workspace.data_ptr())
                if stage is not None and not rc:
                    spaces.issued(stream, device, stage)
        if rc:
            check(rc, self._name)


class PageSelect(_Planned):
    """Planned selection of the `count` pages that each new token reads, for each key head: its sequence's first `first` and last `last` visible pages and those whose
    bounds allow the largest products with the key head's queries.  Pages are counted along a sequence, the shared prefix's first."""

    def __init__(self, heads, cache, batch, count, first=0, last=1):
        super().__init__("page_select", PageSelectPlan(), cache, batch, heads, count, first, last)

    def __call__(self, q, bounds, cache, batch, out=None, stream=None, job_id=0, notifier=None, stage=None, workspace=None):
        """q [tokens, heads, head_dim]; returns int32 [tokens, kv_heads, count], ascending, -1 behind the last (in `out` where given).  stage, workspace: as decode.PrefixAttention;
        the stages of a call have to be given the same `out`."""
        _on_device(q, cache.k, bounds, out, batch.past)
        qp, qs = self._queries(q, cache, batch)
        shape = (batch.tokens, cache.kv_heads, self.plan.count)
        if out is None:
            assert stage is None, "stages have to be given their output"
            out = batch.past.new_empty(shape)
        self._issue(cache, batch, (qp, qs, _bounds(bounds, cache), _ints(out, *shape)), stream, job_id, notifier, stage, workspace)
        return out


class PageAttention(_Planned):
    """Planned attention of each new token over the pages that are listed for it and its key head, `count` at most; scale: 1 / sqrt(head_dim) unless given."""

    def __init__(self, heads, cache, batch, count, scale=0.0):
        super().__init__("page_attention", PageAttentionPlan(), cache, batch, heads, count, scale)

    def __call__(self, q, cache, batch, pages, out=None, stream=None, job_id=0, notifier=None, stage=None, workspace=None):
        """q [tokens, heads, head_dim], pages int32 [tokens, kv_heads, count] as PageSelect returns them; returns the outputs, of q's shape.  stage, workspace: as decode.PrefixAttention."""
        _on_device(q, cache.k, pages, out, batch.past)
        qp, qs = self._queries(q, cache, batch)
        if out is None:
            out = q.new_empty(q.shape)
        else:
            assert out.shape == q.shape and out.dtype is q.dtype and out.is_contiguous()
        self._issue(cache, batch, (qp, qs, _ints(pages, batch.tokens, cache.kv_heads, self.plan.count), out.data_ptr()), stream, job_id, notifier, stage, workspace)
        return out


class KeyWeights(_Planned):
    """Planned sums of the attention weights that the new tokens of a batch give to the own tokens of their sequences; scale: 1 / sqrt(head_dim) unless given."""

    def __init__(self, heads, cache, batch, scale=0.0):
        super().__init__("key_weights", KeyWeightsPlan(), cache, batch, heads, scale)

    def __call__(self, q, cache, batch, weights, stream=None, job_id=0, notifier=None, stage=None, workspace=None):
        """Adds to weights (of new_weights; new tokens' places are begun at 0) and returns them.  The new tokens' keys have to be in the cache.  stage, workspace: as decode.PrefixAttention."""
        _on_device(q, cache.k, weights, batch.past)
        qp, qs = self._queries(q, cache, batch)
        at = _weights(weights, cache, batch.past.shape[0], batch.tables.shape[1])
        self._issue(cache, batch, (qp, qs, at), stream, job_id, notifier, stage, workspace)
        return weights


class Evict:
    """Eviction: of each sequence that is longer, every key head keeps `keep` tokens -- its first `first`, its last `recent` and the heaviest between -- which move to the sequence's
    first places, in order."""

    stages = 2

    def __init__(self, cache, sequences, max_pages, keep, first=0, recent=0):
        self.lib = _abi.ops()
        self.desc = KvEvictDesc(sequences, max_pages, keep, first, recent)
        self._ref = ctypes.byref(self.desc)
        d = LaunchDims()
        check(self.lib.paella_kv_evict_dims(self._ref, cache.ref, 0, ctypes.byref(d)), "paella_kv_evict_dims")

    def dims(self, cache, stage=0):
        d = LaunchDims()
        check(self.lib.paella_kv_evict_dims(self._ref, cache.ref, stage, ctypes.byref(d)), "paella_kv_evict_dims")
        return d

    def __call__(self, cache, weights, past, tables, past_out=None, kept=None, stream=None, job_id=0, notifier=None, stage=None):
        """weights: of new_weights, moved along; past: int32 [sequences], own tokens in the cache; tables: int32 [sequences, max_pages], no page twice.  Returns the lengths (in past_out
        where given, which may be past) and which tokens stayed, int32 [sequences, kv_heads, keep], -1 behind a shorter sequence's last.  stage: one of the two launches alone, for queues that keep
        no order; both have to be given the same past_out and kept."""
        _on_device(cache.k, weights, past, tables, past_out, kept)
        d = self.desc
        at = _weights(weights, cache, d.sequences, d.max_pages)
        assert stage is None or (past_out is not None and kept is not None), "stages have to be given their outputs"
        if past_out is None:
            past_out = past.new_empty(d.sequences)
        shape = (d.sequences, cache.kv_heads, d.keep)
        if kept is None:
            kept = past.new_empty(shape)
        args = (cache.ref, at, _ints(past, d.sequences), _ints(tables, d.sequences, d.max_pages), _ints(kept, *shape), _ints(past_out, d.sequences), _stream(stream), job_id, notifier)
        rc = self.lib.paella_kv_evict_launch(self._ref, *args) if stage is None else self.lib.paella_kv_evict_launch_stage(self._ref, stage, *args)
        if rc:
            check(rc, "paella_kv_evict_launch")
        return past_out, kept
