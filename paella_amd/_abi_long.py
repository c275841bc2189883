"""ctypes declarations for include/paella_long_cache.h."""
import ctypes

from ._abi_decode import KvBatch, KvCache
from ._abi_types import LaunchDims

c_int, c_float, c_double, c_void_p, c_size_t, c_u32, c_i64 = (ctypes.c_int, ctypes.c_float, ctypes.c_double, ctypes.c_void_p, ctypes.c_size_t,
                                                              ctypes.c_uint32, ctypes.c_int64)

_EXTENTS = [(n, c_int) for n in ("dtype", "heads", "kv_heads", "head_dim", "page_size", "sequences", "max_new", "tokens", "max_pages", "prefix_len")]
_COSTS = [("workspace_bytes", c_size_t), ("zero_bytes", c_size_t), ("dims", LaunchDims), ("flops", c_double), ("bytes", c_double)]


class PageSelectPlan(ctypes.Structure):
    _fields_ = _EXTENTS + [(n, c_int) for n in ("count", "first", "last", "splits", "stages")] + _COSTS


class PageAttentionPlan(ctypes.Structure):
    _fields_ = _EXTENTS + [("count", c_int), ("scale", c_float), ("splits", c_int), ("stages", c_int)] + _COSTS


class KeyWeightsPlan(ctypes.Structure):
    _fields_ = _EXTENTS + [("scale", c_float)] + [(n, c_int) for n in ("splits", "own_splits", "stages")] + _COSTS


class KvEvictDesc(ctypes.Structure):
    _fields_ = [(n, c_int) for n in ("sequences", "max_pages", "keep", "first", "recent")]


_p = ctypes.POINTER
_TAIL = [c_void_p, c_u32, c_void_p]  # stream, job_id, notifier


def _planned(name, plan, made_from, operands):
    """The entry points of a plan: make(cache, batch, ...), dims(stage), launch and launch_stage with the operands behind cache and batch."""
    return {
        "paella_%s_plan_make" % name: (c_int, [_p(KvCache), _p(KvBatch)] + made_from + [_p(plan)]),
        "paella_%s_dims" % name: (c_int, [_p(plan), c_int, _p(LaunchDims)]),
        "paella_%s_launch" % name: (c_int, [_p(plan), _p(KvCache), _p(KvBatch)] + operands + _TAIL),
        "paella_%s_launch_stage" % name: (c_int, [_p(plan), c_int, _p(KvCache), _p(KvBatch)] + operands + _TAIL),
    }


LONG_SYMBOLS = {
    "paella_page_bounds_dims": (c_int, [_p(KvCache), _p(KvBatch), _p(LaunchDims)]),
    "paella_page_bounds_launch": (c_int, [_p(KvCache), _p(KvBatch), c_void_p] + _TAIL),
    **_planned("page_select", PageSelectPlan, [c_int] * 4, [c_void_p, c_i64] + [c_void_p] * 3),        # q, stride, bounds, pages, workspace
    **_planned("page_attention", PageAttentionPlan, [c_int, c_int, c_float], [c_void_p, c_i64] + [c_void_p] * 3),  # q, stride, pages, out, workspace
    **_planned("key_weights", KeyWeightsPlan, [c_int, c_float], [c_void_p, c_i64] + [c_void_p] * 2),   # q, stride, weights, workspace
    "paella_kv_evict_dims": (c_int, [_p(KvEvictDesc), _p(KvCache), c_int, _p(LaunchDims)]),
    "paella_kv_evict_launch": (c_int, [_p(KvEvictDesc), _p(KvCache)] + [c_void_p] * 5 + _TAIL),
    "paella_kv_evict_launch_stage": (c_int, [_p(KvEvictDesc), c_int, _p(KvCache)] + [c_void_p] * 5 + _TAIL),
}


def bind(lib):
    for name, (res, args) in LONG_SYMBOLS.items():
        fn = getattr(lib, name)
        fn.restype = res
        fn.argtypes = args
    return lib
