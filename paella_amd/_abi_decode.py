"""ctypes declarations for include/paella_decode.h."""
import ctypes

from ._abi_types import LaunchDims

c_int, c_float, c_double, c_void_p, c_size_t, c_u32, c_i64 = (ctypes.c_int, ctypes.c_float, ctypes.c_double, ctypes.c_void_p, ctypes.c_size_t,
                                                              ctypes.c_uint32, ctypes.c_int64)
F32, BF16, F16 = range(3)


class KvCache(ctypes.Structure):
    _fields_ = [("k", c_void_p), ("v", c_void_p)] + [(n, c_int) for n in ("dtype", "num_pages", "kv_heads", "page_size", "head_dim")]


class KvBatch(ctypes.Structure):
    _fields_ = [(n, c_int) for n in ("sequences", "max_new", "tokens", "max_pages", "prefix_len")] + \
               [(n, c_void_p) for n in ("starts", "past", "tables", "prefix_table")]


class KvAppendDesc(ctypes.Structure):
    _fields_ = [(n, c_int) for n in ("heads", "rotary_dim", "interleaved")] + [("eps", c_float)] + [(n, c_i64) for n in ("q_stride", "k_stride", "v_stride")]


class PrefixAttentionPlan(ctypes.Structure):
    _fields_ = [(n, c_int) for n in ("dtype", "heads", "kv_heads", "head_dim", "page_size", "sequences", "max_new", "tokens", "max_pages", "prefix_len")] + \
               [("scale", c_float)] + [(n, c_int) for n in ("prefix_rows", "own_rows", "prefix_splits", "own_splits", "stages")] + \
               [("workspace_bytes", c_size_t), ("dims", LaunchDims), ("flops", c_double), ("bytes", c_double)]


class BeamSelectPlan(ctypes.Structure):
    _fields_ = [(n, c_int) for n in ("dtype", "groups", "beams", "vocab", "count", "values", "splits")] + \
               [("workspace_bytes", c_size_t), ("dims", LaunchDims), ("flops", c_double), ("bytes", c_double)]


class BeamReorderDesc(ctypes.Structure):
    _fields_ = [(n, c_int) for n in ("groups", "beams", "count", "max_pages")]


_p = ctypes.POINTER
_TAIL = [c_void_p, c_u32, c_void_p]  # stream, job_id, notifier

DECODE_SYMBOLS = {
    "paella_kv_append_dims": (c_int, [_p(KvAppendDesc), _p(KvCache), _p(KvBatch), _p(LaunchDims)]),
    "paella_kv_append_launch": (c_int, [_p(KvAppendDesc), _p(KvCache), _p(KvBatch)] + [c_void_p] * 7 + _TAIL),
    "paella_kv_append_at_launch": (c_int, [_p(KvAppendDesc), _p(KvCache), _p(KvBatch)] + [c_void_p] * 8 + _TAIL),
    "paella_prefix_attention_plan_make": (c_int, [_p(KvCache), _p(KvBatch), c_int, c_float, _p(PrefixAttentionPlan)]),
    "paella_prefix_attention_dims": (c_int, [_p(PrefixAttentionPlan), c_int, _p(LaunchDims)]),
    "paella_prefix_attention_launch_stage": (c_int, [_p(PrefixAttentionPlan), c_int, _p(KvCache), _p(KvBatch), c_void_p, c_i64, c_void_p, c_void_p] + _TAIL),
    "paella_prefix_attention_launch": (c_int, [_p(PrefixAttentionPlan), _p(KvCache), _p(KvBatch), c_void_p, c_i64, c_void_p, c_void_p] + _TAIL),
    "paella_beam_select_plan_make": (c_int, [c_int] * 5 + [_p(BeamSelectPlan)]),
    "paella_beam_select_dims": (c_int, [_p(BeamSelectPlan), _p(LaunchDims)]),
    "paella_beam_select_launch": (c_int, [_p(BeamSelectPlan), c_void_p, c_i64, c_void_p, c_void_p, c_int] + [c_void_p] * 4 + _TAIL),
    "paella_beam_reorder_dims": (c_int, [_p(BeamReorderDesc), _p(KvCache), _p(LaunchDims)]),
    "paella_beam_reorder_launch": (c_int, [_p(BeamReorderDesc), _p(KvCache)] + [c_void_p] * 6 + _TAIL),
}


def bind(lib):
    for name, (res, args) in DECODE_SYMBOLS.items():
        fn = getattr(lib, name)
        fn.restype = res
        fn.argtypes = args
    return lib
