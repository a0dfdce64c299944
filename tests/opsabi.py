"""ctypes mirrors of the device operators' structs and signatures (include/qx_cuda.h), for tests that call the C ABI itself."""
import ctypes as C

import qxlib
from qxops import _Cache as Cache  # noqa: F401


class Drafts(C.Structure):
    _fields_ = [("seqs", C.c_uint32), ("max_nodes", C.c_uint32)] + [(n, C.c_void_p) for n in ("slots", "lens", "nodes")]


class Heads(C.Structure):
    _fields_ = [("data", C.c_void_p)] + [(n, C.c_uint64) for n in ("seq_stride", "node_stride", "head_stride")]


class Rotary(C.Structure):
    _fields_ = [("inv_freq", C.c_void_p), ("amplitude", C.c_double), ("rotary_dim", C.c_uint32), ("interleaved", C.c_uint32)]


class Pick(C.Structure):
    _fields_ = [("logits", C.c_void_p), ("out", C.c_void_p), ("logits_stride", C.c_uint64), ("out_stride", C.c_uint64)] + [
        (n, C.c_uint32) for n in ("rows", "vocab", "dtype", "max_history", "max_bias", "reserved")] + [
        (n, C.c_void_p) for n in ("history", "history_lens", "repetition", "frequency", "presence", "bias_ids", "bias_lens",
                                  "bias_values", "allowed")] + [
        (n, C.c_uint64) for n in ("history_stride", "bias_stride", "allowed_stride")] + [("picked", C.c_void_p)]


def lib():
    so = qxlib.cuda()
    P, U32, U64, D, E = C.c_void_p, C.c_uint32, C.c_uint64, C.c_double, C.c_char_p
    for name, args in {
            "qx_cuda_kv_view": [P, U32, P, E, U64],
            "qx_cuda_rope_frequencies": [U32, U32, D, D, D, D, D, P, P, E, U64],
            "qx_cuda_rope_append": [P, U32, P, P, U32, U32, P, P, P, P, P, P, P, E, U64],
            "qx_cuda_tree_attention": [P, U32, P, U32, U32, P, P, P, C.c_float, P, P, P, U64, P, P, E, U64],
            "qx_cuda_tree_attention_workspace": [U32, U32, U32, U32, U32, U32, P, E, U64],
            "qx_cuda_kv_evict": [P, U32, P, P, P, P, U32, U32, U32, P, P, P, P, E, U64],
            "qx_cuda_pick_tokens": [P, P, E, U64]}.items():
        fn = getattr(so, name)
        fn.argtypes = args
        fn.restype = C.c_int
    return so
