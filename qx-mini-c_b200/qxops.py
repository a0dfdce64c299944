"""The device operators of include/qx_cuda.h for torch tensors.

Like qxlib, nothing here computes: every function hands its tensors to the
native module (csrc/qx_torch.cpp), which checks them and makes one C-ABI call
on their memory, queued on the current stream of their device.  Outputs that
are not given are allocated (and outputs that a call may leave in part
unwritten, zeroed); the scratch of a call comes from torch's allocator.  What
the checks refuse raises ValueError, what the library refuses RuntimeError with
its message.  The operators have no backward pass: where gradients are recorded
(outside torch.no_grad()), tensors that require one are refused.
"""
import ctypes as C

import numpy as np
import torch

import qxlib

qxlib.cuda()              # libqxcuda.so, or a message that says how to build it
try:
    import _qxops as _native
except ImportError as e:
    raise RuntimeError("_qxops.so is not built (run make all qxops in %s)" % qxlib.HERE) from e

STATUS_RANGE = 0x1        # a sequence's slot, length or nodes lie outside the cache
STATUS_SHARED = 0x2       # a slot written by a call is also another sequence's
STATUS_TIMEOUT = 0x4      # a kernel's internal wait ran out: outputs are incomplete

ROPE_SCHEMES = {"none": 0, "linear": 1, "ntk": 2, "yarn": 3, "bands": 4}


class _Cache(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in ("k", "v", "k_scales", "v_scales")] + [
        ("slot_rows", C.c_uint64), ("layer_rows", C.c_uint64)] + [
        (n, C.c_uint32) for n in ("slots", "layers", "ctx_tokens", "kv_heads", "head_dim", "reserved")]


_signed = False


def _cuda():
    """libqxcuda.so with the signatures of the entry points that are called without tensors."""
    global _signed
    lib = qxlib.cuda()
    if not _signed:
        P, U32, U64, D, E = C.c_void_p, C.c_uint32, C.c_uint64, C.c_double, C.c_char_p
        for name, args in {"qx_cuda_kv_view": [P, U32, P, E, U64],
                           "qx_cuda_rope_frequencies": [U32, U32, D, D, D, D, D, P, P, E, U64]}.items():
            fn = getattr(lib, name)
            fn.argtypes = args
            fn.restype = C.c_int
        _signed = True
    return lib


def _call(fn, *args):
    err = C.create_string_buffer(256)
    if not fn(*args, err, 256):
        raise RuntimeError("%s failed: %s" % (fn.__name__, err.value.decode(errors="replace")))


def _device_of(address):
    """The CUDA ordinal of the device that holds an address."""
    n = C.c_int()
    code = C.CDLL("libcuda.so.1").cuPointerGetAttribute(C.byref(n), 9, C.c_uint64(address))      # CU_POINTER_ATTRIBUTE_DEVICE_ORDINAL
    if code:
        raise RuntimeError("cuPointerGetAttribute failed: %d" % code)
    return n.value


class KvCache:
    """A handle on an INT8 cache (qx_cuda_kv_cache): k, v int8
    [slots][layers][ctx][kv_heads][head_dim] and k_scales, v_scales float32
    [slots][layers][ctx], rows contiguous, slots and layers at any stride that
    codes and scales share.  Holds the tensors."""

    def __init__(self, k, v, k_scales, v_scales):
        slots, layers, ctx, kvh, hd = k.shape
        row = kvh * hd
        for t, name in ((k, "k"), (v, "v")):
            if t.dtype is not torch.int8 or t.shape != k.shape or t.device != k.device or t.stride() != k.stride():
                raise ValueError("%s must be an int8 tensor like k" % name)
        for t, name in ((k_scales, "k_scales"), (v_scales, "v_scales")):
            if t.dtype is not torch.float32 or t.shape != k.shape[:3] or t.device != k.device or (ctx > 1 and t.stride(2) != 1):
                raise ValueError("%s must be a float32 tensor of shape %s" % (name, tuple(k.shape[:3])))
        if (hd > 1 and k.stride(4) != 1) or (kvh > 1 and k.stride(3) != hd) or (ctx > 1 and k.stride(2) != row):
            raise ValueError("the rows of a cache must be contiguous")
        step = [0, 0]
        for dim, many in ((0, slots), (1, layers)):
            if many > 1:
                if k.stride(dim) % row or any(t.stride(dim) * row != k.stride(dim) for t in (k_scales, v_scales)):
                    raise ValueError("codes and scales must have the same layout")
                step[dim] = k.stride(dim) // row
        self.k, self.v, self.k_scales, self.v_scales = k, v, k_scales, v_scales
        self.device = k.device
        self.slots, self.layers, self.ctx, self.kv_heads, self.head_dim = slots, layers, ctx, kvh, hd
        self.c = _Cache(k.data_ptr(), v.data_ptr(), k_scales.data_ptr(), v_scales.data_ptr(), step[0], step[1], slots,
                        layers, ctx, kvh, hd, 0)
        self.handle = (C.addressof(self.c), k.device.index if k.is_cuda else -1)


class EngineCache:
    """The same handle on an engine's own cache (qx_cuda_kv_view): its
    single-sequence cache, or with batch=True the slots of decode_batch.
    Calls are refused once the engine is closed; order them after the engine's own work
    (Engine.stream()).  device, if given, must be the engine's."""

    def __init__(self, engine, batch=False, device=None):
        if not engine.h:
            raise ValueError("the engine is closed")
        self.c = _Cache()
        _call(_cuda().qx_cuda_kv_view, engine.h, 1 if batch else 0, C.byref(self.c))
        self.engine = engine
        self.device = torch.device("cuda", _device_of(self.c.k))
        if device is not None and torch.device("cuda", device) != self.device:
            raise ValueError("the engine's cache is on %s" % self.device)
        self._handle = (C.addressof(self.c), self.device.index)
        self.slots, self.layers, self.ctx = self.c.slots, self.c.layers, self.c.ctx_tokens
        self.kv_heads, self.head_dim = self.c.kv_heads, self.c.head_dim

    @property
    def handle(self):
        if not self.engine.h:
            raise ValueError("the engine of this cache is closed")
        return self._handle


def rope_frequencies(rotary_dim, base=1e6, scheme="none", factor=1.0, original_ctx=4096, low=1.0, high=32.0):
    """(inv_freq float64 [rotary_dim / 2], amplitude) of a context-extension
    scheme: none, linear, ntk, yarn or bands (qx_cuda_rope_frequencies)."""
    out = np.zeros(max(1, rotary_dim // 2), np.float64)
    amp = C.c_double()
    _call(_cuda().qx_cuda_rope_frequencies, ROPE_SCHEMES[scheme], rotary_dim, base, factor, original_ctx, low, high,
          out.ctypes.data, C.byref(amp))
    return out, amp.value


def rope_append(cache, layer, slots, lens, q, k, v, inv_freq, positions=None, nodes=None, interleaved=False, factor=1.0,
                q_out=None, status=None, mass=None):
    """Rotate drafted tokens and append their keys and values
    (qx_cuda_rope_append_mass).  q [seqs][nodes][q_heads][head_dim], k and v
    [seqs][nodes][kv_heads][head_dim] of one float type (q, or k and v, may be
    None); inv_freq float64 on the device, factor the amplitude; mass (like the
    cache's scales) becomes 0 for the appended rows.  Returns the
    rotated queries (q_out; q itself rotates in place)."""
    return _native.rope_append(cache.handle, layer, slots, lens, q, k, v, inv_freq, positions, nodes, interleaved, factor, q_out,
                               status, mass)


def tree_attention(cache, layer, slots, lens, q, nodes=None, mask=None, scale=None, out=None, lse=None, mass=None,
                   status=None):
    """Attention of drafted tokens over the cache (qx_cuda_tree_attention).
    q [seqs][nodes][q_heads][head_dim]; mask int64 [seqs][nodes][words] of
    visibility bits, None for a chain; scale None: head_dim ** -0.5; lse
    float32 [seqs][nodes][q_heads] and mass (like the cache's scales) are
    written where given.  out may be q itself where mass is not given.  Returns
    out (like q)."""
    return _native.tree_attention(cache.handle, layer, slots, lens, q, nodes, mask, scale, out, lse, mass, status)


def tree_mask(parents):
    """Visibility bits of trees given by parents (int64 host array
    [seqs][nodes]; -1: the last committed row), int64 [seqs][nodes][words] on
    the host: a node sees itself and its ancestors, which come before it."""
    parents = np.asarray(parents, np.int64)
    seqs, n = parents.shape
    bits = np.zeros((seqs, n, (n + 63) // 64), np.uint64)
    for s in range(seqs):
        for i in range(n):
            p = int(parents[s, i])
            if not -1 <= p < i:
                raise ValueError("a node's parent comes before it")
            if p >= 0:
                bits[s, i] = bits[s, p]
            bits[s, i, i // 64] |= np.uint64(1) << np.uint64(i % 64)
    return torch.from_numpy(bits.view(np.int64))


def evict(cache, slots, lens, mass, budget, sink=0, recent=0, dst_slots=None, kept=None, new_lens=None, status=None):
    """Evict rows by accumulated attention weight in every layer
    (qx_cuda_kv_evict); in place unless dst_slots is given.  Returns (kept int32
    [layers][seqs][budget], new_lens int32 [seqs])."""
    return _native.evict(cache.handle, slots, lens, mass, budget, sink, recent, dst_slots, kept, new_lens, status)


def pick_tokens(logits, history=None, history_lens=None, repetition=None, frequency=None, presence=None, bias_ids=None,
                bias_values=None, bias_lens=None, allowed=None, out=None, picked=None):
    """Penalties, biases, grammar mask and greedy token of each row
    (qx_cuda_pick_tokens).  logits [rows][vocab]; history int32 [rows][...];
    repetition, frequency, presence float32 [rows]; bias_ids int32 and
    bias_values float32 [rows][...]; allowed int32 [rows][(vocab + 31) / 32] of
    bits.  Returns (adjusted logits, int32 tokens, -1 where a row has none); out may be logits."""
    return _native.pick_tokens(logits, history, history_lens, repetition, frequency, presence, bias_ids, bias_values, bias_lens,
                               allowed, out, picked)
