"""The device operators of include/qx_cuda.h for torch tensors.

Like qxlib, nothing here computes: every function checks what it was given and
makes one C-ABI call on the tensors' memory, queued on the current stream of
their device.  Outputs that are not given are allocated (and outputs that a
call may leave in part unwritten, zeroed).  A refused argument raises, with
the library's message.
"""
import ctypes as C

import numpy as np
import torch

import qxlib

_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}

STATUS_RANGE = 0x1        # a sequence's slot, length or nodes lie outside the cache
STATUS_SHARED = 0x2       # a slot written by a call is also another sequence's

ROPE_SCHEMES = {"none": 0, "linear": 1, "ntk": 2, "yarn": 3, "bands": 4}


class _Cache(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in ("k", "v", "k_scales", "v_scales")] + [
        ("slot_rows", C.c_uint64), ("layer_rows", C.c_uint64)] + [
        (n, C.c_uint32) for n in ("slots", "layers", "ctx_tokens", "kv_heads", "head_dim", "reserved")]


class _Drafts(C.Structure):
    _fields_ = [("seqs", C.c_uint32), ("max_nodes", C.c_uint32)] + [(n, C.c_void_p) for n in ("slots", "lens", "nodes")]


class _Heads(C.Structure):
    _fields_ = [("data", C.c_void_p)] + [(n, C.c_uint64) for n in ("seq_stride", "node_stride", "head_stride")]


class _Rotary(C.Structure):
    _fields_ = [("inv_freq", C.c_void_p), ("amplitude", C.c_double), ("rotary_dim", C.c_uint32), ("interleaved", C.c_uint32)]


class _Pick(C.Structure):
    _fields_ = [("logits", C.c_void_p), ("out", C.c_void_p), ("logits_stride", C.c_uint64), ("out_stride", C.c_uint64)] + [
        (n, C.c_uint32) for n in ("rows", "vocab", "dtype", "max_history", "max_bias", "reserved")] + [
        (n, C.c_void_p) for n in ("history", "history_lens", "repetition", "frequency", "presence", "bias_ids", "bias_lens",
                                  "bias_values", "allowed")] + [
        (n, C.c_uint64) for n in ("history_stride", "bias_stride", "allowed_stride")] + [("picked", C.c_void_p)]


_lib = None


def _cuda():
    global _lib
    if _lib is None:
        lib = qxlib.cuda()
        P, U32, U64, D, E = C.c_void_p, C.c_uint32, C.c_uint64, C.c_double, C.c_char_p
        sig = {
            "qx_cuda_kv_view": [P, U32, P, E, U64],
            "qx_cuda_rope_frequencies": [U32, U32, D, D, D, D, D, P, P, E, U64],
            "qx_cuda_rope_append": [P, U32, P, P, U32, U32, P, P, P, P, P, P, P, E, U64],
            "qx_cuda_tree_attention": [P, U32, P, U32, U32, P, P, P, C.c_float, P, P, P, U64, P, P, E, U64],
            "qx_cuda_tree_attention_workspace": [U32, U32, U32, U32, U32, U32, P, E, U64],
            "qx_cuda_kv_evict": [P, U32, P, P, P, P, U32, U32, U32, P, P, P, P, E, U64],
            "qx_cuda_pick_tokens": [P, P, E, U64],
        }
        for name, args in sig.items():
            fn = getattr(lib, name)
            fn.argtypes = args
            fn.restype = C.c_int
        _lib = lib
    return _lib


def _call(fn, *args):
    err = C.create_string_buffer(256)
    if not fn(*args, err, 256):
        raise RuntimeError("%s failed: %s" % (fn.__name__, err.value.decode(errors="replace")))


def _stream(t):
    return torch.cuda.current_stream(t.device).cuda_stream


def _ptr(t, dtype, shape, device, what):
    """The address of a contiguous tensor of this type, shape and device; None stays None."""
    if t is None:
        return None
    if t.dtype is not dtype or t.device != device or t.shape != shape or not t.is_contiguous():
        raise ValueError("%s must be a contiguous %s tensor of shape %s on %s" % (what, dtype, tuple(shape), device))
    return t.data_ptr()


def _heads(t, dtype, shape, device, what):
    if t is None:
        return None
    if t.dtype is not dtype or t.device != device or t.shape != shape or (shape[3] > 1 and t.stride(3) != 1):
        raise ValueError("%s must be a %s tensor of shape %s on %s with a contiguous last dimension" % (
            what, dtype, tuple(shape), device))
    s = t.stride()
    return C.byref(_Heads(t.data_ptr(), s[0], s[1], s[2]))


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
        self.ref = C.byref(self.c)

    def mass_ptr(self, mass):
        """mass is addressed like the scales: same shape and strides."""
        if mass is None:
            return None
        if (mass.dtype is not torch.float32 or mass.shape != self.k_scales.shape or mass.device != self.device
                or mass.stride() != self.k_scales.stride()):
            raise ValueError("mass must be a float32 tensor like the scales")
        return mass.data_ptr()


class EngineCache:
    """The same handle on an engine's own cache (qx_cuda_kv_view): its
    single-sequence cache, or with batch=True the slots of decode_batch.
    Valid while the engine is open; order calls after the engine's own work
    (Engine.stream())."""

    def __init__(self, engine, batch=False, device=None):
        self.c = _Cache()
        _call(_cuda().qx_cuda_kv_view, engine.h, 1 if batch else 0, C.byref(self.c))
        self.engine = engine
        self.device = torch.device("cuda", torch.cuda.current_device() if device is None else device)
        self.slots, self.layers, self.ctx = self.c.slots, self.c.layers, self.c.ctx_tokens
        self.kv_heads, self.head_dim = self.c.kv_heads, self.c.head_dim
        self.ref = C.byref(self.c)

    def mass_ptr(self, mass):
        if mass is None:
            return None
        return _ptr(mass, torch.float32, (self.slots, self.layers, self.ctx), self.device, "mass")


def rope_frequencies(rotary_dim, base=1e6, scheme="none", factor=1.0, original_ctx=4096, low=1.0, high=32.0):
    """(inv_freq float64 [rotary_dim / 2], amplitude) of a context-extension
    scheme: none, linear, ntk, yarn or bands (qx_cuda_rope_frequencies)."""
    out = np.zeros(max(1, rotary_dim // 2), np.float64)
    amp = C.c_double()
    _call(_cuda().qx_cuda_rope_frequencies, ROPE_SCHEMES[scheme], rotary_dim, base, factor, original_ctx, low, high,
          out.ctypes.data, C.byref(amp))
    return out, amp.value


def _drafts(cache, slots, lens, nodes, seqs, max_nodes):
    one = (seqs,)
    return C.byref(_Drafts(seqs, max_nodes, _ptr(slots, torch.int32, one, cache.device, "slots"),
                           _ptr(lens, torch.int32, one, cache.device, "lens"),
                           _ptr(nodes, torch.int32, one, cache.device, "nodes")))


def rope_append(cache, layer, slots, lens, q, k, v, inv_freq, positions=None, nodes=None, interleaved=False, factor=1.0,
                q_out=None, status=None):
    """Rotate drafted tokens and append their keys and values
    (qx_cuda_rope_append).  q [seqs][nodes][q_heads][head_dim], k and v
    [seqs][nodes][kv_heads][head_dim] of one float type (q, or k and v, may be
    None); inv_freq float64 on the device, factor the amplitude.  Returns the
    rotated queries (q_out; q itself rotates in place)."""
    x = q if q is not None else k
    if x is None:
        raise ValueError("nothing to rotate")
    seqs, n, _, hd = x.shape
    dt, dev = x.dtype, cache.device
    if dt not in _TYPES:
        raise ValueError("unsupported element type %s" % dt)
    if q is not None and q_out is None:
        q_out = torch.zeros_like(q, memory_format=torch.contiguous_format)
    kv_shape = (seqs, n, cache.kv_heads, hd)
    if hd != cache.head_dim:
        raise ValueError("head_dim differs from the cache's")
    if q is None and q_out is not None:
        raise ValueError("q_out without q")
    rot = _Rotary(_ptr(inv_freq, torch.float64, (inv_freq.numel(),), dev, "inv_freq"), factor, 2 * inv_freq.numel(),
                  1 if interleaved else 0)
    _call(_cuda().qx_cuda_rope_append, cache.ref, layer, _drafts(cache, slots, lens, nodes, seqs, n), C.byref(rot), _TYPES[dt],
          q.shape[2] if q is not None else 0, _heads(q, dt, x.shape, dev, "q"), _heads(q_out, dt, x.shape, dev, "q_out"),
          _heads(k, dt, kv_shape, dev, "k"), _heads(v, dt, kv_shape, dev, "v"),
          _ptr(positions, torch.int32, (seqs, n), dev, "positions"), _ptr(status, torch.int32, (1,), dev, "status"), _stream(x))
    return q_out


_workspace_bytes = {}


def tree_attention(cache, layer, slots, lens, q, nodes=None, mask=None, scale=None, out=None, lse=None, mass=None,
                   status=None):
    """Attention of drafted tokens over the cache (qx_cuda_tree_attention).
    q [seqs][nodes][q_heads][head_dim]; mask int64 [seqs][nodes][words] of
    visibility bits, None for a chain; scale None: head_dim ** -0.5; lse
    float32 [seqs][nodes][q_heads] and mass (like the cache's scales) are
    written where given.  Returns out (like q)."""
    seqs, n, qh, hd = q.shape
    dt, dev = q.dtype, cache.device
    if dt not in _TYPES:
        raise ValueError("unsupported element type %s" % dt)
    if hd != cache.head_dim:
        raise ValueError("head_dim differs from the cache's")
    if out is None:
        out = torch.zeros(q.shape, dtype=dt, device=q.device)
    shape = (seqs, n, qh, cache.kv_heads, hd, dt)
    need = _workspace_bytes.get(shape)
    if need is None:                                      # a function of these sizes alone
        b = C.c_uint64()
        _call(_cuda().qx_cuda_tree_attention_workspace, seqs, n, qh, cache.kv_heads, hd, _TYPES[dt], C.byref(b))
        need = _workspace_bytes[shape] = b.value
    work = torch.empty(need, dtype=torch.uint8, device=dev)
    _call(_cuda().qx_cuda_tree_attention, cache.ref, layer, _drafts(cache, slots, lens, nodes, seqs, n), _TYPES[dt], qh,
          _heads(q, dt, q.shape, dev, "q"), _heads(out, dt, q.shape, dev, "out"),
          _ptr(mask, torch.int64, (seqs, n, (n + 63) // 64), dev, "mask"), hd ** -0.5 if scale is None else scale,
          _ptr(lse, torch.float32, (seqs, n, qh), dev, "lse"), cache.mass_ptr(mass), work.data_ptr(), need,
          _ptr(status, torch.int32, (1,), dev, "status"), _stream(q))
    return out


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
    seqs, dev = slots.shape[0], cache.device
    if kept is None:
        kept = torch.empty(cache.layers, seqs, budget, dtype=torch.int32, device=dev)
    if new_lens is None:
        new_lens = torch.empty(seqs, dtype=torch.int32, device=dev)
    one = (seqs,)
    _call(_cuda().qx_cuda_kv_evict, cache.ref, seqs, _ptr(slots, torch.int32, one, dev, "slots"),
          _ptr(dst_slots, torch.int32, one, dev, "dst_slots"), _ptr(lens, torch.int32, one, dev, "lens"), cache.mass_ptr(mass),
          budget, sink, recent, _ptr(kept, torch.int32, (cache.layers, seqs, budget), dev, "kept"),
          _ptr(new_lens, torch.int32, one, dev, "new_lens"), _ptr(status, torch.int32, (1,), dev, "status"), _stream(slots))
    return kept, new_lens


def _rows(t, dtype, rows, device, what):
    """(address, columns, row stride) of a [rows][columns] tensor with contiguous rows."""
    if t is None:
        return None, 0, 0
    if t.dtype is not dtype or t.device != device or t.dim() != 2 or t.shape[0] != rows or (t.shape[1] > 1 and t.stride(1) != 1):
        raise ValueError("%s must be a %s tensor [%d][...] on %s with contiguous rows" % (what, dtype, rows, device))
    return t.data_ptr(), t.shape[1], t.stride(0)


def pick_tokens(logits, history=None, history_lens=None, repetition=None, frequency=None, presence=None, bias_ids=None,
                bias_values=None, bias_lens=None, allowed=None, out=None, picked=None):
    """Penalties, biases, grammar mask and greedy token of each row
    (qx_cuda_pick_tokens).  logits [rows][vocab]; history int32 [rows][...];
    repetition, frequency, presence float32 [rows]; bias_ids int32 and
    bias_values float32 [rows][...]; allowed int32 [rows][(vocab + 31) / 32] of
    bits.  Returns (adjusted logits, int32 tokens, -1 where a row has none); out may be logits."""
    rows, vocab = logits.shape
    dt, dev = logits.dtype, logits.device
    if dt not in _TYPES:
        raise ValueError("unsupported element type %s" % dt)
    if out is None:
        out = torch.empty(rows, vocab, dtype=dt, device=dev)
    if picked is None:
        picked = torch.empty(rows, dtype=torch.int32, device=dev)
    x, _, xs = _rows(logits, dt, rows, dev, "logits")
    o, oc, os_ = _rows(out, dt, rows, dev, "out")
    h, hc, hs = _rows(history, torch.int32, rows, dev, "history")
    b, bc, bs = _rows(bias_ids, torch.int32, rows, dev, "bias_ids")
    bv, bvc, bvs = _rows(bias_values, torch.float32, rows, dev, "bias_values")
    m, mc, ms = _rows(allowed, torch.int32, rows, dev, "allowed")
    if oc != vocab or (b and (bvc != bc or (rows > 1 and bvs != bs))) or (m and mc < (vocab + 31) // 32):
        raise ValueError("out, bias_values and allowed must match logits and bias_ids")
    one, f = (rows,), torch.float32
    args = _Pick(x, o, xs, os_, rows, vocab, _TYPES[dt], hc, bc, 0, h, _ptr(history_lens, torch.int32, one, dev, "history_lens"),
                 _ptr(repetition, f, one, dev, "repetition"), _ptr(frequency, f, one, dev, "frequency"),
                 _ptr(presence, f, one, dev, "presence"), b, _ptr(bias_lens, torch.int32, one, dev, "bias_lens"), bv, m, hs, bs,
                 ms, _ptr(picked, torch.int32, one, dev, "picked"))
    _call(_cuda().qx_cuda_pick_tokens, C.byref(args), _stream(logits))
    return out, picked
