// The Python side of the device operators: a CPython module that takes torch
// tensors apart and makes one C-ABI call (include/qx_cuda.h) on their device's
// current stream.  It computes nothing.  It is native because a call's own
// cost counts: building the same arguments through ctypes took 25 us for
// qx_cuda_rope_append, several times what its kernel takes for one token.
#include <Python.h>
#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/Exceptions.h>

#include <cstdio>
#include <string>

#include "qx_cuda.h"

namespace {

[[noreturn]] void bad(const std::string& m) { throw c10::ValueError(c10::SourceLocation{__func__, __FILE__, __LINE__}, m); }

// Argument i as a tensor, or nullptr for None.
const at::Tensor* tensor(PyObject* o, const char* what) {
    if (o == Py_None) return nullptr;
    if (!THPVariable_Check(o)) bad(std::string(what) + " must be a tensor");
    return &THPVariable_Unpack(o);
}
const at::Tensor& needed(PyObject* o, const char* what) {
    const at::Tensor* t = tensor(o, what);
    if (!t) bad(std::string(what) + " must be a tensor");
    return *t;
}

std::string shape_of(at::IntArrayRef s) {
    std::string r = "[";
    for (size_t i = 0; i < s.size(); ++i) r += (i ? ", " : "") + std::to_string(s[i]);
    return r + "]";
}

uint32_t type_of(const at::Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return QX_CUDA_F32;
        case at::kHalf: return QX_CUDA_F16;
        case at::kBFloat16: return QX_CUDA_BF16;
        default: bad(std::string("unsupported element type ") + c10::toString(t.scalar_type()));
    }
}

// The operators have no backward pass: a result without its gradient is refused rather than given.
void no_grad(const at::Tensor& t, const char* what) {
    if (t.requires_grad() && c10::GradMode::is_enabled())
        bad(std::string(what) + " requires grad, and the operators have no backward pass: call them under torch.no_grad()");
}

void same(const at::Tensor& t, at::ScalarType type, at::IntArrayRef shape, c10::Device dev, const char* what, bool ok) {
    if (t.scalar_type() != type || t.device() != dev || t.sizes() != shape || !ok || t.is_conj() || t.is_neg())
        bad(std::string(what) + " must be a contiguous " + c10::toString(type) + " tensor of shape " + shape_of(shape) + " on " +
            dev.str());
    no_grad(t, what);
}

// The address of a contiguous tensor of this type, shape and device; None: NULL.
template <class T>
T* plain(PyObject* o, at::ScalarType type, at::IntArrayRef shape, c10::Device dev, const char* what) {
    const at::Tensor* t = tensor(o, what);
    if (!t) return nullptr;
    same(*t, type, shape, dev, what, t->is_contiguous());
    return (T*)t->data_ptr();
}

// A [seqs][nodes][heads][dim] tensor whose last dimension is contiguous.
qx_cuda_heads heads(const at::Tensor* t, at::ScalarType type, at::IntArrayRef shape, c10::Device dev, const char* what) {
    if (!t) return qx_cuda_heads{};
    same(*t, type, shape, dev, what, t->dim() == 4 && (shape[3] == 1 || t->stride(3) == 1));
    return {t->data_ptr(), (uint64_t)t->stride(0), (uint64_t)t->stride(1), (uint64_t)t->stride(2)};
}

struct Rows {
    void* p = nullptr;
    int64_t cols = 0, stride = 0;
};
Rows rows_of(const at::Tensor* t, at::ScalarType type, int64_t rows, c10::Device dev, const char* what) {
    if (!t) return {};
    if (t->scalar_type() != type || t->device() != dev || t->dim() != 2 || t->size(0) != rows ||
        (t->size(1) > 1 && t->stride(1) != 1) || t->is_conj() || t->is_neg())
        bad(std::string(what) + " must be a " + c10::toString(type) + " tensor [" + std::to_string(rows) +
            "][...] on " + dev.str() + " with contiguous rows");
    no_grad(*t, what);
    return {t->data_ptr(), t->size(1), t->stride(0)};
}

uint32_t u32(PyObject* o, const char* what) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw python_error();
    if (v < 0 || v > 0xffffffffll) bad(std::string(what) + " must fit 32 bits");
    return (uint32_t)v;
}
bool truth(PyObject* o) {
    const int v = PyObject_IsTrue(o);
    if (v < 0) throw python_error();
    return v != 0;
}
double number(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw python_error();
    return v;
}

// A cache handle: (address of a qx_cuda_kv_cache, device index).
struct Handle {
    const qx_cuda_kv_cache* c;
    c10::Device dev;
};
Handle handle(PyObject* o) {
    if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 2) bad("a cache must be a KvCache or an EngineCache");
    const void* p = PyLong_AsVoidPtr(PyTuple_GET_ITEM(o, 0));
    const long d = PyLong_AsLong(PyTuple_GET_ITEM(o, 1));
    if (PyErr_Occurred()) throw python_error();
    return {(const qx_cuda_kv_cache*)p, d < 0 ? c10::Device(c10::kCPU) : c10::Device(c10::kCUDA, (c10::DeviceIndex)d)};
}
// mass has the shape and strides of the scales.
float* mass_of(PyObject* o, const Handle& h) {
    const at::Tensor* t = tensor(o, "mass");
    if (!t) return nullptr;
    const qx_cuda_kv_cache& c = *h.c;
    if (t->scalar_type() != at::kFloat || t->device() != h.dev || t->dim() != 3 || t->size(0) != c.slots ||
        t->size(1) != c.layers || t->size(2) != c.ctx_tokens || (c.slots > 1 && (uint64_t)t->stride(0) != c.slot_rows) ||
        (c.layers > 1 && (uint64_t)t->stride(1) != c.layer_rows) || (c.ctx_tokens > 1 && t->stride(2) != 1))
        bad("mass must be a float32 tensor like the scales");
    no_grad(*t, "mass");
    return (float*)t->data_ptr();
}

void* stream_of(c10::Device d) {
    if (!d.is_cuda()) bad("the operators take CUDA tensors");
    return (void*)c10::cuda::getCurrentCUDAStream(d.index()).stream();
}

void check(int ok, const char* err, const char* what) {
    if (ok) return;
    PyErr_Format(PyExc_RuntimeError, "%s failed: %s", what, err);
    throw python_error();
}

void arity(Py_ssize_t got, Py_ssize_t want) {
    if (got != want) bad("wrong number of arguments");
}

qx_cuda_drafts drafts(const Handle& h, PyObject* slots, PyObject* lens, PyObject* nodes, int64_t seqs, int64_t n) {
    if (seqs > 0xffffffffll || n > 0xffffffffll) bad("too many sequences or nodes");
    return {(uint32_t)seqs, (uint32_t)n, plain<int32_t>(slots, at::kInt, {seqs}, h.dev, "slots"),
            plain<int32_t>(lens, at::kInt, {seqs}, h.dev, "lens"), plain<int32_t>(nodes, at::kInt, {seqs}, h.dev, "nodes")};
}

// cache, layer, slots, lens, q, k, v, inv_freq, positions, nodes, interleaved, factor, q_out, status, mass
PyObject* rope_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    arity(n, 15);
    const Handle h = handle(a[0]);
    const at::Tensor *q = tensor(a[4], "q"), *k = tensor(a[5], "k"), *v = tensor(a[6], "v"), *qo = tensor(a[12], "q_out");
    const at::Tensor* x = q ? q : k;
    if (!x) bad("nothing to rotate");
    if (x->dim() != 4) bad("q, k and v must be [seqs][nodes][heads][head_dim]");
    const uint32_t type = type_of(*x);
    if (x->size(3) != (int64_t)h.c->head_dim) bad("head_dim differs from the cache's");
    if (!q && qo) bad("q_out without q");
    at::Tensor made;
    if (q && !qo) {
        made = at::zeros(q->sizes(), q->options());
        qo = &made;
    }
    const at::ScalarType st = x->scalar_type();
    const int64_t seqs = x->size(0), nodes = x->size(1);
    const int64_t kv_shape[4] = {seqs, nodes, (int64_t)h.c->kv_heads, (int64_t)h.c->head_dim};
    const at::Tensor& inv = needed(a[7], "inv_freq");
    same(inv, at::kDouble, {inv.numel()}, h.dev, "inv_freq", inv.is_contiguous());
    qx_cuda_rotary rot{(const double*)inv.data_ptr(), number(a[11]), (uint32_t)(2 * inv.numel()), truth(a[10]) ? 1u : 0u};
    const qx_cuda_drafts d = drafts(h, a[2], a[3], a[9], seqs, nodes);
    const qx_cuda_heads hq = heads(q, st, x->sizes(), h.dev, "q"), ho = heads(qo, st, x->sizes(), h.dev, "q_out"),
                        hk = heads(k, st, kv_shape, h.dev, "k"), hv = heads(v, st, kv_shape, h.dev, "v");
    const uint32_t layer = u32(a[1], "layer");
    const int32_t* positions = plain<int32_t>(a[8], at::kInt, {seqs, nodes}, h.dev, "positions");
    float* mass = mass_of(a[14], h);
    uint32_t* status = plain<uint32_t>(a[13], at::kInt, {1}, h.dev, "status");
    char err[256];
    check(qx_cuda_rope_append_mass(h.c, layer, &d, &rot, type, q ? (uint32_t)q->size(2) : 0u, &hq, &ho, &hk, &hv, positions, mass,
                                   status, stream_of(h.dev), err, sizeof err),
          err, "qx_cuda_rope_append");
    if (!q) Py_RETURN_NONE;
    return THPVariable_Wrap(*qo);
    END_HANDLE_TH_ERRORS
}

// cache, layer, slots, lens, q, nodes, mask, scale (None: head_dim ** -0.5), out, lse, mass, status
PyObject* tree_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    arity(n, 12);
    const Handle h = handle(a[0]);
    const at::Tensor& q = needed(a[4], "q");
    const at::Tensor* out = tensor(a[8], "out");
    if (q.dim() != 4) bad("q must be [seqs][nodes][heads][head_dim]");
    const uint32_t type = type_of(q);
    if (q.size(3) != (int64_t)h.c->head_dim) bad("head_dim differs from the cache's");
    const int64_t seqs = q.size(0), nodes = q.size(1), qh = q.size(2);
    at::Tensor made;
    if (!out) {
        made = at::zeros(q.sizes(), q.options());
        out = &made;
    }
    const qx_cuda_drafts d = drafts(h, a[2], a[3], a[5], seqs, nodes);
    const qx_cuda_heads hq = heads(&q, q.scalar_type(), q.sizes(), h.dev, "q"),
                        ho = heads(out, q.scalar_type(), q.sizes(), h.dev, "out");
    const uint32_t layer = u32(a[1], "layer");
    const uint64_t* mask = plain<uint64_t>(a[6], at::kLong, {seqs, nodes, (nodes + 63) / 64}, h.dev, "mask");
    const float scale = a[7] == Py_None ? (float)(1.0 / std::sqrt((double)h.c->head_dim)) : (float)number(a[7]);
    float *lse = plain<float>(a[9], at::kFloat, {seqs, nodes, qh}, h.dev, "lse"), *mass = mass_of(a[10], h);
    uint32_t* status = plain<uint32_t>(a[11], at::kInt, {1}, h.dev, "status");
    char err[256];
    uint64_t bytes = 0;
    check(qx_cuda_tree_attention_workspace((uint32_t)seqs, (uint32_t)nodes, (uint32_t)qh, h.c->kv_heads, h.c->head_dim, type, &bytes,
                                           err, sizeof err),
          err, "qx_cuda_tree_attention");
    void* stream = stream_of(h.dev);
    // from torch's stream-ordered allocator, so each call and each captured graph has its own
    const at::Tensor work = at::empty({(int64_t)bytes}, q.options().dtype(at::kByte));
    check(qx_cuda_tree_attention(h.c, layer, &d, type, (uint32_t)qh, &hq, &ho, mask, scale, lse, mass, work.data_ptr(), bytes,
                                 status, stream, err, sizeof err),
          err, "qx_cuda_tree_attention");
    return THPVariable_Wrap(*out);
    END_HANDLE_TH_ERRORS
}

// cache, slots, lens, mass, budget, sink, recent, dst_slots, kept, new_lens, status
PyObject* evict(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    arity(n, 11);
    const Handle h = handle(a[0]);
    const at::Tensor& slots = needed(a[1], "slots");
    if (slots.dim() != 1) bad("slots must have one dimension");
    const int64_t seqs = slots.size(0), layers = h.c->layers;
    const uint32_t budget = u32(a[4], "budget");
    const at::Tensor *kept = tensor(a[8], "kept"), *fresh = tensor(a[9], "new_lens");
    at::Tensor made_kept, made_new;
    if (!kept) {
        made_kept = at::empty({layers, seqs, (int64_t)budget}, slots.options().dtype(at::kInt));
        kept = &made_kept;
    }
    if (!fresh) {
        made_new = at::empty({seqs}, slots.options().dtype(at::kInt));
        fresh = &made_new;
    }
    same(*kept, at::kInt, {layers, seqs, (int64_t)budget}, h.dev, "kept", kept->is_contiguous());
    same(*fresh, at::kInt, {seqs}, h.dev, "new_lens", fresh->is_contiguous());
    if (seqs > 0xffffffffll) bad("too many sequences");
    const int32_t *from = plain<int32_t>(a[1], at::kInt, {seqs}, h.dev, "slots"), *to = plain<int32_t>(a[7], at::kInt, {seqs}, h.dev, "dst_slots"),
                  *lens = plain<int32_t>(a[2], at::kInt, {seqs}, h.dev, "lens");
    float* mass = mass_of(a[3], h);
    const uint32_t sink = u32(a[5], "sink"), recent = u32(a[6], "recent");
    uint32_t* status = plain<uint32_t>(a[10], at::kInt, {1}, h.dev, "status");
    char err[256];
    check(qx_cuda_kv_evict(h.c, (uint32_t)seqs, from, to, lens, mass, budget, sink, recent, (int32_t*)kept->data_ptr(),
                           (int32_t*)fresh->data_ptr(), status, stream_of(h.dev), err, sizeof err),
          err, "qx_cuda_kv_evict");
    return Py_BuildValue("(NN)", THPVariable_Wrap(*kept), THPVariable_Wrap(*fresh));
    END_HANDLE_TH_ERRORS
}

// logits, history, history_lens, repetition, frequency, presence, bias_ids, bias_values, bias_lens, allowed, out, picked
PyObject* pick_tokens(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    arity(n, 12);
    const at::Tensor& x = needed(a[0], "logits");
    if (x.dim() != 2) bad("logits must be [rows][vocab]");
    const c10::Device dev = x.device();
    const int64_t rows = x.size(0), vocab = x.size(1);
    const at::Tensor *out = tensor(a[10], "out"), *picked = tensor(a[11], "picked");
    qx_cuda_pick p{};
    p.dtype = type_of(x);
    if (rows > 0xffffffffll || vocab > 0xffffffffll) bad("too many rows or tokens");
    at::Tensor made_out, made_picked;
    if (!out) {
        made_out = at::empty({rows, vocab}, x.options());
        out = &made_out;
    }
    if (!picked) {
        made_picked = at::empty({rows}, x.options().dtype(at::kInt));
        picked = &made_picked;
    }
    const Rows l = rows_of(&x, x.scalar_type(), rows, dev, "logits"), o = rows_of(out, x.scalar_type(), rows, dev, "out"),
               h = rows_of(tensor(a[1], "history"), at::kInt, rows, dev, "history"),
               b = rows_of(tensor(a[6], "bias_ids"), at::kInt, rows, dev, "bias_ids"),
               bv = rows_of(tensor(a[7], "bias_values"), at::kFloat, rows, dev, "bias_values"),
               m = rows_of(tensor(a[9], "allowed"), at::kInt, rows, dev, "allowed");
    if (o.cols != vocab || (b.p && bv.p && (bv.cols != b.cols || (rows > 1 && bv.stride != b.stride))) ||
        (m.p && m.cols < (vocab + 31) / 32) || h.cols > 0xffffffffll || b.cols > 0xffffffffll)
        bad("out, bias_values and allowed must match logits and bias_ids");
    same(*picked, at::kInt, {rows}, dev, "picked", picked->is_contiguous());
    p.logits = l.p;
    p.out = o.p;
    p.logits_stride = (uint64_t)l.stride;
    p.out_stride = (uint64_t)o.stride;
    p.rows = (uint32_t)rows;
    p.vocab = (uint32_t)vocab;
    p.max_history = (uint32_t)h.cols;
    p.max_bias = (uint32_t)b.cols;
    p.history = (const int32_t*)h.p;
    p.history_lens = plain<int32_t>(a[2], at::kInt, {rows}, dev, "history_lens");
    p.repetition = plain<float>(a[3], at::kFloat, {rows}, dev, "repetition");
    p.frequency = plain<float>(a[4], at::kFloat, {rows}, dev, "frequency");
    p.presence = plain<float>(a[5], at::kFloat, {rows}, dev, "presence");
    p.bias_ids = (const int32_t*)b.p;
    p.bias_lens = plain<int32_t>(a[8], at::kInt, {rows}, dev, "bias_lens");
    p.bias_values = (const float*)bv.p;
    p.allowed = (const uint32_t*)m.p;
    p.history_stride = (uint64_t)h.stride;
    p.bias_stride = (uint64_t)b.stride;
    p.allowed_stride = (uint64_t)m.stride;
    p.picked = (uint32_t*)picked->data_ptr();
    char err[256];
    check(qx_cuda_pick_tokens(&p, stream_of(dev), err, sizeof err), err, "qx_cuda_pick_tokens");
    return Py_BuildValue("(NN)", THPVariable_Wrap(*out), THPVariable_Wrap(*picked));
    END_HANDLE_TH_ERRORS
}

#define FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(f)), METH_FASTCALL, nullptr
PyMethodDef kMethods[] = {{"rope_append", FAST(rope_append)},
                          {"tree_attention", FAST(tree_attention)},
                          {"evict", FAST(evict)},
                          {"pick_tokens", FAST(pick_tokens)},
                          {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_qxops", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__qxops(void) { return PyModule_Create(&kModule); }
