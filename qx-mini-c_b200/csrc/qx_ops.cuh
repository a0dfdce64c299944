// What the device operators share (qx_rope.cu, qx_tree.cu, qx_evict.cu,
// qx_pick.cu): argument checks on the host, the choice of device, element
// types, and the device-side check of a call's sequences.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <cstdio>

#include "qx_cuda.h"

#define QX_API extern "C" __attribute__((visibility("default")))

namespace qx {
namespace ops {

constexpr uint32_t kMaxSeqs = 4096, kMaxNodes = 4096, kMaxHeads = 1024, kMaxRow = 16384;

inline int refuse(char* err, uint64_t n, const char* m) {
    if (err && n) snprintf(err, (size_t)n, "%s", m);
    return 0;
}

inline int elem_bytes(uint32_t dtype) { return dtype == QX_CUDA_F32 ? 4 : 2; }
inline bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

// The device of the caller's memory becomes the current one for the call.
struct DeviceOf {
    int was = -1;
    bool ok = false;
    DeviceOf(const void* p, char* err, uint64_t n) {
        cudaPointerAttributes a{};
        cudaError_t e = cudaPointerGetAttributes(&a, p);
        if (e == cudaSuccess && a.type != cudaMemoryTypeDevice && a.type != cudaMemoryTypeManaged) {
            refuse(err, n, "the operators take device pointers");
            return;
        }
        int cur = 0;
        if (e == cudaSuccess) e = cudaGetDevice(&cur);
        if (e == cudaSuccess && cur != a.device) {
            e = cudaSetDevice(a.device);
            if (e == cudaSuccess) was = cur;
        }
        if (e != cudaSuccess) {
            cudaGetLastError();
            refuse(err, n, cudaGetErrorString(e));
            return;
        }
        ok = true;
    }
    ~DeviceOf() {
        if (was >= 0) cudaSetDevice(was);
    }
    DeviceOf(const DeviceOf&) = delete;
    DeviceOf& operator=(const DeviceOf&) = delete;
};

inline int finish(cudaError_t e, char* err, uint64_t n) {
    if (e == cudaSuccess) e = cudaGetLastError();
    if (e == cudaSuccess) return 1;
    cudaGetLastError();
    return refuse(err, n, cudaGetErrorString(e));
}

inline const char* check_cache(const qx_cuda_kv_cache* c) {
    if (!c || !c->k || !c->v || !c->k_scales || !c->v_scales) return "invalid cache argument";
    if (!c->slots || !c->layers || !c->ctx_tokens || !c->kv_heads || !c->head_dim) return "the cache has no rows";
    if (c->slots > 1u << 20 || c->layers > 4096 || c->ctx_tokens > 1u << 24 || c->kv_heads > kMaxHeads || c->head_dim > 4096)
        return "the cache is larger than the operators support";
    const uint64_t row = (uint64_t)c->kv_heads * c->head_dim;
    if (row % 16 || row > kMaxRow) return "a cache row must be a multiple of 16 bytes and at most 16384";
    if (!aligned(c->k, 16) || !aligned(c->v, 16)) return "cache codes must be 16-byte aligned";
    if (!aligned(c->k_scales, 4) || !aligned(c->v_scales, 4)) return "cache scales must be 4-byte aligned";
    if (c->slot_rows > 1ull << 40 || c->layer_rows > 1ull << 40) return "cache strides are too large";
    if (c->layers > 1 && c->layer_rows < c->ctx_tokens) return "the layers of the cache overlap";
    // [slot][layer][row] or [layer][slot][row]
    if (c->slots > 1) {
        const uint64_t slot_span = (uint64_t)(c->layers - 1) * c->layer_rows + c->ctx_tokens;
        const uint64_t inner = (uint64_t)(c->slots - 1) * c->slot_rows + c->ctx_tokens;
        if (!(c->slot_rows >= slot_span || (c->slot_rows >= c->ctx_tokens && (c->layers == 1 || c->layer_rows >= inner))))
            return "the slots of the cache overlap";
    }
    return nullptr;
}

inline const char* check_drafts(const qx_cuda_drafts* d) {
    if (!d || !d->slots || !d->lens) return "invalid drafts argument";
    if (d->seqs == 0 || d->max_nodes == 0) return "a call needs at least one sequence and one node";
    if (d->seqs > kMaxSeqs || d->max_nodes > kMaxNodes) return "at most 4096 sequences and 4096 nodes";
    if (!aligned(d->slots, 4) || !aligned(d->lens, 4) || !aligned(d->nodes, 4)) return "slots, lengths and nodes must be 4-byte aligned";
    return nullptr;
}

inline const char* check_heads(const qx_cuda_heads* t, uint32_t seqs, uint32_t nodes, uint32_t heads, uint32_t dim,
                               uint32_t dtype, bool written) {
    if (!t || !t->data) return "invalid tensor argument";
    if (dtype > QX_CUDA_BF16) return "unsupported element type";
    if (!aligned(t->data, (uintptr_t)elem_bytes(dtype))) return "tensors must be aligned to their element";
    const uint64_t most = 1ull << 40;
    if (t->seq_stride > most || t->node_stride > most || t->head_stride > most) return "tensor strides are too large";
    if (written) {
        // disjoint if, smallest stride first, each stride reaches past what lies within it
        uint64_t st[3] = {t->seq_stride, t->node_stride, t->head_stride};
        uint32_t n[3] = {seqs, nodes, heads};
        for (int i = 0; i < 2; ++i)
            for (int j = 0; j < 2 - i; ++j)
                if (st[j] > st[j + 1]) {
                    const uint64_t a = st[j]; st[j] = st[j + 1]; st[j + 1] = a;
                    const uint32_t b = n[j]; n[j] = n[j + 1]; n[j + 1] = b;
                }
        uint64_t span = dim;
        for (int i = 0; i < 3; ++i)
            if (n[i] > 1) {
                if (st[i] < span) return "an output tensor overlaps itself";
                span += (uint64_t)(n[i] - 1) * st[i];
            }
    }
    return nullptr;
}

// ---- device side -------------------------------------------------------------

template <class T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// N consecutive elements, as one access when N * sizeof(T) is 16 and the
// caller has checked the alignment.
template <class T, int N>
struct alignas(sizeof(T) * N) Pack {
    T v[N];
};

// Division by a number that the host knows.  (2^32 / d + 1) x / 2^32 is too
// large by less than x / 2^32 < 1, so the quotient by one at most.
struct Over {
    uint32_t d, by;
    Over(uint32_t d = 1) : d(d), by(d > 1 ? (uint32_t)((1ull << 32) / d + 1) : 0) {}
    __device__ __forceinline__ uint32_t operator()(uint32_t x) const {
        const uint32_t q = d > 1 ? __umulhi(x, by) : x;
        return q - (q * d > x);
    }
};

// Where the rows of a sequence lie.
struct Cache {
    int8_t *k, *v;
    float *ks, *vs;
    size_t slot_rows, layer_rows;
    int slots, layers, ctx, kv_heads, head_dim;
};
inline Cache cache_of(const qx_cuda_kv_cache* c) {
    return {c->k, c->v, c->k_scales, c->v_scales, (size_t)c->slot_rows, (size_t)c->layer_rows, (int)c->slots,
            (int)c->layers, (int)c->ctx_tokens, (int)c->kv_heads, (int)c->head_dim};
}

// Rows from the first to the end of the last.
inline size_t cache_rows(const Cache& c) {
    return (size_t)(c.slots - 1) * c.slot_rows + (size_t)(c.layers - 1) * c.layer_rows + (size_t)c.ctx;
}

struct Drafts {
    int seqs, max_nodes;
    const int *slots, *lens, *nodes;
    __device__ __forceinline__ int count(int s) const { return nodes ? nodes[s] : max_nodes; }
};
inline Drafts drafts_of(const qx_cuda_drafts* d) {
    return {(int)d->seqs, (int)d->max_nodes, d->slots, d->lens, d->nodes};
}

// Whether slot, len committed rows and n drafted ones lie inside the cache.
__device__ __forceinline__ bool fits(const Cache& c, const Drafts& d, int slot, int len, int n) {
    return slot >= 0 && slot < c.slots && n >= 0 && n <= d.max_nodes && len >= 0 && len <= c.ctx && n <= c.ctx - len;
}

}  // namespace ops
}  // namespace qx
