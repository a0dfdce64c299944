// Penalties, biases and a grammar mask on logits, and the greedy token of each
// row (qx_cuda_pick_tokens).
//
// A cluster of CTAs takes one row; each CTA owns a slice of the vocabulary and
// keeps one 32-bit word per token of it in shared memory: the token's count in
// the history (low 20 bits) and the last bias entry that names it, plus one
// (high 12 bits).  Every CTA reads the whole history and counts what falls in
// its slice, in its own shared memory: counting each part of the history once
// and into other CTAs' memory instead reads an eighth, but histories repeat
// few tokens, whose CTA then takes thousands of single remote additions (256
// rows of 151936, histories of 4096: 155 us against XX).  Integer atomics, so
// the order they land in changes nothing.  Then each CTA streams its slice of
// the logits once, the first of it in registers since before the counting
// began, and the row's best is joined through the cluster, with no workspace
// and one launch.
//
// Rows need not start on 16-byte boundaries: a row's tokens are numbered from
// the boundary before it ("places"), and slices and packs are of places.
#include <cooperative_groups.h>

#include <cmath>

#include "qx_ops.cuh"

namespace {

using namespace qx::ops;
namespace cg = cooperative_groups;

constexpr int kPickCluster = 8;                        // CTAs a row
constexpr uint32_t kMaxVocab = 393216, kCountBits = 20, kCountMask = (1u << kCountBits) - 1;

struct PickArgs {
    const void* logits;
    void* out;
    size_t logits_stride, out_stride;
    int vocab, slice, max_history, max_bias;
    const int *history, *history_lens;
    const float *repetition, *frequency, *presence;
    const int *bias_ids, *bias_lens;
    const float* bias_values;
    const uint32_t* allowed;
    size_t history_stride, bias_stride, allowed_stride;
    uint32_t* picked;
};

struct Best {
    float v;
    int i;
    int bad;      // an x that is NaN or +infinity
};

__device__ __forceinline__ void better(Best& a, float v, int i) {
    if (v > a.v || (v == a.v && i < a.i)) a.v = v, a.i = i;
}

__device__ __forceinline__ bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
__device__ __forceinline__ int clamped(const int* lens, int r, int most) {
    return lens ? max(0, min(lens[r], most)) : most;
}

template <class T, int THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) k_pick(const __grid_constant__ PickArgs a) {
    constexpr int V = 16 / sizeof(T), kAhead = V == 4 ? 4 : 2;         // packs a thread has in flight
    extern __shared__ __align__(16) uint32_t words[];
    __shared__ Best wbest[THREADS / 32], cbest;
    cg::cluster_group cl = cg::this_cluster();
    const int rank = (int)cl.block_rank(), r = blockIdx.x / kPickCluster, tid = threadIdx.x;
    const bool touched = a.history || a.bias_ids;
    // token t is at place t + shift
    const T* x = (const T*)a.logits + r * a.logits_stride;
    T* o = a.out ? (T*)a.out + r * a.out_stride : nullptr;
    const int shift = (int)(reinterpret_cast<uintptr_t>(x) / sizeof(T) % V);
    const bool wide_out = o && (int)(reinterpret_cast<uintptr_t>(o) / sizeof(T) % V) == shift;
    const int lo = rank * a.slice, hi = min(lo + a.slice, a.vocab + shift);      // places of this CTA, from shift on in the first
    const uint32_t* allowed = a.allowed ? a.allowed + r * a.allowed_stride : nullptr;
    auto whole = [&](int p) { return p >= shift && p + V <= min(hi, a.vocab + shift); };
    // a pack's logits, and its tokens' bits of the mask
    auto load = [&](int p, Pack<T, V>& v, uint32_t& bits) {
        bits = ~0u;
        if (whole(p)) {
            const int t = p - shift;
            v = *reinterpret_cast<const Pack<T, V>*>(x + t);
            if (allowed) bits = __funnelshift_r(allowed[t >> 5], allowed[(t + V - 1) >> 5], t & 31);
        }
    };
    Pack<T, V> pack[kAhead];
    uint32_t bits[kAhead];
    int p0 = lo + tid * V;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) load(p0 + i * THREADS * V, pack[i], bits[i]);
    const float rep = a.repetition ? a.repetition[r] : 1.f, freq = a.frequency ? a.frequency[r] : 0.f,
                pres = a.presence ? a.presence[r] : 0.f;
    if (touched) {
        for (int i = tid * 4; i < a.slice; i += THREADS * 4) *reinterpret_cast<uint4*>(words + i) = make_uint4(0, 0, 0, 0);
        __syncthreads();
        const int l0 = max(lo - shift, 0), n = hi - shift - l0;          // the slice's tokens l0 .. l0 + n
        uint32_t* word = words + (l0 + shift - lo);
        if (a.bias_ids) {
            const int nb = clamped(a.bias_lens, r, a.max_bias);
            for (int j = tid; j < nb; j += THREADS) {
                const int k = a.bias_ids[r * a.bias_stride + j] - l0;
                if ((unsigned)k < (unsigned)max(n, 0) && k + l0 >= 0) atomicMax(&word[k], (uint32_t)(j + 1) << kCountBits);
            }
            __syncthreads();
        }
        if (a.history) {
            const int nh = clamped(a.history_lens, r, a.max_history);
            const int* h = a.history + r * a.history_stride;
            auto count = [&](int id) {
                const unsigned k = (unsigned)id - (unsigned)l0;
                if (k < (unsigned)max(n, 0)) atomicAdd(&word[k], 1u);
            };
            int j = tid * 4;
            if (aligned16(h))
                for (; j + 4 <= nh; j += THREADS * 4) {
                    const int4 q = *reinterpret_cast<const int4*>(h + j);
                    count(q.x), count(q.y), count(q.z), count(q.w);
                }
            else
                for (; j + 4 <= nh; j += THREADS * 4) {
                    const int q0 = h[j], q1 = h[j + 1], q2 = h[j + 2], q3 = h[j + 3];
                    count(q0), count(q1), count(q2), count(q3);
                }
            for (int e = j; e < min(j + 4, nh); ++e) count(h[e]);
        }
        __syncthreads();
    }
    Best best{-INFINITY, 0x7fffffff, 0};
    auto touch = [&](float v, uint32_t w) {
        const uint32_t c = w & kCountMask, b = w >> kCountBits;
        if (c) {
            v = v > 0.f ? __fdiv_rn(v, rep) : __fmul_rn(v, rep);
            v = __fsub_rn(v, __fmul_rn(freq, (float)c));
            v = __fsub_rn(v, pres);
        }
        if (b) v = __fadd_rn(v, a.bias_values[r * a.bias_stride + b - 1]);
        return v;
    };
    for (; p0 < hi; p0 += kAhead * THREADS * V) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int p = p0 + i * THREADS * V, t = p - shift;
            if (whole(p)) {
                float v[V];
#pragma unroll
                for (int u = 0; u < V; ++u) v[u] = to_f32(pack[i].v[u]);
                const uint32_t ok = bits[i];
                load(p + kAhead * THREADS * V, pack[i], bits[i]);        // on its way while this one is worked on
                if (touched)
#pragma unroll
                    for (int u = 0; u < V; u += 4) {
                        const uint4 q = *reinterpret_cast<const uint4*>(words + (p - lo) + u);
                        if (q.x | q.y | q.z | q.w) {
                            if (q.x) v[u] = touch(v[u], q.x);
                            if (q.y) v[u + 1] = touch(v[u + 1], q.y);
                            if (q.z) v[u + 2] = touch(v[u + 2], q.z);
                            if (q.w) v[u + 3] = touch(v[u + 3], q.w);
                        }
                    }
                float big = -INFINITY;
                Pack<T, V> y;
#pragma unroll
                for (int u = 0; u < V; ++u) {
                    if (!(ok >> u & 1u)) v[u] = -INFINITY;
                    best.bad |= !(v[u] < INFINITY);
                    big = fmaxf(big, v[u]);
                    y.v[u] = from_f32<T>(v[u]);
                }
                if (big > best.v) {
                    best.v = big;
#pragma unroll
                    for (int u = V - 1; u >= 0; --u)
                        if (v[u] == big) best.i = t + u;
                }
                if (wide_out) {
                    *reinterpret_cast<Pack<T, V>*>(o + t) = y;
                } else if (o) {
#pragma unroll
                    for (int u = 0; u < V; ++u) o[t + u] = y.v[u];
                }
            } else {
                if (p < hi)
#pragma unroll 1
                    for (int u = 0; u < V; ++u) {                        // the row's ends
                        const int e = t + u;
                        if (e < 0 || p + u >= hi || e >= a.vocab) continue;
                        float v = to_f32(x[e]);
                        if (touched && words[p + u - lo]) v = touch(v, words[p + u - lo]);
                        if (allowed && !(allowed[e >> 5] >> (e & 31) & 1u)) v = -INFINITY;
                        best.bad |= !(v < INFINITY);
                        if (v > best.v) best.v = v, best.i = e;
                        if (o) o[e] = from_f32<T>(v);
                    }
                load(p + kAhead * THREADS * V, pack[i], bits[i]);
            }
        }
    }
    for (int s = 16; s; s >>= 1) {
        const float v = __shfl_xor_sync(~0u, best.v, s);
        const int i = __shfl_xor_sync(~0u, best.i, s);
        better(best, v, i);
    }
    best.bad = __any_sync(~0u, best.bad);
    if ((tid & 31) == 0) wbest[tid >> 5] = best;
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < THREADS / 32; ++w) {
            better(best, wbest[w].v, wbest[w].i);
            best.bad |= wbest[w].bad;
        }
        cbest = best;
    }
    cl.sync();
    if (rank == 0 && tid == 0) {
        for (int c = 1; c < kPickCluster; ++c) {
            const Best* p = cl.map_shared_rank(&cbest, c);
            better(best, p->v, p->i);
            best.bad |= p->bad;
        }
        a.picked[r] = best.bad || !(best.v > -INFINITY) ? 0xffffffffu : (uint32_t)best.i;
    }
    cl.sync();                                           // the others' words live until they are read
}

template <class T, int THREADS>
cudaError_t launch_pick(const PickArgs& a, int rows, cudaStream_t st) {
    const size_t sm = a.history || a.bias_ids ? (size_t)a.slice * 4 : 0;
    cudaError_t e = cudaFuncSetAttribute((const void*)k_pick<T, THREADS>, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(rows * kPickCluster));
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = sm;
    cfg.stream = st;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = kPickCluster;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, k_pick<T, THREADS>, a);
}

}  // namespace

QX_API int qx_cuda_pick_tokens(const qx_cuda_pick* p, void* stream, char* err, uint64_t n) {
    if (!p || !p->logits || !p->picked) return refuse(err, n, "invalid pick argument");
    if (!p->rows || !p->vocab) return refuse(err, n, "a call needs at least one row and one token");
    if (p->rows > 1u << 20) return refuse(err, n, "at most 1048576 rows");
    if (p->vocab > kMaxVocab) return refuse(err, n, "vocab is at most 393216");
    if (p->dtype > QX_CUDA_BF16) return refuse(err, n, "unsupported element type");
    if (p->history && p->max_history > kCountMask) return refuse(err, n, "max_history must be below 2^20");
    if (p->bias_ids && p->max_bias > 4095) return refuse(err, n, "max_bias is at most 4095");
    if ((p->bias_ids != nullptr) != (p->bias_values != nullptr)) return refuse(err, n, "bias ids go with bias values");
    const uint64_t most = 1ull << 40;
    if (p->logits_stride > most || p->out_stride > most || p->history_stride > most || p->bias_stride > most ||
        p->allowed_stride > most)
        return refuse(err, n, "strides are too large");
    if (p->out && p->rows > 1 && p->out_stride < p->vocab) return refuse(err, n, "an output tensor overlaps itself");
    if (p->out == p->logits && p->rows > 1 && p->out_stride != p->logits_stride)
        return refuse(err, n, "out in place of logits must have their stride");
    const int eb = elem_bytes(p->dtype);
    if (!aligned(p->logits, eb) || !aligned(p->out, eb)) return refuse(err, n, "tensors must be aligned to their element");
    for (const void* q : {(const void*)p->history, (const void*)p->history_lens, (const void*)p->repetition,
                          (const void*)p->frequency, (const void*)p->presence, (const void*)p->bias_ids,
                          (const void*)p->bias_lens, (const void*)p->bias_values, (const void*)p->allowed,
                          (const void*)p->picked})
        if (!aligned(q, 4)) return refuse(err, n, "penalty, bias, mask and pick buffers must be 4-byte aligned");
    DeviceOf dev(p->logits, err, n);
    if (!dev.ok) return 0;
    PickArgs a{};
    a.logits = p->logits;
    a.out = p->out;
    a.logits_stride = p->logits_stride;
    a.out_stride = p->out_stride;
    a.vocab = (int)p->vocab;
    a.slice = (int)((p->vocab + 7 + kPickCluster * 64 - 1) / (kPickCluster * 64) * 64);      // of vocab and up to 7 places before it
    a.max_history = (int)p->max_history;
    a.max_bias = (int)p->max_bias;
    a.history = p->max_history ? p->history : nullptr;
    a.history_lens = p->history_lens;
    a.repetition = p->repetition;
    a.frequency = p->frequency;
    a.presence = p->presence;
    a.bias_ids = p->max_bias ? p->bias_ids : nullptr;
    a.bias_lens = p->bias_lens;
    a.bias_values = p->bias_values;
    a.allowed = p->allowed;
    a.history_stride = p->history_stride;
    a.bias_stride = p->bias_stride;
    a.allowed_stride = p->allowed_stride;
    a.picked = p->picked;
    cudaStream_t st = (cudaStream_t)stream;
    // few rows leave SMs to spare: one CTA of 1024 threads each, else two of 512
    const bool few = p->rows * kPickCluster <= 148;
    const int rows = (int)p->rows;
    cudaError_t e;
    if (p->dtype == QX_CUDA_F32) e = few ? launch_pick<float, 1024>(a, rows, st) : launch_pick<float, 512>(a, rows, st);
    else if (p->dtype == QX_CUDA_F16) e = few ? launch_pick<__half, 1024>(a, rows, st) : launch_pick<__half, 512>(a, rows, st);
    else e = few ? launch_pick<__nv_bfloat16, 1024>(a, rows, st) : launch_pick<__nv_bfloat16, 512>(a, rows, st);
    return finish(e, err, n);
}
