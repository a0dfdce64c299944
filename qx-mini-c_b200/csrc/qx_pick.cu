// Penalties, biases and a grammar mask on logits, and the greedy token of each
// row (qx_cuda_pick_tokens).
//
// A cluster of CTAs takes one row; each CTA owns a slice of the vocabulary and
// keeps one 32-bit word per token of it in shared memory: the token's count in
// the history (low 20 bits) and the last bias entry that names it, plus one
// (high 12 bits).  The cluster reads the history once, every CTA a part, and
// counts into the owner's words through distributed shared memory; integer
// atomics, so the order they land in changes nothing.  Then each CTA streams
// its slice of the logits once, and the row's best is joined through the
// cluster, with no workspace and one launch.
#include <cooperative_groups.h>

#include <cmath>

#include "qx_ops.cuh"

namespace {

using namespace qx::ops;
namespace cg = cooperative_groups;

constexpr int kPickThreads = 512, kPickCluster = 8;
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

__device__ __forceinline__ int clamped(const int* lens, int r, int most) {
    return lens ? max(0, min(lens[r], most)) : most;
}

template <class T, int V>
__global__ void __launch_bounds__(kPickThreads) k_pick(PickArgs a) {
    extern __shared__ uint32_t words[];
    __shared__ Best wbest[kPickThreads / 32], cbest;
    cg::cluster_group cl = cg::this_cluster();
    const int rank = (int)cl.block_rank(), r = blockIdx.x / kPickCluster, tid = threadIdx.x;
    const int lo = rank * a.slice, hi = min(lo + a.slice, a.vocab);
    const bool counts = a.history != nullptr, biases = a.bias_ids != nullptr;
    const float rep = a.repetition ? a.repetition[r] : 1.f, freq = a.frequency ? a.frequency[r] : 0.f,
                pres = a.presence ? a.presence[r] : 0.f;
    if (counts || biases) {
        for (int i = tid; i < a.slice; i += kPickThreads) words[i] = 0;
        __syncthreads();
        if (biases) {
            const int nb = clamped(a.bias_lens, r, a.max_bias);
            for (int j = tid; j < nb; j += kPickThreads) {
                const int id = a.bias_ids[r * a.bias_stride + j];
                if (id >= lo && id < hi) atomicMax(&words[id - lo], (uint32_t)(j + 1) << kCountBits);
            }
        }
        cl.sync();                                       // every CTA's words hold 0 and its biases
        if (counts) {
            const int nh = clamped(a.history_lens, r, a.max_history);
            for (int j = rank * kPickThreads + tid; j < nh; j += kPickCluster * kPickThreads) {
                const int id = a.history[r * a.history_stride + j];
                if (id >= 0 && id < a.vocab) atomicAdd(cl.map_shared_rank(words, id / a.slice) + id % a.slice, 1u);
            }
        }
        cl.sync();
    }
    const T* x = (const T*)a.logits + r * a.logits_stride;
    T* o = a.out ? (T*)a.out + r * a.out_stride : nullptr;
    const uint32_t* allowed = a.allowed ? a.allowed + r * a.allowed_stride : nullptr;
    Best best{-INFINITY, 0x7fffffff, 0};
    auto one = [&](float v, int t) -> float {
        if (counts || biases) {
            const uint32_t w = words[t - lo];
            if (w) {
                const uint32_t c = w & kCountMask, b = w >> kCountBits;
                if (c) {
                    v = v > 0.f ? __fdiv_rn(v, rep) : __fmul_rn(v, rep);
                    v = __fsub_rn(v, __fmul_rn(freq, (float)c));
                    v = __fsub_rn(v, pres);
                }
                if (b) v = __fadd_rn(v, a.bias_values[r * a.bias_stride + b - 1]);
            }
        }
        if (allowed && !(allowed[t >> 5] >> (t & 31) & 1u)) v = -INFINITY;
        if (v != v || v == INFINITY) best.bad = 1;
        better(best, v, t);
        return v;
    };
    // slices start at multiples of 64 tokens: a pack never straddles two
    for (int t = lo + tid * V; t < hi; t += kPickThreads * V) {
        if (V > 1 && t + V <= hi) {
            Pack<T, V> p = *reinterpret_cast<const Pack<T, V>*>(x + t);
#pragma unroll
            for (int u = 0; u < V; ++u) p.v[u] = from_f32<T>(one(to_f32(p.v[u]), t + u));
            if (o) *reinterpret_cast<Pack<T, V>*>(o + t) = p;
        } else {
            for (int u = t; u < min(t + V, hi); ++u) {
                const T y = from_f32<T>(one(to_f32(x[u]), u));
                if (o) o[u] = y;
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
        for (int w = 1; w < kPickThreads / 32; ++w) {
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

template <class T, int V>
cudaError_t launch_pick(const PickArgs& a, int rows, cudaStream_t st) {
    const size_t sm = a.history || a.bias_ids ? (size_t)a.slice * 4 : 0;
    cudaError_t e = cudaFuncSetAttribute((const void*)k_pick<T, V>, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(rows * kPickCluster));
    cfg.blockDim = dim3(kPickThreads);
    cfg.dynamicSmemBytes = sm;
    cfg.stream = st;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = kPickCluster;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, k_pick<T, V>, a);
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
    const int eb = elem_bytes(p->dtype), V = 16 / eb;
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
    a.slice = (int)((p->vocab + kPickCluster * 64 - 1) / (kPickCluster * 64) * 64);
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
    // 16-byte packs where every row starts on such a boundary
    const bool wide = aligned(p->logits, 16) && aligned(p->out, 16) &&
                      (p->rows == 1 || (p->logits_stride % V == 0 && (!p->out || p->out_stride % V == 0)));
    cudaStream_t st = (cudaStream_t)stream;
    cudaError_t e;
    if (p->dtype == QX_CUDA_F32) e = wide ? launch_pick<float, 4>(a, (int)p->rows, st) : launch_pick<float, 1>(a, (int)p->rows, st);
    else if (p->dtype == QX_CUDA_F16) e = wide ? launch_pick<__half, 8>(a, (int)p->rows, st) : launch_pick<__half, 1>(a, (int)p->rows, st);
    else e = wide ? launch_pick<__nv_bfloat16, 8>(a, (int)p->rows, st) : launch_pick<__nv_bfloat16, 1>(a, (int)p->rows, st);
    return finish(e, err, n);
}
