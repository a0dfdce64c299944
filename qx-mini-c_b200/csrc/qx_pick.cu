// Penalties, biases and a grammar mask on logits, and the greedy token of each
// row (qx_cuda_pick_tokens).
//
// A cluster of CTAs takes row after row; each CTA owns a slice of the
// vocabulary (of eight CTAs every eighth 64 tokens: frequent tokens lie together, and one CTA
// with all of them held the others up, 131 us against 111 for 256 rows of
// 151936) and keeps one 32-bit word per token of it in shared memory: the
// token's count in the history (low 20 bits) and the last bias entry that names
// it, plus one (high 12 bits).  Every CTA reads the whole history and counts
// what falls in its slice: counting an eighth each into the others' memory reads
// less, but histories repeat few tokens, whose CTA then takes thousands of
// single remote additions (256 rows of 151936 with histories of 4096: 155 us,
// where this way took 135).  Integer atomics, so the order they land in changes
// nothing.  Then each CTA streams its slice of the logits once, putting the
// words it finds back to 0 for the next row, and leaves its best with the
// cluster's first CTA, which joins a row's parts while the next is counted: no
// workspace, one launch, and no wait between rows that the next row's first
// loads do not overlap.
//
// 256 rows of 151936 F32 logits with a mask, 64 biases and histories of 4096
// move 311 MB, 49 us at the memory's rate, and take 111 us, bound by
// instructions and the latency of a row's steps: of each 128 tokens a warp looks at, three or four are in the
// history (a branch for each of a lane's four words instead of a loop over those that are: 113 us).  Dearer were: a queue
// of such tokens per warp, emptied 32 at a time (134 us: its scans), and a second
// walk over the history that changes them after the pass (134 us: it reads
// every id again in every CTA).
//
// Rows need not start on 16-byte boundaries: a row's tokens are numbered from
// the boundary before it ("places"), and slices and packs are of places.
#include <cooperative_groups.h>

#include <cmath>

#include "qx_ops.cuh"

namespace {

using namespace qx::ops;
namespace cg = cooperative_groups;

constexpr uint32_t kMaxVocab = 393216, kCountBits = 20, kCountMask = (1u << kCountBits) - 1;

struct PickArgs {
    const void* logits;
    void* out;
    size_t logits_stride, out_stride;
    int rows, vocab, slice, max_history, max_bias;
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

// The cluster's barrier, its two halves apart.
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }
__device__ __forceinline__ bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
__device__ __forceinline__ int clamped(const int* lens, int r, int most) {
    return lens ? max(0, min(lens[r], most)) : most;
}

// Of a cluster of CL CTAs, place p is word p / (64 CL) * 64 + p % 64 of CTA p / 64 % CL.
constexpr int kChunk = 64;
template <int CL>
__device__ __forceinline__ int place_of(int word, int rank) {
    return word / kChunk * (kChunk * CL) + rank * kChunk + word % kChunk;
}

// A row's addresses, and where its tokens are.
template <class T>
struct Row {
    static constexpr int V = 16 / sizeof(T);
    const T* x;
    T* o;
    const uint32_t* allowed;
    int shift, end;                  // token t is at place t + shift; the row ends before place `end`
    bool wide_out;
    __device__ __forceinline__ Row(const PickArgs& a, int row) {
        x = (const T*)a.logits + row * a.logits_stride;
        o = a.out ? (T*)a.out + row * a.out_stride : nullptr;
        allowed = a.allowed ? a.allowed + row * a.allowed_stride : nullptr;
        shift = (int)(reinterpret_cast<uintptr_t>(x) / sizeof(T) % V);
        wide_out = o && (int)(reinterpret_cast<uintptr_t>(o) / sizeof(T) % V) == shift;
        end = a.vocab + shift;
    }
    __device__ __forceinline__ bool whole(int p) const { return p >= shift && p + V <= end; }
    // a pack's logits, and the mask word of its first token
    __device__ __forceinline__ void load(int p, Pack<T, V>& v, uint32_t& bits) const {
        if (whole(p)) {
            v = *reinterpret_cast<const Pack<T, V>*>(x + (p - shift));
            bits = allowed ? allowed[(p - shift) >> 5] : ~0u;
        }
    }
};

// Words of a CTA: of vocab and up to 7 places before it.
inline int slice_of(int vocab, int ctas) { return (vocab + 7 + kChunk * ctas - 1) / (kChunk * ctas) * kChunk; }

template <class T, int THREADS, int CL>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) k_pick(const __grid_constant__ PickArgs a) {
    constexpr int V = 16 / sizeof(T), kAhead = V == 4 ? 3 : 1, kRound = kChunk * CL;   // kAhead: packs a thread has in flight
    extern __shared__ __align__(16) uint32_t words[];
    __shared__ Best wbest[THREADS / 32], row_best[2][CL];     // row_best: in the cluster's first CTA
    cg::cluster_group cl = cg::this_cluster();
    const int rank = (int)cl.block_rank(), step = gridDim.x / CL, tid = threadIdx.x;
    const bool touched = a.history || a.bias_ids;
    cluster_arrive();                                        // this CTA has started: its memory may be written by the others
    if (touched) {
        for (int i = tid * 4; i < a.slice; i += THREADS * 4) *reinterpret_cast<uint4*>(words + i) = make_uint4(0, 0, 0, 0);
        __syncthreads();
    }
    // the best of the row before, whose eight parts are in once its barrier is passed
    auto join = [&](int r, int slot) {
        if (rank || tid) return;
        Best best = row_best[slot][0];
        for (int c = 1; c < CL; ++c) {
            better(best, row_best[slot][c].v, row_best[slot][c].i);
            best.bad |= row_best[slot][c].bad;
        }
        a.picked[r] = best.bad || !(best.v > -INFINITY) ? 0xffffffffu : (uint32_t)best.i;
    };
    Pack<T, V> pack[kAhead];
    uint32_t bits[kAhead];
    const int first = blockIdx.x / CL;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) Row<T>(a, first).load(place_of<CL>((i * THREADS + tid) * V, rank), pack[i], bits[i]);
    int slot = 0;
    for (int r = first; r < a.rows; r += step, slot ^= 1) {
        const Row<T> row(a, r);
        const int shift = row.shift;
        const float rep = a.repetition ? a.repetition[r] : 1.f, freq = a.frequency ? a.frequency[r] : 0.f,
                    pres = a.presence ? a.presence[r] : 0.f;
        if (touched) {
            // the word of a token, if it is this CTA's
            auto word = [&](int id) -> uint32_t* {
                const int p = id + shift;
                return (unsigned)id < (unsigned)a.vocab && (p / kChunk) % CL == rank ? words + p / kRound * kChunk + p % kChunk
                                                                                             : nullptr;
            };
            if (a.bias_ids) {
                const int nb = clamped(a.bias_lens, r, a.max_bias);
                for (int j = tid; j < nb; j += THREADS)
                    if (uint32_t* w = word(a.bias_ids[r * a.bias_stride + j])) atomicMax(w, (uint32_t)(j + 1) << kCountBits);
                __syncthreads();
            }
            if (a.history) {
                const int nh = clamped(a.history_lens, r, a.max_history);
                const int* h = a.history + r * a.history_stride;
                auto count = [&](int id) {
                    if (uint32_t* w = word(id)) atomicAdd(w, 1u);
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
        }
        cluster_wait();                                                  // first row: every CTA has started
        if (r != first) join(r - step, slot ^ 1);
        __syncthreads();
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
        for (int w0 = tid * V; place_of<CL>(w0, rank) < row.end; w0 += kAhead * THREADS * V) {
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                const int at = w0 + i * THREADS * V, p = place_of<CL>(at, rank), t = p - shift, later = place_of<CL>(at + kAhead * THREADS * V, rank);
                if (row.whole(p)) {
                    float v[V];
#pragma unroll
                    for (int u = 0; u < V; ++u) v[u] = to_f32(pack[i].v[u]);
                    uint32_t ok = bits[i];
                    if (row.allowed) {                                       // the pack's bits, which two words may hold
                        ok >>= t & 31;
                        if ((t & 31) + V > 32) ok = __funnelshift_r(bits[i], row.allowed[(t >> 5) + 1], t & 31);
                    }
                    row.load(later, pack[i], bits[i]);                       // on its way while this one is worked on
                    if (touched)
#pragma unroll
                        for (int u = 0; u < V; u += 4) {
                            uint4* word4 = reinterpret_cast<uint4*>(words + at + u);
                            const uint4 q = *word4;
                            if (q.x | q.y | q.z | q.w) {
                                *word4 = make_uint4(0, 0, 0, 0);
                                uint32_t left = (q.x ? 1u : 0u) | (q.y ? 2u : 0u) | (q.z ? 4u : 0u) | (q.w ? 8u : 0u);
                                do {                                         // most lanes that have one have no other
                                    const bool hi = !(left & 3u), odd = !(left & (hi ? 4u : 1u));
                                    const uint32_t w = hi ? (odd ? q.w : q.z) : (odd ? q.y : q.x);
                                    const float x = touch(hi ? (odd ? v[u + 3] : v[u + 2]) : (odd ? v[u + 1] : v[u]), w);
                                    if (!hi && !odd) v[u] = x;
                                    if (!hi && odd) v[u + 1] = x;
                                    if (hi && !odd) v[u + 2] = x;
                                    if (hi && odd) v[u + 3] = x;
                                    left &= left - 1;
                                } while (left);
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
                    if (row.wide_out) {
                        *reinterpret_cast<Pack<T, V>*>(row.o + t) = y;
                    } else if (row.o) {
#pragma unroll
                        for (int u = 0; u < V; ++u) row.o[t + u] = y.v[u];
                    }
                } else {
                    if (p < row.end)
#pragma unroll 1
                        for (int u = 0; u < V; ++u) {                        // the row's ends
                            const int e = t + u;
                            if (e < 0 || e >= a.vocab) continue;
                            float v = to_f32(row.x[e]);
                            if (touched && words[at + u]) {
                                v = touch(v, words[at + u]);
                                words[at + u] = 0;
                            }
                            if (row.allowed && !(row.allowed[e >> 5] >> (e & 31) & 1u)) v = -INFINITY;
                            best.bad |= !(v < INFINITY);
                            if (v > best.v) best.v = v, best.i = e;
                            if (row.o) row.o[e] = from_f32<T>(v);
                        }
                    row.load(later, pack[i], bits[i]);
                }
            }
        }
        if (r + step < a.rows) {                                         // the next row's first packs
            const Row<T> next(a, r + step);
#pragma unroll
            for (int i = 0; i < kAhead; ++i) next.load(place_of<CL>((i * THREADS + tid) * V, rank), pack[i], bits[i]);
        }
        for (int s = 16; s; s >>= 1) {
            const float v = __shfl_xor_sync(~0u, best.v, s);
            const int i = __shfl_xor_sync(~0u, best.i, s);
            better(best, v, i);
        }
        best.bad = __any_sync(~0u, best.bad);
        if ((tid & 31) == 0) wbest[tid >> 5] = best;
        __syncthreads();                                                 // and every word is 0 again
        if (tid == 0) {
            for (int w = 1; w < THREADS / 32; ++w) {
                better(best, wbest[w].v, wbest[w].i);
                best.bad |= wbest[w].bad;
            }
            *cl.map_shared_rank(&row_best[slot][rank], 0) = best;
        }
        __syncwarp();
        cluster_arrive();
    }
    cluster_wait();                                                      // the first CTA's memory lives until all have left theirs
    const int rows = (a.rows - first + step - 1) / step;
    join(first + (rows - 1) * step, slot ^ 1);
}

template <class T, int THREADS, int CL>
cudaError_t launch_pick(PickArgs a, cudaStream_t st) {
    a.slice = slice_of(a.vocab, CL);
    const size_t sm = a.history || a.bias_ids ? (size_t)a.slice * 4 : 0;
    cudaError_t e = cudaFuncSetAttribute((const void*)k_pick<T, THREADS, CL>, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = sm;
    cfg.stream = st;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = CL;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    int clusters = 1;
    if (a.rows > 1) {
        cfg.gridDim = dim3((unsigned)(a.rows * CL));
        e = cudaOccupancyMaxActiveClusters(&clusters, k_pick<T, THREADS, CL>, &cfg);
        if (e != cudaSuccess) return e;
        if (clusters < 1) clusters = 1;
        if (clusters > a.rows) clusters = a.rows;
    }
    cfg.gridDim = dim3((unsigned)(clusters * CL));
    return cudaLaunchKernelEx(&cfg, k_pick<T, THREADS, CL>, a);
}

template <class T>
cudaError_t run_pick(const PickArgs& a, cudaStream_t st) {
    // Few rows leave SMs to spare: one CTA of 1024 threads each.  Else two of 512.
    if (a.rows * 8 <= 148) return launch_pick<T, 1024, 8>(a, st);
    // More rows than there are clusters: smaller ones read the histories less often and wait for fewer, if two of their
    // larger slices fit an SM (256 rows of 32000 took 33 us by clusters of four, take 25 by two; 64 rows of 50257 took
    // 17 us by eight, take 12 by four; one CTA of 1024 threads with a slice of a quarter was no faster for rows of 151936).
    if (a.rows * 4 > 2 * 148 && slice_of(a.vocab, 2) * 4 <= 100 * 1024) return launch_pick<T, 512, 2>(a, st);
    if (a.rows * 8 > 2 * 148 && slice_of(a.vocab, 4) * 4 <= 100 * 1024) return launch_pick<T, 512, 4>(a, st);
    return launch_pick<T, 512, 8>(a, st);
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
    a.rows = (int)p->rows;
    a.vocab = (int)p->vocab;
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
    cudaError_t e;
    if (p->dtype == QX_CUDA_F32) e = run_pick<float>(a, st);
    else if (p->dtype == QX_CUDA_F16) e = run_pick<__half>(a, st);
    else e = run_pick<__nv_bfloat16>(a, st);
    return finish(e, err, n);
}
