// Eviction of cache rows by accumulated attention weight (qx_cuda_kv_evict).
//
// k_evict_select: one CTA per (layer, sequence) finds which rows stay: a radix
// selection (8 bits at a time) of the smallest weight that still stays, then
// an ordered compaction.  k_evict_move: moves the rows.  In place the kept
// rows only ever move towards row 0, and row r's source is at or behind r, so
// a CTA that owns a column slice of a sequence can go through the kept rows in
// chunks: load a chunk, wait for its loads, store it.  What a later chunk reads lies behind
// everything stored so far.  Columns are independent, so the slices of a row
// go to different CTAs without a word between them.
#include <cmath>

#include "qx_ops.cuh"

namespace {

using namespace qx::ops;

constexpr int kSelThreads = 1024;
constexpr int kMoveThreads = 256, kMoveDepth = 4;

struct EvictArgs {
    Cache c;
    int seqs, budget, sink, recent;
    const int *slots, *dst_slots, *lens;
    float* mass;
    int *kept, *new_lens;
    uint32_t* status;
};

// Larger weight, larger key; +0 and -0 alike; NaN below every number.
__device__ __forceinline__ uint32_t weight_key(float w) {
    if (w != w) return 0u;
    const uint32_t b = __float_as_uint(w == 0.f ? 0.f : w);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// Exclusive prefix sum over the CTA of one packed pair of counts per thread.
__device__ __forceinline__ unsigned long long block_exclusive(unsigned long long v, unsigned long long* warp_sum) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    unsigned long long s = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long t = __shfl_up_sync(~0u, s, o);
        if (lane >= o) s += t;
    }
    if (lane == 31) warp_sum[w] = s;
    __syncthreads();
    if (w == 0) {
        unsigned long long t = lane < (int)(blockDim.x >> 5) ? warp_sum[lane] : 0ull, u = t;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned long long x = __shfl_up_sync(~0u, u, o);
            if (lane >= o) u += x;
        }
        warp_sum[lane] = u - t;
    }
    __syncthreads();
    return warp_sum[w] + s - v;
}

__device__ __forceinline__ bool evict_fits(const EvictArgs& a, int s) {
    const int slot = a.slots[s], dst = a.dst_slots ? a.dst_slots[s] : slot, len = a.lens[s];
    return slot >= 0 && slot < a.c.slots && dst >= 0 && dst < a.c.slots && len >= 0 && len <= a.c.ctx;
}

// 1025 weights take 8 us: bound by latency, four passes of count, scan and
// three barriers.  (Keeping the weights in registers between the passes and counting the
// first digit warp by warp took longer, 15 against 12 us with the move.)
__global__ void __launch_bounds__(kSelThreads) k_evict_select(EvictArgs a) {
    __shared__ unsigned hist[256];
    __shared__ unsigned long long warp_sum[32];
    __shared__ int clash, digit_s, need_s;
    const int s = blockIdx.x, l = blockIdx.y, tid = threadIdx.x;
    int* kept = a.kept + ((size_t)l * a.seqs + s) * a.budget;
    const int len = a.lens[s], slot = a.slots[s], dst = a.dst_slots ? a.dst_slots[s] : slot;
    const bool ok = evict_fits(a, s);
    if (tid == 0) clash = 0;
    __syncthreads();
    if (ok && len > 0)
        for (int j = tid; j < a.seqs; j += kSelThreads)
            if (j != s && evict_fits(a, j) && a.lens[j] > 0 &&
                (a.slots[j] == dst || (a.dst_slots && a.dst_slots[j] == dst)))
                clash = 1;
    __syncthreads();
    if (!ok || clash) {
        for (int r = tid; r < a.budget; r += kSelThreads) kept[r] = -1;
        if (l == 0 && tid == 0) {
            a.new_lens[s] = len;
            if (a.status) atomicOr(a.status, ok ? QX_CUDA_STATUS_SHARED : QX_CUDA_STATUS_RANGE);
        }
        return;
    }
    const int keep = min(len, a.budget);
    if (l == 0 && tid == 0) a.new_lens[s] = keep;
    if (len <= a.budget) {
        for (int r = tid; r < a.budget; r += kSelThreads) kept[r] = r < len ? r : -1;
        return;
    }
    const float* mass = a.mass + (size_t)slot * a.c.slot_rows + (size_t)l * a.c.layer_rows;
    const int first = a.sink, last = len - a.recent, n = last - first;
    int need = a.budget - a.sink - a.recent;             // rows that stay of [first, last)
    uint32_t bound = 0xffffffffu, want_eq = 0;           // stay: key > bound, and the first want_eq with key == bound
    if (need > 0) {
        uint32_t prefix = 0, mask = 0;
        for (int shift = 24; shift >= 0; shift -= 8) {
            if (tid < 256) hist[tid] = 0;
            __syncthreads();
            for (int i = tid; i < n; i += kSelThreads) {
                const uint32_t key = weight_key(mass[first + i]);
                if ((key & mask) == prefix) atomicAdd(&hist[(key >> shift) & 255u], 1u);
            }
            __syncthreads();
            if (tid < 32) {                              // the digit at which `need` is reached, from the top
                unsigned c[8], t = 0;
#pragma unroll
                for (int u = 0; u < 8; ++u) t += c[u] = hist[255 - (tid * 8 + u)];
                unsigned inc = t;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const unsigned x = __shfl_up_sync(~0u, inc, o);
                    if (tid >= o) inc += x;
                }
                unsigned above = inc - t;
                if (above < (unsigned)need && inc >= (unsigned)need) {
#pragma unroll
                    for (int u = 0; u < 8; ++u) {
                        if (above < (unsigned)need && above + c[u] >= (unsigned)need) {
                            digit_s = 255 - (tid * 8 + u);
                            need_s = need - (int)above;
                        }
                        above += c[u];
                    }
                }
            }
            __syncthreads();
            prefix |= (uint32_t)digit_s << shift;
            mask |= 255u << shift;
            need = need_s;
            __syncthreads();
        }
        bound = prefix;
        want_eq = (uint32_t)need;
    }
    // each thread a run of consecutive rows, so one scan orders all of them
    const int per = (n + kSelThreads - 1) / kSelThreads, i0 = min(n, tid * per), i1 = min(n, i0 + per);
    unsigned gt = 0, eq = 0;
    for (int i = i0; i < i1; ++i) {
        const uint32_t key = weight_key(mass[first + i]);
        gt += key > bound;
        eq += want_eq && key == bound;
    }
    const unsigned long long before = block_exclusive(((unsigned long long)gt << 32) | eq, warp_sum);
    unsigned nge = (unsigned)(before >> 32), neq = (unsigned)before;
    for (int i = i0; i < i1; ++i) {
        const uint32_t key = weight_key(mass[first + i]);
        const bool is_eq = want_eq && key == bound;
        if (key > bound || (is_eq && neq < want_eq)) kept[a.sink + nge + min(neq, want_eq)] = first + i;
        nge += key > bound;
        neq += is_eq;
    }
    for (int r = tid; r < a.sink; r += kSelThreads) kept[r] = r;
    for (int r = tid; r < a.recent; r += kSelThreads) kept[a.budget - a.recent + r] = last + r;
}

// Moves the kept rows of one column slice, kMoveDepth rows of `rows` threads'
// each to a chunk; every thread of the CTA calls it.  The next chunk's loads
// and the indexes of the one after are on their way while a chunk is stored.
template <class W>
__device__ __forceinline__ void move_columns(const W* src, W* dst, size_t row_words, int col, int row_in_chunk,
                                             int rows, const int* kept, int keep, bool live) {
    const int chunk = rows * kMoveDepth;
    W w[kMoveDepth], w_next[kMoveDepth];
    int from[kMoveDepth], from_next[kMoveDepth];
    auto index = [&](int r0, int (&f)[kMoveDepth]) {
#pragma unroll
        for (int u = 0; u < kMoveDepth; ++u) {
            const int r = r0 + u * rows + row_in_chunk;
            f[u] = live && r < keep ? kept[r] : -1;
        }
    };
    auto load = [&](const int (&f)[kMoveDepth], W (&x)[kMoveDepth]) {
#pragma unroll
        for (int u = 0; u < kMoveDepth; ++u)
            if (f[u] >= 0) x[u] = src[(size_t)f[u] * row_words + col];
    };
    index(0, from);
    load(from, w);
    index(chunk, from_next);
    for (int r0 = 0; r0 < keep; r0 += chunk) {
        int from_last[kMoveDepth];
        load(from_next, w_next);
        index(r0 + 2 * chunk, from_last);
        __syncthreads();                                 // every load of the chunk has arrived
#pragma unroll
        for (int u = 0; u < kMoveDepth; ++u) {
            const int r = r0 + u * rows + row_in_chunk;
            if (from[u] >= 0) dst[(size_t)r * row_words + col] = w[u];
            w[u] = w_next[u];
            from[u] = from_next[u];
            from_next[u] = from_last[u];
        }
    }
}

// Bound by the memory where there is much to move: 48 layers of 8 sequences of
// 4096 rows, half of them kept, are 1.6 GB, 250 us at the memory's rate, and take 307 us.  A single
// sequence is bound by the chain of index, load and store per chunk: slices of
// 32 bytes make 128 rows of 256 threads' accesses instead of 32, and four times the CTAs (8192
// rows of one layer, with the selection: 20 us, against 74 us for slices of 128 bytes without
// the loads ahead).
//
// grid: (sequence, layer, slice); slices of 16 LANES bytes of K, then of V,
// then the key scales, the value scales and the mass.
template <int LANES>
__global__ void __launch_bounds__(kMoveThreads) k_evict_move(const __grid_constant__ EvictArgs a) {
    const int s = blockIdx.x, l = blockIdx.y, tid = threadIdx.x;
    const int* kept = a.kept + ((size_t)l * a.seqs + s) * a.budget;
    asm volatile("griddepcontrol.wait;" ::: "memory");   // launched while the selection still runs
    if (!evict_fits(a, s)) return;
    const int len = a.lens[s], slot = a.slots[s], dst = a.dst_slots ? a.dst_slots[s] : slot, keep = min(len, a.budget);
    if (keep == 0 || kept[0] < 0) return;                // nothing there, or left out
    if (dst == slot && len <= a.budget) return;
    const size_t from = (size_t)slot * a.c.slot_rows + (size_t)l * a.c.layer_rows;
    const size_t to = (size_t)dst * a.c.slot_rows + (size_t)l * a.c.layer_rows;
    const int KV = a.c.kv_heads * a.c.head_dim, slices = (KV / 16 + LANES - 1) / LANES;
    int slice = blockIdx.z;
    if (slice < 2 * slices) {
        const bool isv = slice >= slices;
        if (isv) slice -= slices;
        int8_t* base = isv ? a.c.v : a.c.k;
        const int col = tid % LANES + slice * LANES;
        const bool live = col < KV / 16;
        move_columns<uint4>((const uint4*)(base + from * KV), (uint4*)(base + to * KV), (size_t)KV / 16, live ? col : 0,
                            tid / LANES, kMoveThreads / LANES, kept, keep, live);
        return;
    }
    float* col = slice == 2 * slices ? a.c.ks : slice == 2 * slices + 1 ? a.c.vs : a.mass;
    move_columns<float>(col + from, col + to, 1, 0, tid, kMoveThreads, kept, keep, true);
    if (slice == 2 * slices + 2) {
        __syncthreads();
        for (int r = keep + tid; r < len; r += kMoveThreads) a.mass[to + r] = 0.f;
    }
}

template <int LANES>
cudaError_t launch_move(const EvictArgs& a, cudaStream_t st) {
    const unsigned slices = (unsigned)(a.c.kv_heads * a.c.head_dim / 16 + LANES - 1) / LANES;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)a.seqs, (unsigned)a.c.layers, 2 * slices + 3);
    cfg.blockDim = dim3(kMoveThreads);
    cfg.stream = st;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, k_evict_move<LANES>, a);
}

}  // namespace

QX_API int qx_cuda_kv_evict(const qx_cuda_kv_cache* cache, uint32_t seqs, const int32_t* slots, const int32_t* dst_slots,
                            const int32_t* lens, float* mass, uint32_t budget, uint32_t sink, uint32_t recent,
                            int32_t* kept, int32_t* new_lens, uint32_t* status, void* stream, char* err, uint64_t n) {
    if (const char* m = check_cache(cache)) return refuse(err, n, m);
    if (!slots || !lens || !mass || !kept || !new_lens) return refuse(err, n, "invalid eviction argument");
    if (!seqs || seqs > kMaxSeqs) return refuse(err, n, "1 to 4096 sequences");
    if (!budget || (uint64_t)sink + recent > budget) return refuse(err, n, "sink + recent must fit the budget, which is at least 1");
    if (budget > 1u << 24) return refuse(err, n, "the budget is larger than any cache");
    if (new_lens == lens) return refuse(err, n, "new_lens may not be lens itself");
    for (const void* p : {(const void*)slots, (const void*)dst_slots, (const void*)lens, (const void*)mass,
                          (const void*)kept, (const void*)new_lens, (const void*)status})
        if (!aligned(p, 4)) return refuse(err, n, "eviction buffers must be 4-byte aligned");
    DeviceOf dev(cache->k, err, n);
    if (!dev.ok) return 0;
    EvictArgs a{cache_of(cache), (int)seqs, (int)budget, (int)sink, (int)recent, slots, dst_slots, lens, mass, kept,
                new_lens, status};
    cudaStream_t st = (cudaStream_t)stream;
    k_evict_select<<<dim3(seqs, cache->layers), kSelThreads, 0, st>>>(a);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return finish(e, err, n);
    const uint64_t slices = ((uint64_t)cache->kv_heads * cache->head_dim + 127) / 128;
    // slices of 32 bytes while those of 128 would leave SMs without two CTAs
    const bool few = seqs * (uint64_t)cache->layers * 2 * slices < 2 * 148;
    return finish(few ? launch_move<2>(a, st) : launch_move<8>(a, st), err, n);
}
