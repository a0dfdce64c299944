// Rotary positions of drafted tokens and their quantized append to the INT8
// cache (qx_cuda_rope_append), and the frequencies of the context-extension
// schemes (qx_cuda_rope_frequencies).
//
// With a = position * inv_freq[i] (one double product), c = amplitude cos a,
// s = amplitude sin a, a pair (x0, x1) becomes (x0 c - x1 s, x0 s + x1 c).
// Keys turn in double without contraction and are rounded to F32, the engine's
// own order (head_norm_rope), so that a code does not depend on how a product
// was fused; queries turn in F32 with c and s rounded to F32, since nothing
// is quantized from them and their result is rounded to F32 or less anyway.
#include <cmath>

#include "qx_ops.cuh"

namespace {

using namespace qx::ops;


struct Heads {
    const void* p;
    size_t seq, node, head;
};


// A tensor's items for V-wide accesses: first every head's `pairs` items of V
// rotated pairs (half layout: V values at i and V at rd / 2 + i; interleaved:
// 2 V consecutive values), then every head's `pass` items of V values that go
// through, so that a warp mostly has items of one kind.
struct Items {
    Over pairs, pass;
    int rotated;                                         // in all heads
    // head, item within it
    __device__ __forceinline__ bool at(int w, int& h, int& it) const {
        const bool rot = w < rotated;
        const Over& o = rot ? pairs : pass;
        const uint32_t x = rot ? w : w - rotated;
        h = (int)o(x);
        it = (int)(x - h * o.d);
        return rot;
    }
};
template <class T, int V, bool IL>
__device__ __forceinline__ void load_item(const T* h, int item, int rd, bool rot, T (&a)[V], T (&b)[V]) {
    const int i0 = rot ? (IL ? 2 * V * item : V * item) : rd + V * item;
    const int i1 = IL ? i0 + V : rd / 2 + i0;
    const Pack<T, V> x = *reinterpret_cast<const Pack<T, V>*>(h + i0);
#pragma unroll
    for (int u = 0; u < V; ++u) a[u] = x.v[u];
    if (rot) {
        const Pack<T, V> y = *reinterpret_cast<const Pack<T, V>*>(h + i1);
#pragma unroll
        for (int u = 0; u < V; ++u) b[u] = y.v[u];
    }
}

struct RopeArgs {
    Cache c;
    Drafts d;
    int layer, q_heads, rd, interleaved;
    const double* inv_freq;
    double amplitude;
    Heads q, qo, k, v;
    Items q_items, k_items;
    Over v_packs;                                        // V-wide packs of a head
    const int* positions;
    float* mass;                                         // 0 for an appended row, or null
    uint32_t* status;
};

// rint(x / scale), clamped, for |x| <= 127.5 scale.  The product with 1 / scale
// is within 2^-21 of the quotient's size, so below 2^-14 of it, and rounds to
// the same integer unless that near a half; then the quotient itself decides.
__device__ __forceinline__ int code_of(float x, float scale, float inv) {
    if (!isfinite(x)) return 0;
    const float q = x * inv;
    float r = rintf(q);
    if (!(fabsf(q - r) < 0.5f - 0x1p-14f)) r = rintf(__fdiv_rn(x, scale));
    return max(-127, min(127, (int)r));
}

// One CTA per drafted token: a token's 40 heads of 128 are 10 KB, read once
// into registers (queries) or shared memory as F32 (keys and values, which
// need their row's largest magnitude before they can be quantized).
//
// A prompt of 4096 tokens moves 76 MB, 12 us at the memory's rate, and takes
// 28 us fully rotated, 24 us with half of each head rotated in pairs.  What is left is a token's chain: the
// scheduler issues in 48 and 52 of 100 cycles, and warps wait most for loads and
// at the barrier behind the sines, which a part of the threads works out in
// double.  8 CTAs to an SM and one item ahead did best: 2 items 33 us, 3 items
// and 5 CTAs 40 us.
template <class T, int V, bool IL, int THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) k_rope_append(RopeArgs a) {
    extern __shared__ __align__(16) float kvrow[];       // [2][kv]: rotated key, value
    __shared__ double cs_d[2][256 + 1];
    __shared__ float cs_f[2][256 + 1];
    __shared__ float wmax[2][THREADS / 32];
    __shared__ int clash;
    const int node = blockIdx.x, s = blockIdx.y, tid = threadIdx.x;
    const int D = a.c.head_dim, KV = a.c.kv_heads * D, rd = a.rd, half = rd / 2;
    const int slot = a.d.slots[s], len = a.d.lens[s], n = a.d.count(s);
    const bool ok = fits(a.c, a.d, slot, len, n);
    if (!ok) {
        if (node == 0 && tid == 0 && a.status) atomicOr(a.status, QX_CUDA_STATUS_RANGE);
        return;
    }
    if (node >= n) return;
    if (tid == 0) clash = 0;
    const int pos = a.positions ? a.positions[(size_t)s * a.d.max_nodes + node] : len + node;
    const T* qp = (const T*)a.q.p + s * a.q.seq + node * a.q.node;
    const T* kp = (const T*)a.k.p + s * a.k.seq + node * a.k.node;
    const T* vp = (const T*)a.v.p + s * a.v.seq + node * a.v.node;
    const int per_head = (IL ? rd / (2 * V) : half / V) + (D - rd) / V;
    const int k_items = a.k.p ? a.c.kv_heads * per_head : 0, v_packs = a.k.p ? KV / V : 0, q_items = a.q.p ? a.q_heads * per_head : 0;
    auto load_k = [&](int w, T (&x)[V], T (&y)[V]) {
        int h, it;
        const bool rot = a.k_items.at(w, h, it);
        load_item<T, V, IL>(kp + h * a.k.head, it, rd, rot, x, y);
    };
    auto load_q = [&](int w, T (&x)[V], T (&y)[V]) {
        int h, it;
        const bool rot = a.q_items.at(w, h, it);
        load_item<T, V, IL>(qp + h * a.q.head, it, rd, rot, x, y);
    };
    auto load_v = [&](int w) {
        const int h = (int)a.v_packs(w);
        return *reinterpret_cast<const Pack<T, V>*>(vp + h * a.v.head + (w * V - h * D));
    };
    // a thread's first items are on their way before the sines are worked out
    T kx[V], ky[V], qx[V], qy[V];
    Pack<T, V> vx;
    if (tid < k_items) load_k(tid, kx, ky);
    if (tid < v_packs) vx = load_v(tid);
    if (tid < q_items) load_q(tid, qx, qy);
    for (int i = tid; i < half; i += THREADS) {
        double sn, cn;
        sincos(__dmul_rn((double)pos, a.inv_freq[i]), &sn, &cn);
        cs_f[0][i] = (float)(cs_d[0][i] = __dmul_rn(cn, a.amplitude));
        cs_f[1][i] = (float)(cs_d[1][i] = __dmul_rn(sn, a.amplitude));
    }
    __syncthreads();
    if (a.k.p)                                           // another sequence of the call that appends to this slot
        for (int j = tid; j < a.d.seqs; j += THREADS)
            if (j != s && a.d.slots[j] == slot) {
                const int m = a.d.count(j);
                if (m > 0 && fits(a.c, a.d, slot, a.d.lens[j], m)) clash = 1;
            }
    float ka = 0.f, va = 0.f;
    if (a.k.p) {
        auto key = [&](int w, const T (&x)[V], const T (&y)[V]) {
            int h, it;
            const bool rot = a.k_items.at(w, h, it);
            float* o = kvrow + h * D;
            if (rot) {
#pragma unroll
                for (int u = 0; u < V; ++u) {
                    // the u-th pair of the item, and where its halves lie
                    const int p = V * it + u;
                    const float x0 = IL ? (2 * u < V ? to_f32(x[(2 * u) % V]) : to_f32(y[(2 * u) % V])) : to_f32(x[u]);
                    const float x1 = IL ? (2 * u + 1 < V ? to_f32(x[(2 * u + 1) % V]) : to_f32(y[(2 * u + 1) % V])) : to_f32(y[u]);
                    const double c = cs_d[0][p], sn = cs_d[1][p];
                    const float r0 = (float)__dsub_rn(__dmul_rn((double)x0, c), __dmul_rn((double)x1, sn));
                    const float r1 = (float)__dadd_rn(__dmul_rn((double)x0, sn), __dmul_rn((double)x1, c));
                    o[IL ? 2 * p : p] = r0;
                    o[IL ? 2 * p + 1 : half + p] = r1;
                    ka = fmaxf(ka, isfinite(r0) ? fabsf(r0) : 0.f);
                    ka = fmaxf(ka, isfinite(r1) ? fabsf(r1) : 0.f);
                }
            } else {
#pragma unroll
                for (int u = 0; u < V; ++u) {
                    const float r = to_f32(x[u]);
                    o[rd + V * it + u] = r;
                    ka = fmaxf(ka, isfinite(r) ? fabsf(r) : 0.f);
                }
            }
        };
        auto value = [&](int w, const Pack<T, V>& x) {
#pragma unroll
            for (int u = 0; u < V; ++u) {
                const float r = to_f32(x.v[u]);
                kvrow[KV + w * V + u] = r;
                va = fmaxf(va, isfinite(r) ? fabsf(r) : 0.f);
            }
        };
        if (tid < k_items) key(tid, kx, ky);
        for (int w = tid + THREADS; w < k_items; w += THREADS) {
            T x[V], y[V];
            load_k(w, x, y);
            key(w, x, y);
        }
        if (tid < v_packs) value(tid, vx);
        for (int w = tid + THREADS; w < v_packs; w += THREADS)
            value(w, load_v(w));
        for (int o = 16; o; o >>= 1) {
            ka = fmaxf(ka, __shfl_xor_sync(~0u, ka, o));
            va = fmaxf(va, __shfl_xor_sync(~0u, va, o));
        }
        if ((tid & 31) == 0) wmax[0][tid >> 5] = ka, wmax[1][tid >> 5] = va;
    }
    __syncthreads();
    if (clash) {
        if (node == 0 && tid == 0 && a.status) atomicOr(a.status, QX_CUDA_STATUS_SHARED);
        return;
    }
    if (a.q.p) {
        T* qo = (T*)const_cast<void*>(a.qo.p) + s * a.qo.seq + node * a.qo.node;
        auto query = [&](int w, const T (&x)[V], const T (&y)[V]) {
            int h, it;
            const bool rot = a.q_items.at(w, h, it);
            T* o = qo + h * a.qo.head;
            Pack<T, V> ox, oy;
            if (rot) {
#pragma unroll
                for (int u = 0; u < V; ++u) {
                    const int p = V * it + u;
                    const float x0 = IL ? (2 * u < V ? to_f32(x[(2 * u) % V]) : to_f32(y[(2 * u) % V])) : to_f32(x[u]);
                    const float x1 = IL ? (2 * u + 1 < V ? to_f32(x[(2 * u + 1) % V]) : to_f32(y[(2 * u + 1) % V])) : to_f32(y[u]);
                    const float c = cs_f[0][p], sn = cs_f[1][p];
                    const T r0 = from_f32<T>(x0 * c - x1 * sn), r1 = from_f32<T>(x0 * sn + x1 * c);
                    if (IL) {
                        if (2 * u < V) ox.v[(2 * u) % V] = r0; else oy.v[(2 * u) % V] = r0;
                        if (2 * u + 1 < V) ox.v[(2 * u + 1) % V] = r1; else oy.v[(2 * u + 1) % V] = r1;
                    } else {
                        ox.v[u] = r0;
                        oy.v[u] = r1;
                    }
                }
                const int i0 = IL ? 2 * V * it : V * it;
                *reinterpret_cast<Pack<T, V>*>(o + i0) = ox;
                *reinterpret_cast<Pack<T, V>*>(o + (IL ? i0 + V : half + i0)) = oy;
            } else {
#pragma unroll
                for (int u = 0; u < V; ++u) ox.v[u] = x[u];
                *reinterpret_cast<Pack<T, V>*>(o + rd + V * it) = ox;
            }
        };
        if (tid < q_items) query(tid, qx, qy);
        for (int w = tid + THREADS; w < q_items; w += THREADS) {
            T x[V], y[V];
            load_q(w, x, y);
            query(w, x, y);
        }
    }
    if (!a.k.p) return;
    ka = va = 0.f;
    for (int w = 0; w < THREADS / 32; ++w) {
        ka = fmaxf(ka, wmax[0][w]);
        va = fmaxf(va, wmax[1][w]);
    }
    float ksc = __fdiv_rn(ka, 127.0f), vsc = __fdiv_rn(va, 127.0f);
    if (!(ksc > 0.f)) ksc = 1.0f;                        // a row of zeros, or one whose quotient underflows
    if (!(vsc > 0.f)) vsc = 1.0f;
    const size_t row = (size_t)slot * a.c.slot_rows + (size_t)a.layer * a.c.layer_rows + (size_t)(len + node);
    for (int w = tid; w < 2 * KV / 4; w += THREADS) {
        const bool isv = w >= KV / 4;
        const float4 x = *reinterpret_cast<const float4*>(kvrow + 4 * w);
        const float sc = isv ? vsc : ksc, inv = 1.0f / sc;
        uint32_t word = 0;
        const float e[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            word |= (uint32_t)(uint8_t)(int8_t)code_of(e[u], sc, inv) << (8 * u);
        }
        reinterpret_cast<uint32_t*>((isv ? a.c.v : a.c.k) + row * KV)[isv ? w - KV / 4 : w] = word;
    }
    if (tid == 0) {
        a.c.ks[row] = ksc;
        a.c.vs[row] = vsc;
        if (a.mass) a.mass[row] = 0.f;
    }
}

template <class T, int V>
cudaError_t launch_rope(RopeArgs a, cudaStream_t st) {
    const uint32_t pairs = (uint32_t)a.rd / (2 * V), pass = (uint32_t)(a.c.head_dim - a.rd) / V;
    a.q_items = {Over(pairs), Over(pass ? pass : 1), (int)(a.q_heads * pairs)};
    a.k_items = {Over(pairs), Over(pass ? pass : 1), (int)(a.c.kv_heads * pairs)};
    a.v_packs = Over((uint32_t)a.c.head_dim / V);
    const dim3 grid((unsigned)a.d.max_nodes, (unsigned)a.d.seqs);
    const size_t sm = a.k.p ? (size_t)2 * a.c.kv_heads * a.c.head_dim * 4 : 0;
    // 256 threads a token while all of them run at once (one token 5.6 -> 4.8 us, 64 trees of 16 nodes 7.5 -> 6.9 us; a
    // prompt of 4096 tokens 28 -> 37 us)
    const bool few = (uint64_t)a.d.max_nodes * a.d.seqs <= 148 * 8;
    auto fn = a.interleaved ? (few ? k_rope_append<T, V, true, 256> : k_rope_append<T, V, true, 128>)
                            : (few ? k_rope_append<T, V, false, 256> : k_rope_append<T, V, false, 128>);
    cudaError_t e = cudaSuccess;
    // what the widest row needs, whatever this one does: the attribute is every thread's, and another may be about to launch
    if (sm > 40 * 1024) e = cudaFuncSetAttribute((const void*)fn, cudaFuncAttributeMaxDynamicSharedMemorySize, 2 * kMaxRow * 4);
    if (e != cudaSuccess) return e;
    fn<<<grid, few ? 256 : 128, sm, st>>>(a);
    return cudaGetLastError();
}

bool packs(const qx_cuda_heads* t, int v, int eb) {
    return !t || !t->data || (aligned(t->data, 16) && t->seq_stride % v == 0 && t->node_stride % v == 0 &&
                              t->head_stride % v == 0 && v * eb == 16);
}

}  // namespace

QX_API int qx_cuda_rope_frequencies(uint32_t scheme, uint32_t rotary_dim, double base, double factor,
                                    double original_ctx, double low, double high, double* inv_freq, double* amplitude,
                                    char* err, uint64_t n) {
    if (!inv_freq || !amplitude) return refuse(err, n, "invalid rotary argument");
    if (scheme > QX_CUDA_ROPE_BANDS) return refuse(err, n, "unknown rotary scaling scheme");
    if (rotary_dim < 2 || rotary_dim % 2 || rotary_dim > 512) return refuse(err, n, "rotary_dim must be even, 2 to 512");
    if (!(base > 1.0) || !std::isfinite(base)) return refuse(err, n, "the rotary base must be above 1");
    if (scheme != QX_CUDA_ROPE_NONE && (!(factor >= 1.0) || !std::isfinite(factor)))
        return refuse(err, n, "the scaling factor must be at least 1");
    if (scheme >= QX_CUDA_ROPE_YARN && (!(original_ctx >= 1.0) || !(low > 0.0) || !(high > low) ||
                                        !std::isfinite(original_ctx) || !std::isfinite(high)))
        return refuse(err, n, "scaling by parts needs original_ctx >= 1 and 0 < low < high");
    if (scheme == QX_CUDA_ROPE_NTK && rotary_dim == 2) return refuse(err, n, "NTK scaling needs rotary_dim above 2");
    const double rd = rotary_dim, two_pi = 6.283185307179586476925286766559;
    if (scheme == QX_CUDA_ROPE_NTK) base *= pow(factor, rd / (rd - 2.0));
    // the dimension whose pair turns r times within original_ctx
    auto dim_of = [&](double r) { return rd * log(original_ctx / (r * two_pi)) / (2.0 * log(base)); };
    double first = 0.0, last = 0.0;
    if (scheme == QX_CUDA_ROPE_YARN) {
        first = std::fmax(floor(dim_of(high)), 0.0);
        last = std::fmin(ceil(dim_of(low)), rd - 1.0);
        if (last <= first) last = first + 0.001;
    }
    for (uint32_t i = 0; i < rotary_dim / 2; ++i) {
        const double f = pow(base, -2.0 * (double)i / rd);
        double w = 0.0;                                  // the share of the slowed frequency
        if (scheme == QX_CUDA_ROPE_LINEAR) w = 1.0;
        if (scheme == QX_CUDA_ROPE_YARN) w = std::fmin(std::fmax(((double)i - first) / (last - first), 0.0), 1.0);
        if (scheme == QX_CUDA_ROPE_BANDS)
            w = 1.0 - std::fmin(std::fmax((original_ctx * f / two_pi - low) / (high - low), 0.0), 1.0);
        inv_freq[i] = w == 0.0 ? f : w == 1.0 ? f / factor : f * (1.0 - w) + f / factor * w;
    }
    *amplitude = scheme == QX_CUDA_ROPE_YARN ? 0.1 * log(factor) + 1.0 : 1.0;
    return 1;
}

QX_API int qx_cuda_rope_append(const qx_cuda_kv_cache* cache, uint32_t layer, const qx_cuda_drafts* drafts,
                               const qx_cuda_rotary* rotary, uint32_t dtype, uint32_t q_heads, const qx_cuda_heads* q,
                               const qx_cuda_heads* q_out, const qx_cuda_heads* k, const qx_cuda_heads* v,
                               const int32_t* positions, uint32_t* status, void* stream, char* err, uint64_t n) {
    return qx_cuda_rope_append_mass(cache, layer, drafts, rotary, dtype, q_heads, q, q_out, k, v, positions, nullptr, status,
                                    stream, err, n);
}

QX_API int qx_cuda_rope_append_mass(const qx_cuda_kv_cache* cache, uint32_t layer, const qx_cuda_drafts* drafts,
                                    const qx_cuda_rotary* rotary, uint32_t dtype, uint32_t q_heads, const qx_cuda_heads* q,
                                    const qx_cuda_heads* q_out, const qx_cuda_heads* k, const qx_cuda_heads* v,
                                    const int32_t* positions, float* mass, uint32_t* status, void* stream, char* err,
                                    uint64_t n) {
    const char* m = check_cache(cache);
    if (!m) m = check_drafts(drafts);
    if (m) return refuse(err, n, m);
    if (layer >= cache->layers) return refuse(err, n, "layer outside the cache");
    if (!rotary || !rotary->inv_freq) return refuse(err, n, "invalid rotary argument");
    const uint32_t D = cache->head_dim, rd = rotary->rotary_dim;
    if (rd < 2 || rd % 2 || rd > D || rd > 512) return refuse(err, n, "rotary_dim must be even, 2 to 512, and at most head_dim");
    if (!aligned(rotary->inv_freq, 8) || !aligned(positions, 4) || !aligned(status, 4))
        return refuse(err, n, "frequencies must be 8-byte, positions and status 4-byte aligned");
    if (!std::isfinite(rotary->amplitude)) return refuse(err, n, "the rotary amplitude must be finite");
    const bool has_q = q && q->data, has_k = k && k->data;
    if (has_q != (q_out && q_out->data) || has_k != (v && v->data)) return refuse(err, n, "q goes with q_out, k with v");
    if (!has_q && !has_k) return refuse(err, n, "nothing to rotate");
    if (mass && !has_k) return refuse(err, n, "mass goes with k and v");
    if (!aligned(mass, 4)) return refuse(err, n, "mass must be 4-byte aligned");
    if (has_q) {
        if (!q_heads || q_heads > kMaxHeads) return refuse(err, n, "1 to 1024 query heads");
        m = check_heads(q, drafts->seqs, drafts->max_nodes, q_heads, D, dtype, false);
        if (!m) m = check_heads(q_out, drafts->seqs, drafts->max_nodes, q_heads, D, dtype, true);
        if (!m && q->data == q_out->data && (q->seq_stride != q_out->seq_stride || q->node_stride != q_out->node_stride ||
                                             q->head_stride != q_out->head_stride))
            m = "q_out in place of q must have its strides";
        if (m) return refuse(err, n, m);
    }
    if (has_k) {
        m = check_heads(k, drafts->seqs, drafts->max_nodes, cache->kv_heads, D, dtype, false);
        if (!m) m = check_heads(v, drafts->seqs, drafts->max_nodes, cache->kv_heads, D, dtype, false);
        if (m) return refuse(err, n, m);
    }
    DeviceOf dev(cache->k, err, n);
    if (!dev.ok) return 0;
    auto heads = [](const qx_cuda_heads* t, bool has) {
        return has ? Heads{t->data, (size_t)t->seq_stride, (size_t)t->node_stride, (size_t)t->head_stride} : Heads{};
    };
    RopeArgs a{cache_of(cache), drafts_of(drafts), (int)layer, (int)q_heads, (int)rd, rotary->interleaved ? 1 : 0,
               rotary->inv_freq, rotary->amplitude, heads(q, has_q), heads(q_out, has_q), heads(k, has_k),
               heads(v, has_k), {Over(1), Over(1), 0}, {Over(1), Over(1), 0}, Over(1), positions, mass, status};
    // 16-byte accesses where pointers, strides and the rotated part allow; else
    // element by element (odd strides or parts, which a view of a larger
    // projection can have)
    const int eb = elem_bytes(dtype), V = 16 / eb;
    const bool wide = D % V == 0 && (rotary->interleaved ? rd % (2 * V) == 0 : rd % (2 * V) == 0) && (D - rd) % V == 0 &&
                      packs(has_q ? q : nullptr, V, eb) && packs(has_q ? q_out : nullptr, V, eb) &&
                      packs(has_k ? k : nullptr, V, eb) && packs(has_k ? v : nullptr, V, eb);
    cudaStream_t st = (cudaStream_t)stream;
    cudaError_t e;
    if (dtype == QX_CUDA_F32) e = wide ? launch_rope<float, 4>(a, st) : launch_rope<float, 1>(a, st);
    else if (dtype == QX_CUDA_F16) e = wide ? launch_rope<__half, 8>(a, st) : launch_rope<__half, 1>(a, st);
    else e = wide ? launch_rope<__nv_bfloat16, 8>(a, st) : launch_rope<__nv_bfloat16, 1>(a, st);
    return finish(e, err, n);
}
