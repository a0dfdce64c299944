// Attention of drafted tokens over the INT8 cache (qx_cuda_tree_attention):
// the entry point, the kernel for small trees, the joining of parts, and the
// weights each cache row got.  The mathematics and the cut of the work are in
// qx_tree.cuh, the kernel for larger trees in qx_tree_tc.cu.
#include <cmath>

#include "qx_tree.cuh"

namespace {

using namespace qx::ops;

constexpr int kTreeThreads = 128, kTreeWarps = 4;

__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {   // not volatile: products may be interleaved
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}


// ---- one warp's 16 cache rows --------------------------------------------------

// A warp's steps of 16 cache rows come through a ring of its own in shared
// memory, filled by asynchronous copies.  A step: the K codes [16][HD], the V
// codes, then ks[16], vs[16] and log2(vs), 1 / vs, which the warp adds when the
// step has arrived.  16-byte chunks are swizzled so that what eight lanes read at a time
// lies in different banks: K by the row's lowest bit, V by row / 4.
//
// Rows 4 j .. 4 j + 3 of a step belong to the lanes with lane % 4 = j, in both
// products: accumulator column 2 j + c of key tile h is row 4 j + 2 h + c.
template <int HD>
struct Step {
    static constexpr int kCodes = 16 * HD, kBytes = 2 * kCodes + 4 * 64, kChunks = HD / 16;
    __device__ static __forceinline__ int k_chunk(int row, int c) { return HD == 128 ? c ^ ((row & 1) << 2) : c; }
    __device__ static __forceinline__ int v_chunk(int row, int c) { return c ^ ((row >> 2) * 2 % kChunks); }
};
__device__ __forceinline__ void copy16(uint32_t to, const void* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t to, const void* from) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to), "l"(from) : "memory");
}
// Rows row0 .. of KV head g (k, v, ks, vs: the sequence's row 0); rows past the last repeat it.
template <int HD>
__device__ __forceinline__ void copy_step(const int8_t* k, const int8_t* v, const float* ks, const float* vs, int row_bytes,
                                          int row0, int last, uint32_t to) {
    constexpr int C = Step<HD>::kChunks;
    const int lane = threadIdx.x & 31, c = lane % C;
#pragma unroll
    for (int i = 0; i < 16 * C / 32; ++i) {
        const int r = i * (32 / C) + lane / C;
        const size_t at = (size_t)min(row0 + r, last) * row_bytes + 16 * c;
        copy16(to + r * HD + 16 * Step<HD>::k_chunk(r, c), k + at);
        copy16(to + Step<HD>::kCodes + r * HD + 16 * Step<HD>::v_chunk(r, c), v + at);
    }
    copy4(to + 2 * Step<HD>::kCodes + 4 * lane, (lane < 16 ? ks : vs) + min(row0 + (lane & 15), last));
}
// log2(vs) and 1 / vs beside the step's scales; whole warp.
template <int HD>
__device__ __forceinline__ void finish_step(uint8_t* step) {
    float* f = reinterpret_cast<float*>(step + 2 * Step<HD>::kCodes);
    const int lane = threadIdx.x & 31;
    const float v = f[16 + (lane & 15)];
    f[32 + lane] = lane < 16 ? log_vs(v) : inv_vs(v);
    __syncwarp();
}

// A block of 16 query rows as the products' A operand, in the order in which the
// lanes take it: 16 bytes a lane (rows n and n + 8 of dims d, d + 1, then of d + 2,
// d + 3; n = lane / 4, d = 64 c + 16 j + 4 i, j = lane % 4) for each c, i and F16 term.
template <int HD, int NT>
struct QBlock {
    static constexpr int kFrag = 512 + 32;                 // the gap keeps the staging's stores apart
    static constexpr int kTerm = HD / 16 * kFrag, kBytes = NT * kTerm;
};

// Stages rows 2 part, 2 part + 1 and those 8 further of the block at row0 of KV
// head g, `rows` rows in all; undo: the factors that undo their powers of two.
// Whole warp, four rows at a time for the latency of their loads.
template <class T, int HD, int NT>
__device__ __forceinline__ void stage_rows(const TreeArgs& a, int s, int g, int row0, int rows, int part, uint8_t* block,
                                           float (&undo)[4]) {
    constexpr int E = HD / 32;                             // dims of a lane
    const int lane = threadIdx.x & 31;
    Pack<T, E> x[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const int r = row0 + 2 * part + (u >> 1) + 8 * (u & 1);
        const T* q = (const T*)a.q.p + s * a.q.seq + (size_t)(r / a.group) * a.q.node +
                     (size_t)(g * a.group + r % a.group) * a.q.head + lane * E;
        if (r < rows && a.wide) {
            x[u] = *reinterpret_cast<const Pack<T, E>*>(q);
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) x[u].v[e] = r < rows ? q[e] : from_f32<T>(0.f);
        }
    }
    float big[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        big[u] = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float y = to_f32(x[u].v[e]);
            big[u] = fmaxf(big[u], isfinite(y) ? fabsf(y) : 0.f);
        }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1)
#pragma unroll
        for (int u = 0; u < 4; ++u) big[u] = fmaxf(big[u], __shfl_xor_sync(~0u, big[u], o));
    uint32_t w[NT][4][E / 2];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const RowScale rs(big[u]);
#pragma unroll
        for (int e = 0; e < E; e += 2) {
            const float y0 = to_f32(x[u].v[e]) * rs.f0 * rs.f1, y1 = to_f32(x[u].v[e + 1]) * rs.f0 * rs.f1;
            w[0][u][e / 2] = pack_half(y0, y1);
            if (NT == 2) w[NT - 1][u][e / 2] = rest_half(y0, y1, w[0][u][e / 2]);
        }
        undo[u] = rs.undo(a.scale);
    }
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int v = 0; v < 2; ++v) {
            uint8_t* to = block + t * QBlock<HD, NT>::kTerm + (2 * part + v) * 64;
            if (HD == 128)
                *reinterpret_cast<uint4*>(to + ((lane >> 4) * 4 + (lane & 3)) * QBlock<HD, NT>::kFrag + (lane >> 2 & 3) * 16) =
                    make_uint4(w[t][2 * v][0], w[t][2 * v + 1][0], w[t][2 * v][E / 2 - 1], w[t][2 * v + 1][E / 2 - 1]);
            else
                *reinterpret_cast<uint2*>(to + (lane >> 1 & 3) * QBlock<HD, NT>::kFrag + (lane >> 3) * 16 + (lane & 1) * 8) =
                    make_uint2(w[t][2 * v][0], w[t][2 * v + 1][0]);
        }
}

// Key codes as the B operand: 16 bytes of a lane are eight words.
__device__ __forceinline__ void key_halves(const uint4& k, uint32_t* b) {
    const uint32_t w[4] = {k.x, k.y, k.z, k.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t u = w[i] ^ 0x80808080u;
        b[2 * i] = low_pair(u);
        b[2 * i + 1] = high_pair(u);
    }
}
// acc[h] += q . k of a staged block and key tile h, dims 64 c to 64 c + 63 (b: their key_halves).
// The smaller term first: the tensor cores cut what they add to a sum off at its last bit, and what comes first meets small sums.
template <int HD, int NT>
__device__ __forceinline__ void dot_block(const uint8_t* block, int c, const uint32_t* b0, const uint32_t* b1, float (&acc)[2][4]) {
#pragma unroll
    for (int t = NT - 1; t >= 0; --t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint4 q = *reinterpret_cast<const uint4*>(block + t * QBlock<HD, NT>::kTerm + (4 * c + i) * QBlock<HD, NT>::kFrag +
                                                            16 * (threadIdx.x & 31));
            const uint32_t af[4] = {q.x, q.y, q.z, q.w};
            mma16816(acc[0], af, b0[2 * i], b0[2 * i + 1]);
            mma16816(acc[1], af, b1[2 * i], b1[2 * i + 1]);
        }
}

// ---- the kernel for small trees ------------------------------------------------

// For trees with few query rows to a KV head, where reading the cache is most
// of the work.  64 sequences of one token over 4096 rows (BF16, 4 KV heads of
// 128; 271 MB, 41 us at the memory's rate) take 68 us, F32 81 us; with 32 query rows 103
// us.  Bound by instructions and their latency: turning the codes to F16 costs as many as
// the products, and registers allow 12 warps an SM (8 with 32 rows).  One token over 32768 rows takes 26 us,
// over 513 rows 12 us, which is launching, finding one's tiles and joining parts.
//
// Blocks of 16 MT query rows; each of the 4 warps takes 16 of a tile's 64 cache
// rows, kRing - 1 tiles ahead, keeps its own m, sum and o, and the four are
// joined when the unit's part ends.
constexpr int kRing = 3;
template <int HD, int NT, int MT>
struct Small {
    static constexpr int kQ = MT * QBlock<HD, NT>::kBytes, kRingBytes = kTreeWarps * kRing * Step<HD>::kBytes;
    static constexpr int kO = kTreeWarps * MT * 16 * (HD + 4) * 4;           // the warps' o, over the ring
    static constexpr int kBytes = kQ + (kRingBytes > kO ? kRingBytes : kO);
};
template <class T, int HD, int NT, int MT>
__global__ void __launch_bounds__(kTreeThreads, MT == 1 ? 3 : 2) k_tree_small(const __grid_constant__ TreeArgs a) {
    constexpr int BM = 16 * MT, NV = HD / 8;
    extern __shared__ __align__(128) uint8_t dyn[];
    float (*wo)[BM][HD + 4] = reinterpret_cast<float (*)[BM][HD + 4]>(dyn + Small<HD, NT, MT>::kQ);
    __shared__ float qfac[BM];
    __shared__ float wm[kTreeWarps][BM], wl[kTreeWarps][BM];
    __shared__ PieceList list;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, j = lane & 3, n8 = lane >> 2;
    uint8_t* ring = dyn + Small<HD, NT, MT>::kQ + warp * kRing * Step<HD>::kBytes;
    const uint32_t ring_a = (uint32_t)__cvta_generic_to_shared(ring);
    const int row_bytes = a.c.kv_heads * HD;
    int batch = 0, at = 0;
    list_pieces(a, list, 0);
    while (at < list.count) {
        const Piece p = list.piece[at];
        const int last = p.len + p.n - 1, stop = p.tile1 * kTile;
        const int8_t *k0 = a.c.k + p.base_row * row_bytes + p.g * HD, *v0 = a.c.v + p.base_row * row_bytes + p.g * HD;
        const float *ks0 = a.c.ks + p.base_row, *vs0 = a.c.vs + p.base_row;
        int r0 = p.tile0 * kTile + 16 * warp, slot = 0;
        auto copy = [&](int row, int s) {
            if (row < stop) copy_step<HD>(k0, v0, ks0, vs0, row_bytes, row, last, ring_a + s * Step<HD>::kBytes);
            asm volatile("cp.async.commit_group;" ::: "memory");      // empty past the end: the groups stay countable
        };
#pragma unroll
        for (int i = 0; i < kRing - 1; ++i) copy(r0 + i * kTile, i);
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            float undo[4];
            stage_rows<T, HD, NT>(a, p.s, p.g, p.row0 + 16 * t, p.row0 + p.have, warp, dyn + t * QBlock<HD, NT>::kBytes, undo);
            if (lane < 4) qfac[16 * t + 2 * warp + (lane >> 1) + 8 * (lane & 1)] = lane == 0 ? undo[0] : lane == 1 ? undo[1] : lane == 2 ? undo[2] : undo[3];
        }
        __syncthreads();
        // row [t][u] of a lane is the block's row 16 t + 8 u + lane / 4
        // (top: what raises m; ref: what the exponents are relative to)
        float m[MT][2], l[MT][2], o[MT][NV][4], fac[MT][2], top[MT][2], ref[MT][2];
        const unsigned long long* mrow[MT][2];
        int node[MT][2];
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int r = 16 * t + n8 + 8 * u;
                m[t][u] = top[t][u] = -INFINITY, l[t][u] = ref[t][u] = 0.f;
                fac[t][u] = qfac[r];
                node[t][u] = r < p.have ? (p.row0 + r) / a.group : -1;
                mrow[t][u] = a.mask && r < p.have ? a.mask + ((size_t)p.s * a.d.max_nodes + node[t][u]) * a.words : nullptr;
            }
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int d = 0; d < NV; ++d) o[t][d][0] = o[t][d][1] = o[t][d][2] = o[t][d][3] = 0.f;
        for (; r0 < stop; r0 += kTile) {
            __syncwarp();                                              // the slot to fill has been read
            copy(r0 + (kRing - 1) * kTile, slot == 0 ? kRing - 1 : slot - 1);
            asm volatile("cp.async.wait_group %0;" ::"n"(kRing - 1) : "memory");
            __syncwarp();
            uint8_t* step = ring + slot * Step<HD>::kBytes;
            slot = slot == kRing - 1 ? 0 : slot + 1;
            finish_step<HD>(step);
            const float* f = reinterpret_cast<const float*>(step + 2 * Step<HD>::kCodes);
            float ks[4], lv[4], iv[4];
            *reinterpret_cast<float4*>(ks) = *reinterpret_cast<const float4*>(f + 4 * j);
            *reinterpret_cast<float4*>(lv) = *reinterpret_cast<const float4*>(f + 32 + 4 * j);
            *reinterpret_cast<float4*>(iv) = *reinterpret_cast<const float4*>(f + 48 + 4 * j);
            float acc[MT][2][4] = {};
#pragma unroll
            for (int c = 0; c < HD / 64; ++c) {
                uint32_t b[2][8];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int row = 4 * (n8 >> 1) + 2 * h + (n8 & 1);
                    key_halves(*reinterpret_cast<const uint4*>(step + row * HD + 16 * Step<HD>::k_chunk(row, 4 * c + j)), b[h]);
                }
#pragma unroll
                for (int t = 0; t < MT; ++t) dot_block<HD, NT>(dyn + t * QBlock<HD, NT>::kBytes, c, b[0], b[1], acc[t]);
            }
            // acc[t][h][2 u + c]: row [t][u], cache row r0 + 4 j + 2 h + c
#pragma unroll
            for (int t = 0; t < MT; ++t)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int u = e >> 1 & 1, i = (e >> 2) * 2 + (e & 1);
                    acc[t][e >> 2][e & 3] = fmaf(acc[t][e >> 2][e & 3] * fac[t][u], ks[i], lv[i]);
                }
            if (r0 + 16 > p.len) {
#pragma unroll
                for (int t = 0; t < MT; ++t)
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        uint32_t seen = 0;
                        if (node[t][u] >= 0) seen = (uint32_t)sees64(mrow[t][u], a.words, node[t][u], r0 + 4 * j, p.len, p.n);
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (!(seen >> i & 1u)) acc[t][i >> 1][2 * u + (i & 1)] = -INFINITY;
                    }
            }
            uint32_t w[MT][NT][4];
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                float mx[2];
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    mx[u] = fmaxf(fmaxf(acc[t][0][2 * u], acc[t][0][2 * u + 1]), fmaxf(acc[t][1][2 * u], acc[t][1][2 * u + 1]));
                    mx[u] = fmaxf(mx[u], __shfl_xor_sync(~0u, mx[u], 1));
                    mx[u] = fmaxf(mx[u], __shfl_xor_sync(~0u, mx[u], 2));
                }
                if (__any_sync(~0u, mx[0] > top[t][0] || mx[1] > top[t][1])) {
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        if (!(mx[u] > top[t][u])) mx[u] = m[t][u];
                        const float f = mx[u] > m[t][u] ? exp2_fast(m[t][u] - mx[u]) : 1.f;
                        l[t][u] *= f;
#pragma unroll
                        for (int d = 0; d < NV; ++d) o[t][d][2 * u] *= f, o[t][d][2 * u + 1] *= f;
                        m[t][u] = mx[u];
                        top[t][u] = mx[u] + kSlack;
                        ref[t][u] = mx[u] == -INFINITY ? 0.f : mx[u] - kPBias;
                    }
                }
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    float e[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        e[i] = exp2_fast(acc[t][i >> 1][2 * u + (i & 1)] - ref[t][u]);
                        l[t][u] = fmaf(e[i], iv[i], l[t][u]);
                    }
                    w[t][0][u] = pack_half(e[0], e[1]);
                    w[t][0][2 + u] = pack_half(e[2], e[3]);
                    if (NT == 2) {
                        w[t][NT - 1][u] = rest_half(e[0], e[1], w[t][0][u]);
                        w[t][NT - 1][2 + u] = rest_half(e[2], e[3], w[t][0][2 + u]);
                    }
                }
            }
            // values: dims (lane / 4) * NV + d of rows 4 j .. 4 j + 3 are column lane / 4 of value tile d
            uint32_t v[4][HD / 32];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int row = 4 * j + i;
                const uint8_t* at_v = step + Step<HD>::kCodes + row * HD;
                if (HD == 128) {
                    const uint4 w4 = *reinterpret_cast<const uint4*>(at_v + 16 * Step<HD>::v_chunk(row, n8));
                    v[i][0] = w4.x ^ 0x80808080u, v[i][1] = w4.y ^ 0x80808080u;
                    v[i][HD / 32 - 2] = w4.z ^ 0x80808080u, v[i][HD / 32 - 1] = w4.w ^ 0x80808080u;
                } else {
                    const uint2 w2 = *reinterpret_cast<const uint2*>(at_v + 16 * Step<HD>::v_chunk(row, n8 >> 1) + 8 * (n8 & 1));
                    v[i][0] = w2.x ^ 0x80808080u, v[i][1] = w2.y ^ 0x80808080u;
                }
            }
#pragma unroll
            for (int d4 = 0; d4 < HD / 32; ++d4) {
                const uint32_t a0 = __byte_perm(v[0][d4], v[1][d4], 0x5140), a1 = __byte_perm(v[0][d4], v[1][d4], 0x7362);
                const uint32_t c0 = __byte_perm(v[2][d4], v[3][d4], 0x5140), c1 = __byte_perm(v[2][d4], v[3][d4], 0x7362);
                const uint32_t b0[4] = {low_pair(a0), high_pair(a0), low_pair(a1), high_pair(a1)};
                const uint32_t b1[4] = {low_pair(c0), high_pair(c0), low_pair(c1), high_pair(c1)};
#pragma unroll
                for (int d = 0; d < 4; ++d)
#pragma unroll
                    for (int t = 0; t < MT; ++t)
#pragma unroll
                        for (int q = 0; q < NT; ++q) mma16816(o[t][4 * d4 + d], w[t][q], b0[d], b1[d]);
            }
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncthreads();                                               // every warp's steps are read: its o may go over them
        // join the four warps
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int r = 16 * t + n8 + 8 * u;
                l[t][u] += __shfl_xor_sync(~0u, l[t][u], 1);
                l[t][u] += __shfl_xor_sync(~0u, l[t][u], 2);
                if (j == 0) wm[warp][r] = m[t][u], wl[warp][r] = l[t][u];
                // columns 2 j, 2 j + 1 of value tile d are dims 2 j NV + d and (2 j + 1) NV + d
#pragma unroll
                for (int c = 0; c < 2; ++c)
#pragma unroll
                    for (int d = 0; d < NV; d += 4)
                        *reinterpret_cast<float4*>(&wo[warp][r][(2 * j + c) * NV + d]) = make_float4(
                            o[t][d][2 * u + c], o[t][d + 1][2 * u + c], o[t][d + 2][2 * u + c], o[t][d + 3][2 * u + c]);
            }
        __syncthreads();
        float* part = part_of(a, blockIdx.x, p.begins);
        for (int i = tid; i < BM * (HD / 8); i += kTreeThreads) {
            const int r = i / (HD / 8), d0 = i % (HD / 8) * 8;
            if (r >= p.have) continue;
            float mx = -INFINITY, sum = 0.f, y[8] = {};
            for (int w = 0; w < kTreeWarps; ++w) mx = fmaxf(mx, wm[w][r]);
            for (int w = 0; w < kTreeWarps; ++w) {
                const float f = part_weight(wm[w][r], wl[w][r], mx);
                sum = fmaf(f, wl[w][r], sum);
#pragma unroll
                for (int e = 0; e < 8; ++e) y[e] = fmaf(f, wo[w][r][d0 + e], y[e]);
            }
            if (p.whole) {
                const int nd = (p.row0 + r) / a.group, h = p.g * a.group + (p.row0 + r) % a.group;
                T* dst = (T*)a.out.p + p.s * a.out.seq + nd * a.out.node + h * a.out.head + d0;
#pragma unroll
                for (int e = 0; e < 8; ++e) dst[e] = from_f32<T>(sum == 0.f ? 0.f : y[e] / sum);
                if (d0 == 0) write_lse(a, p.s, nd, h, mx, sum);
            } else {
                float* dst = part + (size_t)r * (kPartHead + HD);
                *reinterpret_cast<float4*>(dst + kPartHead + d0) = make_float4(y[0], y[1], y[2], y[3]);
                *reinterpret_cast<float4*>(dst + kPartHead + d0 + 4) = make_float4(y[4], y[5], y[6], y[7]);
                if (d0 == 0) dst[0] = mx, dst[1] = sum;
            }
        }
        __syncthreads();
        if (++at == list.count && list.more) {
            __syncthreads();                             // everyone has read the counts
            list_pieces(a, list, ++batch);
            at = 0;
        }
    }
}

// Adds the parts of the units that several CTAs worked on, by the records they
// left.  A unit of few parts is joined by a warp a row, one of many by a CTA a
// row, whose warps take every eighth part: items of eight rows or one, counted
// from the records by every CTA for itself.  A row's first parts are asked for before
// their factors are known.  What it adds to a call: 9 us for 64 x 16 nodes over 4096 rows (147
// units of two or three parts, 20 MB), 7 us for 13 nodes over 32768 rows (4 units of 37 parts).  A CTA for each
// record and eight rows, most of them with nothing to do, added 10 and 15 us.
constexpr int kJoinThreads = 256, kJoinWarps = kJoinThreads / 32, kFewParts = 8, kJoinAhead = 4, kJoinList = 64;
struct JoinItem {
    Join j;
    int c, local;                                          // the record, and the item among its own
};
template <class T, int HD>
__global__ void __launch_bounds__(kJoinThreads, 4) k_tree_join(const __grid_constant__ TreeArgs a) {
    constexpr int kLanes = HD / 4, S = 32 / kLanes;        // lanes of a part's row, parts a warp reads at a time
    __shared__ int warp_sum[kJoinWarps];
    __shared__ JoinItem list[kJoinList];
    __shared__ float4 shares[kJoinWarps][kLanes];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, sub = lane / kLanes, d = lane % kLanes;
    asm volatile("griddepcontrol.wait;" ::: "memory");     // launched while the kernel before still runs
    const int per = (a.ctas + kJoinThreads - 1) / kJoinThreads, c0 = min(a.ctas, tid * per), c1 = min(a.ctas, c0 + per);
    auto items_of = [&](const Join& j) { return j.parts == 0 ? 0 : j.parts <= kFewParts ? (j.have + kJoinWarps - 1) / kJoinWarps : j.have; };
    Join one{};                                            // kept where a thread has one record
    int mine = 0;
    for (int c = c0; c < c1; ++c) {
        one = a.joins[c];
        mine += items_of(one);
    }
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int t = __shfl_up_sync(~0u, upto, o);
        if (lane >= o) upto += t;
    }
    if (lane == 31) warp_sum[warp] = upto;
    __syncthreads();
    int total = 0;
#pragma unroll
    for (int w = 0; w < kJoinWarps; ++w) {
        if (w < warp) upto += warp_sum[w];
        total += warp_sum[w];
    }
    const int row_floats = kPartHead + HD, step = 2 * a.block_rows * row_floats;   // all parts are below 2^24 floats
    const int each = (total + gridDim.x - 1) / gridDim.x, end = min(total, (int)(blockIdx.x + 1) * each);
    for (int i0 = blockIdx.x * each; i0 < end; i0 += kJoinList) {
        const int i1 = min(end, i0 + kJoinList);
        int b = upto - mine;
        if (b < i1 && upto > i0)
            for (int c = c0; c < c1; ++c) {
                const Join j = per == 1 ? one : a.joins[c];
                const int n = items_of(j);
                for (int i = max(b, i0); i < min(b + n, i1); ++i) list[i - i0] = {j, c, i - b};
                b += n;
            }
        __syncthreads();
        for (int item = 0; item < i1 - i0; ++item) {
            const Join& j = list[item].j;
            const int parts_n = j.parts, local = list[item].local;
            const bool few = parts_n <= kFewParts;
            const int row = few ? local * kJoinWarps + warp : local;
            if (row >= j.have) continue;                   // (never in part of a CTA that joins a row together)
            // the first part begins the unit, the others are what their CTAs began with
            const float* parts = part_of(a, list[item].c - 1, false) + row * row_floats;
            auto part = [&](int i) { return parts + max(i * step, step / 2); };
            float4 v[kJoinAhead], y = make_float4(0.f, 0.f, 0.f, 0.f);
            auto add = [&](float f, const float4& x) {
                y = make_float4(fmaf(f, x.x, y.x), fmaf(f, x.y, y.y), fmaf(f, x.z, y.z), fmaf(f, x.w, y.w));
            };
            float mx, sum;
            if (few) {
                // lanes i, i + 8, .. have part i's factor
#pragma unroll
                for (int u = 0; u < kJoinAhead; ++u)
                    if (u * S < parts_n) v[u] = *reinterpret_cast<const float4*>(part(min(u * S + sub, parts_n - 1)) + kPartHead + 4 * d);
                const int mine = lane & (kFewParts - 1);
                float2 ml = make_float2(-INFINITY, 0.f);
                if (mine < parts_n) ml = *reinterpret_cast<const float2*>(part(mine));
                mx = ml.x;
#pragma unroll
                for (int o = kFewParts / 2; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, o));
                const float f = part_weight(ml.x, ml.y, mx);
                sum = f * ml.y;
#pragma unroll
                for (int o = kFewParts / 2; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
#pragma unroll
                for (int u = 0; u < kFewParts / S; ++u)
                    if (u * S < parts_n) {
                        const float fu = __shfl_sync(~0u, f, u * S + sub);
                        if (u >= kJoinAhead) v[u % kJoinAhead] = *reinterpret_cast<const float4*>(part(min(u * S + sub, parts_n - 1)) + kPartHead + 4 * d);
                        if (u * S + sub < parts_n) add(fu, v[u % kJoinAhead]);
                    }
            } else {
                const int first = warp * S + sub, by = kJoinWarps * S;
#pragma unroll
                for (int u = 0; u < kJoinAhead; ++u)
                    if (first + u * by < parts_n) v[u] = *reinterpret_cast<const float4*>(part(first + u * by) + kPartHead + 4 * d);
                mx = -INFINITY, sum = 0.f;
                for (int i = lane; i < parts_n; i += 32) mx = fmaxf(mx, part(i)[0]);
#pragma unroll
                for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, o));
                for (int i = lane; i < parts_n; i += 32) {
                    const float2 ml = *reinterpret_cast<const float2*>(part(i));
                    sum = fmaf(part_weight(ml.x, ml.y, mx), ml.y, sum);
                }
#pragma unroll
                for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
                for (int i = first; i < parts_n; i += kJoinAhead * by) {
                    if (i != first)
#pragma unroll
                        for (int u = 0; u < kJoinAhead; ++u)
                            if (i + u * by < parts_n) v[u] = *reinterpret_cast<const float4*>(part(i + u * by) + kPartHead + 4 * d);
#pragma unroll
                    for (int u = 0; u < kJoinAhead; ++u)
                        if (i + u * by < parts_n) {
                            const float2 ml = *reinterpret_cast<const float2*>(part(i + u * by));
                            add(part_weight(ml.x, ml.y, mx), v[u]);
                        }
                }
            }
            if (S == 2) {
                __syncwarp();
                y.x += __shfl_xor_sync(~0u, y.x, 16), y.y += __shfl_xor_sync(~0u, y.y, 16);
                y.z += __shfl_xor_sync(~0u, y.z, 16), y.w += __shfl_xor_sync(~0u, y.w, 16);
            }
            if (!few) {
                if (sub == 0) shares[warp][d] = y;
                __syncthreads();
                if (warp == 0) {
#pragma unroll
                    for (int w = 1; w < kJoinWarps; ++w) {
                        const float4 z = shares[w][d];
                        y = make_float4(y.x + z.x, y.y + z.y, y.z + z.z, y.w + z.w);
                    }
                }
                __syncthreads();                               // the next item's shares may go over these
                if (warp) continue;
            }
            if (sub) continue;
            const float scale = sum == 0.f ? 0.f : 1.f / sum;
            const int nd = (int)a.per_group(j.row0 + row), h = j.g * a.group + (j.row0 + row) - nd * a.group;
            T* dst = (T*)a.out.p + j.s * a.out.seq + nd * a.out.node + h * a.out.head + 4 * d;
            const float out[4] = {y.x * scale, y.y * scale, y.z * scale, y.w * scale};
            Pack<T, 4> z;
#pragma unroll
            for (int e = 0; e < 4; ++e) z.v[e] = from_f32<T>(sum == 0.f ? 0.f : out[e]);
            if (a.wide) {
                *reinterpret_cast<Pack<T, 4>*>(dst) = z;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) dst[e] = z.v[e];
            }
            if (d == 0) write_lse(a, j.s, nd, h, mx, sum);
        }
        __syncthreads();                                   // the list has been read
    }
}

// ---- what each cache row got ---------------------------------------------------

// mass[t] += sum over the sequence's query rows of 2^(x_t - lse), x_t without
// vs_t.  The steps of 16 cache rows of all sequences, laid end to end, are
// shared out evenly over the CTAs.  A CTA holds its sequence's queries in
// shared memory as F16 operands (in several passes where they are too many),
// and a warp goes through them with a step's keys in registers: it alone adds
// to the step's rows, in one order, without atomics.
//
// For 64 ragged sequences of one token over up to 4096 rows it is 25 us of the
// call's 61, bound by instructions and by steps that come out uneven (25 for 16 warps); for 64 trees of 16 nodes (512
// query rows) over 4096 rows 183 of 333, bound by mma.sync, whose pipe 16 products of 16 x 8 x 16 a block keep busy
// (staging the queries anew for every tile and block took 1150 us).
constexpr int kMassWarps = 16, kMassThreads = kMassWarps * 32;
template <int HD, int NT>
struct Held {                                              // a QBlock, and its rows' factors and lse
    static constexpr int kFacs = QBlock<HD, NT>::kBytes, kBytes = kFacs + 16 * 8, kMost = 200 * 1024 / kBytes;
};
template <int HD>
struct StepKeys {
    uint4 k[2][HD / 64];                                   // key tile h: row 4 (n / 2) + 2 h + n % 2 of the step, n = lane / 4
    float ks[4];                                           // rows 4 j .. 4 j + 3, j = lane % 4
    __device__ __forceinline__ void load(const int8_t* k0, const float* ks0, int row_bytes, int r0, int last) {
        const int lane = threadIdx.x & 31, j = lane & 3, n = lane >> 2;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int c = 0; c < HD / 64; ++c)
                k[h][c] = *reinterpret_cast<const uint4*>(k0 + (size_t)min(r0 + 4 * (n >> 1) + 2 * h + (n & 1), last) * row_bytes +
                                                          64 * c + 16 * j);
#pragma unroll
        for (int i = 0; i < 4; ++i) ks[i] = ks0[min(r0 + 4 * j + i, last)];
    }
};
// ONE: a KV head's query rows are one block at most.  Its keys are needed once, and those of three steps are on their
// way (64 ragged sequences of one token: 63 us for the call with one, 61 with three).
template <class T, int HD, int NT, bool ONE>
__global__ void __launch_bounds__(kMassThreads, 1) k_tree_mass(const __grid_constant__ TreeArgs a) {
    using Block = Held<HD, NT>;
    constexpr int kAhead = ONE ? 3 : 1;
    extern __shared__ __align__(128) uint8_t dyn[];
    __shared__ int warp_sum[kScanThreads / 32], at_seq, at_first, clash;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, j = lane & 3, n8 = lane >> 2;
    const int per = (a.d.seqs + kScanThreads - 1) / kScanThreads;
    const int s0 = tid < kScanThreads ? min(a.d.seqs, tid * per) : 0, s1 = tid < kScanThreads ? min(a.d.seqs, s0 + per) : 0;
    auto steps_of = [&](int s) {
        const int len = a.d.lens[s], n = a.d.count(s);
        return n && fits(a.c, a.d, a.d.slots[s], len, n) ? (len + n + 15) / 16 : 0;
    };
    int mine = 0;
    for (int s = s0; s < s1; ++s) mine += steps_of(s);
    int inc = mine;
    if (tid < kScanThreads) {
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int t = __shfl_up_sync(~0u, inc, o);
            if (lane >= o) inc += t;
        }
        if (lane == 31) warp_sum[warp] = inc;
    }
    __syncthreads();
    int first = inc - mine, total = 0;
    for (int i = 0; i < kScanThreads / 32; ++i) {
        if (i < warp) first += warp_sum[i];
        total += warp_sum[i];
    }
    const int each = total / gridDim.x, extra = total % gridDim.x, cta = blockIdx.x;
    int at = each * cta + min(cta, extra);
    const int end = at + each + (cta < extra ? 1 : 0), row_bytes = a.c.kv_heads * HD;
    while (at < end) {
        __syncthreads();
        if (tid == 0) clash = 0;
        int f = first;
        for (int s = s0; s < s1; ++s) {
            const int t = steps_of(s);
            if (at >= f && at < f + t) at_seq = s, at_first = f;
            f += t;
        }
        __syncthreads();
        const int s = at_seq, slot = a.d.slots[s], len = a.d.lens[s], n = a.d.count(s), last = len + n - 1;
        const int step0 = at - at_first, step1 = min((last + 16) / 16, end - at_first);
        for (int i = tid; i < a.d.seqs; i += kMassThreads)
            if (i != s && a.d.slots[i] == slot && steps_of(i)) clash = 1;
        at += step1 - step0;
        const size_t base_row = (size_t)slot * a.c.slot_rows + (size_t)a.layer * a.c.layer_rows;
        const int8_t* k0 = a.c.k + base_row * row_bytes;
        const float* ks0 = a.c.ks + base_row;
        const int rows = n * a.group, per_head = (rows + 15) / 16, blocks = per_head * a.c.kv_heads;
        for (int b0 = 0; b0 < blocks; b0 += Block::kMost) {
            const int b1 = min(blocks, b0 + Block::kMost);
            const int g0 = b0 / per_head, g1 = (b1 - 1) / per_head;
            StepKeys<HD> next[kAhead];
            int next_st = step0 + warp, next_g = g0;
            auto fetch = [&](StepKeys<HD>& k) {            // the warp's next step and head
                if (next_st >= step1) return;
                k.load(k0 + next_g * HD, ks0, row_bytes, next_st * 16, last);
                if (++next_g > g1) next_g = g0, next_st += kMassWarps;
            };
#pragma unroll
            for (int i = 0; i < kAhead; ++i) fetch(next[i]);
            __syncthreads();                               // the blocks before have been used
            if (clash) break;
            for (int i = warp; i < 4 * (b1 - b0); i += kMassWarps) {
                const int b = b0 + i / 4, part = i % 4, g = b / per_head, row0 = b % per_head * 16;
                uint8_t* block = dyn + (size_t)(b - b0) * Block::kBytes;
                const int row = 2 * part + (lane >> 1 & 1) + 8 * (lane & 1), r = row0 + row;
                const float lg = lane < 4 && r < rows ? a.lse2[((size_t)s * a.d.max_nodes + r / a.group) * a.q_heads + g * a.group + r % a.group] : 0.f;
                float undo[4];
                stage_rows<T, HD, NT>(a, s, g, row0, rows, part, block, undo);
                if (lane < 4)
                    reinterpret_cast<float2*>(block + Block::kFacs)[row] =
                        make_float2(lane == 0 ? undo[0] : lane == 1 ? undo[1] : lane == 2 ? undo[2] : undo[3], lg);
            }
            __syncthreads();
            float got[4] = {};
            // the weights of the block's rows for rows r0 + 4 j .. + 3 of the cache, from their products
            auto weigh = [&](const float (&part)[HD / 64][2][4], const float (&ks)[4], const uint8_t* block, int row0, int r0) {
                const float2* facs = reinterpret_cast<const float2*>(block + Block::kFacs);
                const bool edge = r0 + 16 > len;
                float e[2][4];
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const float2 fl = facs[n8 + 8 * u];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float x = part[0][i >> 1][2 * u + (i & 1)];
                        if (HD == 128) x += part[HD / 64 - 1][i >> 1][2 * u + (i & 1)];
                        e[u][i] = exp2_fast(fmaf(x * fl.x, ks[i], -fl.y));
                    }
                }
                if (edge || row0 + 16 > rows) {
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const int r = row0 + n8 + 8 * u, node = (int)a.per_group(r);
                        uint32_t seen = r < rows ? 15u : 0u;
                        if (edge && r < rows)
                            seen = (uint32_t)sees64(a.mask ? a.mask + ((size_t)s * a.d.max_nodes + node) * a.words : nullptr,
                                                    a.words, node, r0 + 4 * j, len, n);
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (!(seen >> i & 1u)) e[u][i] = 0.f;
                    }
                    __syncwarp();                          // the next products are the whole warp's
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) got[i] += e[0][i] + e[1][i];
            };
            auto put = [&](int r0) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    got[i] += __shfl_xor_sync(~0u, got[i], 4);
                    got[i] += __shfl_xor_sync(~0u, got[i], 8);
                    got[i] += __shfl_xor_sync(~0u, got[i], 16);
                }
                const float x = n8 == 0 ? got[0] : n8 == 1 ? got[1] : n8 == 2 ? got[2] : got[3];
                const int t = r0 + 4 * j + n8;
                if (n8 < 4 && t <= last) a.mass[base_row + t] += x;
#pragma unroll
                for (int i = 0; i < 4; ++i) got[i] = 0.f;
            };
            int st = step0 + warp, g = g0;
            while (ONE && st < step1)
#pragma unroll
                for (int i = 0; i < kAhead; ++i) {
                    if (st >= step1) break;
                    const uint8_t* block = dyn + (size_t)(g - g0) * Block::kBytes;
                    const float ks[4] = {next[i].ks[0], next[i].ks[1], next[i].ks[2], next[i].ks[3]};
                    float part[HD / 64][2][4] = {};                  // apart, for shorter chains of products
#pragma unroll
                    for (int c = 0; c < HD / 64; ++c) {
                        uint32_t key[2][8];
                        key_halves(next[i].k[0][c], key[0]);
                        key_halves(next[i].k[1][c], key[1]);
                        dot_block<HD, NT>(block, c, key[0], key[1], part[c]);
                    }
                    fetch(next[i]);
                    weigh(part, ks, block, 0, st * 16);
                    if (++g > g1) {
                        put(st * 16);
                        st += kMassWarps;
                        g = g0;
                    }
                }
            for (; !ONE && st < step1; st += kMassWarps) {
                for (g = g0; g <= g1; ++g) {
                    const float ks[4] = {next[0].ks[0], next[0].ks[1], next[0].ks[2], next[0].ks[3]};
                    uint32_t key[2][HD / 8];
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int c = 0; c < HD / 64; ++c) key_halves(next[0].k[h][c], key[h] + 8 * c);
                    fetch(next[0]);
                    const int first_b = max(b0, g * per_head), end_b = min(b1, (g + 1) * per_head);
                    for (int b = first_b; b < end_b; ++b) {
                        const uint8_t* block = dyn + (size_t)(b - b0) * Block::kBytes;
                        float part[HD / 64][2][4] = {};
#pragma unroll
                        for (int c = 0; c < HD / 64; ++c) dot_block<HD, NT>(block, c, key[0] + 8 * c, key[1] + 8 * c, part[c]);
                        weigh(part, ks, block, (b - g * per_head) * 16, st * 16);
                    }
                }
                put(st * 16);
            }
        }
        if (clash && tid == 0 && a.status) atomicOr(a.status, QX_CUDA_STATUS_SHARED);
    }
}

// ---- host side -----------------------------------------------------------------

struct Plan {
    bool tc;                         // blocks of 128 rows on tcgen05
    int block_rows, row_blocks;
    uint64_t parts, joins, lse2;     // bytes of workspace
    uint64_t all() const { return (parts + joins + lse2 + 255) / 256 * 256; }
};
// the most CTAs that a call with blocks of so many rows has: they set what the workspace holds
constexpr int most_ctas(int block_rows) { return block_rows == 128 ? kMaxCtas / 8 : block_rows == 32 ? kMaxCtas / 4 : kMaxCtas; }
Plan plan_of(uint32_t seqs, uint32_t max_nodes, uint32_t q_heads, uint32_t kv_heads, uint32_t head_dim) {
    Plan p{};
    const uint64_t rows = (uint64_t)max_nodes * (q_heads / kv_heads);
    p.tc = rows > 32;
    // 64 sequences of 4096 rows, BF16, 4 KV heads of 128: 16 query rows to a KV head take 71 us in blocks of 16; 32 rows
    // 103 us in blocks of 32, 147 us in two of 16; 64 rows 136 us on tcgen05, whose time depends little on how many of
    // its 128 rows there are (128: 151 us).
    p.block_rows = p.tc ? 128 : rows > 16 ? 32 : 16;
    p.row_blocks = (int)((rows + p.block_rows - 1) / p.block_rows);
    p.parts = (uint64_t)2 * most_ctas(p.block_rows) * p.block_rows * (kPartHead + head_dim) * 4;
    p.joins = (uint64_t)(kMaxCtas * sizeof(Join) + 255) / 256 * 256;
    p.lse2 = (uint64_t)seqs * max_nodes * q_heads * 4;
    return p;
}

const char* check_shape(uint32_t q_heads, uint32_t kv_heads, uint32_t head_dim, uint32_t dtype) {
    if (head_dim != 64 && head_dim != 128) return "tree attention needs head_dim 64 or 128";
    if (!kv_heads || kv_heads > kMaxHeads || !q_heads || q_heads > kMaxHeads || q_heads % kv_heads)
        return "q_heads must be a multiple of kv_heads, at most 1024";
    if (dtype > QX_CUDA_BF16) return "unsupported element type";
    return nullptr;
}

template <class T, int HD, int NT, int MT>
cudaError_t launch_small(TreeArgs& a, int sms, cudaStream_t st) {
    int per = 0;
    constexpr int kBytes = Small<HD, NT, MT>::kBytes;
    const auto kernel = k_tree_small<T, HD, NT, MT>;
    cudaError_t e = cudaFuncSetAttribute((const void*)kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes);
    if (e == cudaSuccess) e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, kernel, kTreeThreads, kBytes);
    if (e != cudaSuccess) return e;
    a.ctas = sms * (per < 1 ? 1 : per);
    if (a.ctas > most_ctas(16 * MT)) a.ctas = most_ctas(16 * MT);
    a.per_cta = Over((uint32_t)a.ctas);
    kernel<<<a.ctas, kTreeThreads, kBytes, st>>>(a);
    return cudaGetLastError();
}
template <class T, int HD, int NT>
cudaError_t run_typed(TreeArgs& a, bool tc, uint32_t type, int sms, cudaStream_t st) {
    cudaError_t e = tc                   ? launch_tree_tc(a, type, sms, st)
                    : a.block_rows == 16 ? launch_small<T, HD, NT, 1>(a, sms, st)
                                         : launch_small<T, HD, NT, 2>(a, sms, st);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)sms * 4);
    cfg.blockDim = dim3(kJoinThreads);
    cfg.stream = st;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, k_tree_join<T, HD>, a);
    if (e != cudaSuccess || !a.mass) return e;
    constexpr int kHeld = Held<HD, NT>::kMost * Held<HD, NT>::kBytes;
    const auto kernel = a.block_rows == 16 ? k_tree_mass<T, HD, NT, true> : k_tree_mass<T, HD, NT, false>;
    e = cudaFuncSetAttribute((const void*)kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kHeld);
    if (e != cudaSuccess) return e;
    kernel<<<sms, kMassThreads, kHeld, st>>>(a);
    return cudaGetLastError();
}

template <class T, int NT>
cudaError_t run_tree(TreeArgs& a, bool tc, uint32_t type, int sms, cudaStream_t st) {
    return a.c.head_dim == 128 ? run_typed<T, 128, NT>(a, tc, type, sms, st) : run_typed<T, 64, NT>(a, tc, type, sms, st);
}

}  // namespace

QX_API int qx_cuda_tree_attention_workspace(uint32_t seqs, uint32_t max_nodes, uint32_t q_heads, uint32_t kv_heads,
                                            uint32_t head_dim, uint32_t dtype, uint64_t* bytes, char* err, uint64_t n) {
    if (!bytes) return refuse(err, n, "invalid workspace argument");
    if (!seqs || seqs > kMaxSeqs || !max_nodes || max_nodes > kMaxNodes)
        return refuse(err, n, "at least one and at most 4096 sequences and nodes");
    if (const char* m = check_shape(q_heads, kv_heads, head_dim, dtype)) return refuse(err, n, m);
    const Plan p = plan_of(seqs, max_nodes, q_heads, kv_heads, head_dim);
    *bytes = p.all();
    return 1;
}

QX_API int qx_cuda_tree_attention(const qx_cuda_kv_cache* cache, uint32_t layer, const qx_cuda_drafts* drafts,
                                  uint32_t dtype, uint32_t q_heads, const qx_cuda_heads* q, const qx_cuda_heads* out,
                                  const uint64_t* mask, float scale, float* lse, float* mass, void* workspace,
                                  uint64_t workspace_bytes, uint32_t* status, void* stream, char* err, uint64_t n) {
    const char* m = check_cache(cache);
    if (!m) m = check_drafts(drafts);
    if (!m) m = check_shape(q_heads, cache->kv_heads, cache->head_dim, dtype);
    if (!m) m = check_heads(q, drafts->seqs, drafts->max_nodes, q_heads, cache->head_dim, dtype, false);
    if (!m) m = check_heads(out, drafts->seqs, drafts->max_nodes, q_heads, cache->head_dim, dtype, true);
    if (m) return refuse(err, n, m);
    if (layer >= cache->layers) return refuse(err, n, "layer outside the cache");
    if (!std::isfinite(scale)) return refuse(err, n, "the score scale must be finite");
    if (!aligned(mask, 8)) return refuse(err, n, "the mask must be 8-byte aligned");
    if (!aligned(lse, 4) || !aligned(mass, 4) || !aligned(status, 4))
        return refuse(err, n, "lse, mass and status must be 4-byte aligned");
    const Plan p = plan_of(drafts->seqs, drafts->max_nodes, q_heads, cache->kv_heads, cache->head_dim);
    if (!workspace || !aligned(workspace, 16) || workspace_bytes < p.all())
        return refuse(err, n, "the workspace is missing, misaligned or too small");
    const uint64_t tiles = ((uint64_t)cache->ctx_tokens + kTile - 1) / kTile;
    // (what each row got is summed in steps of 16 rows)
    if ((uint64_t)drafts->seqs * cache->kv_heads * p.row_blocks * tiles > 0x7fffffffull ||
        (mass && drafts->seqs * tiles * (kTile / 16) > 0x7fffffffull))
        return refuse(err, n, "more rows and cache than one call can take");
    if (cache_rows(cache_of(cache)) > 0x7fffffffull - kTile) return refuse(err, n, "the cache has more rows than the operator supports");
    if (q->data == out->data) {
        // each block of rows is read by the CTA that writes it, or by all before the join; the mass reads q after that
        if (mass) return refuse(err, n, "out may not be q itself where mass is collected");
        if ((drafts->seqs > 1 && q->seq_stride != out->seq_stride) || (drafts->max_nodes > 1 && q->node_stride != out->node_stride) ||
            (q_heads > 1 && q->head_stride != out->head_stride))
            return refuse(err, n, "out in place of q must have its strides");
    }
    DeviceOf dev(cache->k, err, n);
    if (!dev.ok) return 0;
    TreeArgs a{};
    a.c = cache_of(cache);
    a.d = drafts_of(drafts);
    a.layer = (int)layer;
    a.q_heads = (int)q_heads;
    a.group = (int)(q_heads / cache->kv_heads);
    a.block_rows = p.block_rows;
    a.row_blocks = p.row_blocks;
    a.per_block = Over((uint32_t)p.block_rows);
    a.per_heads = Over(cache->kv_heads);
    a.per_group = Over((uint32_t)a.group);
    a.q = {q->data, (size_t)q->seq_stride, (size_t)q->node_stride, (size_t)q->head_stride};
    a.out = {out->data, (size_t)out->seq_stride, (size_t)out->node_stride, (size_t)out->head_stride};
    a.mask = (const unsigned long long*)mask;
    a.words = (int)((drafts->max_nodes + 63) / 64);
    a.scale = scale;
    a.lse = lse;
    a.mass = mass;
    a.parts = (float*)workspace;
    a.joins = (Join*)((uint8_t*)workspace + p.parts);
    a.lse2 = mass ? (float*)((uint8_t*)workspace + p.parts + p.joins) : nullptr;
    a.status = status;
    const uint64_t step = 16 / elem_bytes(dtype);
    a.wide = aligned(q->data, 16) && aligned(out->data, 16) && q->seq_stride % step == 0 && q->node_stride % step == 0 &&
             q->head_stride % step == 0 && out->seq_stride % step == 0 && out->node_stride % step == 0 &&
             out->head_stride % step == 0;
    int id = 0, sms = 0;
    cudaError_t e = cudaGetDevice(&id);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, id);
    if (e != cudaSuccess) return finish(e, err, n);
    cudaStream_t st = (cudaStream_t)stream;
    if (dtype == QX_CUDA_F32) e = run_tree<float, 2>(a, p.tc, dtype, sms, st);
    else if (dtype == QX_CUDA_F16) e = run_tree<__half, 1>(a, p.tc, dtype, sms, st);
    else e = run_tree<__nv_bfloat16, 1>(a, p.tc, dtype, sms, st);
    return finish(e, err, n);
}
