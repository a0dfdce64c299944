// Tree attention on the tcgen05 tensor cores (qx_tree.cuh has the mathematics
// and the cut of the work): blocks of 128 query rows against tiles of 64 cache
// rows, one persistent CTA per SM.
//
// Roles, by warp:
//   0-3, 4-7   two softmax groups, which take the tiles in turn; a thread has
//              one query row (TMEM lane), and each group its own reference,
//              sum and output accumulator
//   8          issues S = Q K^T (128 x 64), up to four tiles ahead
//   9          makes the per-row constants of the scores
//   10         asks for the codes, by TMA some tiles ahead
//   11         issues O += P V, P read from TMEM, where it overwrites the S it
//              came from
//   12-15      turn the INT8 codes into F16 operands, and bring the next piece's
//              query block (the first one everybody)
//
// 64 sequences with trees of 16 nodes over 4096 rows (BF16, 4 KV heads of 128:
// 128 query rows to a KV head, 16640 tiles, 69 GFLOP and 288 MB, 44 us at the memory's rate) take 151
// us, F32 173 us; one sequence with 13 nodes over 32768 rows (F32) takes 45.  That is
// 0.9 us a tile and SM, with no unit above half of what it can do (issue slots 45 %, shared memory 45 %,
// tensor cores 23 %): a tile's chain of product, softmax and product is what takes the time, so two
// groups of softmax warps take turns, S runs four tiles ahead, and codes come two or three tiles
// ahead.  A call with one tile a CTA costs about 20 us: instruction fetch,
// queries, and the length of that chain.
//
// F16 operands are in the no-swizzle core-matrix layout: 8 rows x 16 bytes
// each, [row / 8][dim / 8][row % 8].  That one layout is K-major for K (rows =
// N, dims = K) and for Q, and MN-major for V (dims = N, rows = K), so nothing is
// transposed.  The codes arrive in TMA's 128-byte (64 dims: 64-byte) swizzle,
// from which eight rows of one 16-byte chunk, what a quarter-warp reads and
// writes at a time, lie in different banks.
#include <cuda.h>

#include <cmath>

#include "qx_tree.cuh"

namespace qx {
namespace ops {
namespace {

constexpr int kRows = 128, kGroup = 128, kTeam = 128, kTcThreads = 512;
constexpr int kKs = 2, kVs = 4;            // operand tiles: K goes once S is computed, V stays through the softmax
constexpr int kScores = 4;                 // S buffers
// Row factors and "queries are there" of so many pieces: the queries of piece
// P + 8 are brought once S of all of P + 6 is computed, a tile that is at least 6
// past P's first; S runs less than 4 tiles ahead of O, so by then both groups
// have had their first tiles of P.
constexpr int kFacs = 8;

template <int HD, int NT>
struct Shape {
    static constexpr int kTileBytes = kTile * HD * 2;          // K or V of a tile
    static constexpr int kQBytes = kRows * HD * 2;             // one term of Q
    static constexpr int kQs = NT == 1 ? 2 : 1;                // query blocks
    static constexpr int kRawBytes = kTile * HD;               // codes of K or V of a tile
    static constexpr int kAhead = NT == 1 ? 3 : 2;             // tiles of codes on their way
    static constexpr int kQAt = kAhead * 2 * kRawBytes, kKvAt = kQAt + kQs * NT * kQBytes;
    static constexpr int kSmem = kKvAt + (kKs + kVs) * kTileBytes + 1024;
    static constexpr int kO = kScores * kTile;                 // TMEM column of group 0's output
    static constexpr int kTmem = 512;                          // 256 + 2 HD, to a power of two
};

struct Bars {
    unsigned long long raw[4], raw_free[4], k_full[kKs], k_free[kKs], v_full[kVs], v_free[kVs], c_full[kVs], s_ready[kScores], p_ready[kScores], o_done[2], q_full[kFacs], q_free[2],
        both, o_free;
};
struct alignas(16) Columns {
    float ks[kTile], lv[kTile], iv[kTile];
};

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void bar_init(unsigned long long* b, unsigned count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_addr(b)), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_arrive(unsigned long long* b) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(b)) : "memory");
}
// One arrival for the warp, after what its lanes did (32 arrivals on one word
// take their turns in shared memory).
__device__ __forceinline__ void warp_arrive(unsigned long long* b) {
    __syncwarp();
    if ((threadIdx.x & 31) == 0) bar_arrive(b);
}
__device__ __forceinline__ bool bar_try(unsigned long long* b, unsigned parity) {
    uint32_t done;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
        : "=r"(done)
        : "r"(smem_addr(b)), "r"(parity)
        : "memory");
    return done != 0;
}
__device__ __forceinline__ bool elected() {
    uint32_t is;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(is));
    return is != 0;
}
// Bounded wait for a phase (2 s; a healthy one takes microseconds).  Gives up
// soon after another role has, unless it is for work of its own in flight.
__device__ __noinline__ bool bar_wait_slow(unsigned long long* b, unsigned parity, volatile int* gave_up, bool own) {
    unsigned long long t0 = 0;
    for (unsigned i = 1;; ++i) {
        if (bar_try(b, parity)) return true;
        if ((i & 255u) == 0u) {
            unsigned long long t;
            asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
            if (!t0) t0 = t;
            if ((*gave_up && !own) || t - t0 > 2000000000ull) {
                *gave_up = 1;
                return false;
            }
        }
    }
}
__device__ __forceinline__ bool bar_wait(unsigned long long* b, unsigned parity, volatile int* gave_up, bool own = false) {
    return bar_try(b, parity) || bar_wait_slow(b, parity, gave_up, own);
}

__device__ __forceinline__ uint64_t umma_desc(uint32_t addr, uint32_t lbo, uint32_t sbo) {
    return (uint64_t)((addr >> 4) & 0x3fffu) | ((uint64_t)((lbo >> 4) & 0x3fffu) << 16) |
           ((uint64_t)((sbo >> 4) & 0x3fffu) << 32) | (1ull << 46);
}
// kind::f16: D F32 (bits 4-5 = 1), A and B F16, B MN-major at bit 16, N >> 3 at 17-22, M >> 4 at 24-28.
__host__ __device__ constexpr uint32_t idesc_f16(int m, int n, bool b_mn) {
    return (1u << 4) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void mma_commit(unsigned long long* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar)) : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

#define QX_R8(r, i) "=r"(r[i]), "=r"(r[i + 1]), "=r"(r[i + 2]), "=r"(r[i + 3]), "=r"(r[i + 4]), "=r"(r[i + 5]), "=r"(r[i + 6]), "=r"(r[i + 7])
#define QX_I8(r, i) "r"(r[i]), "r"(r[i + 1]), "r"(r[i + 2]), "r"(r[i + 3]), "r"(r[i + 4]), "r"(r[i + 5]), "r"(r[i + 6]), "r"(r[i + 7])
// 32 (16) consecutive 32-bit TMEM columns of this thread's lane.
__device__ __forceinline__ void tmem_ld32(uint32_t t, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,"
        "%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : QX_R8(r, 0), QX_R8(r, 8), QX_R8(r, 16), QX_R8(r, 24)
        : "r"(t)
        : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t t, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : QX_R8(r, 0), QX_R8(r, 8)
        : "r"(t)
        : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t t, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::QX_I8(r, 0),
        QX_I8(r, 8), "r"(t)
        : "memory");
}

// After the wait for a load: what reads the registers stays behind it.
template <int N>
__device__ __forceinline__ void loaded(float2 (&x)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+f"(x[i].x), "+f"(x[i].y));
}

// Two F32 operations an instruction.
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 r;
    asm("mul.rn.f32x2 %0, %1, %2;"
        : "=l"(reinterpret_cast<unsigned long long&>(r))
        : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)));
    return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 r;
    asm("add.rn.f32x2 %0, %1, %2;"
        : "=l"(reinterpret_cast<unsigned long long&>(r))
        : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)));
    return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;"
        : "=l"(reinterpret_cast<unsigned long long&>(r))
        : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)),
          "l"(reinterpret_cast<unsigned long long&>(c)));
    return r;
}

// ---- bringing the cache --------------------------------------------------------

// 16 codes as F16: two 16-byte units of an operand tile.
__device__ __forceinline__ void widen(const uint4& w, uint8_t* to) {
    const uint32_t c[4] = {w.x ^ 0x80808080u, w.y ^ 0x80808080u, w.z ^ 0x80808080u, w.w ^ 0x80808080u};
    *reinterpret_cast<uint4*>(to) = make_uint4(low_pair(c[0]), high_pair(c[0]), low_pair(c[1]), high_pair(c[1]));
    *reinterpret_cast<uint4*>(to + 128) = make_uint4(low_pair(c[2]), high_pair(c[2]), low_pair(c[3]), high_pair(c[3]));
}
// A tile's codes of K or V to F16, by four warps: a warp takes eight rows of
// four 16-byte chunks at a time, all its reads before its writes.
template <int HD>
__device__ __forceinline__ void widen_tile(const uint8_t* raw, int bt, uint8_t* to) {
    constexpr int kMine = kTile / 8 * (HD / 64) / 4;
    const int lane = bt & 31, r8 = lane & 7, c4 = lane >> 3, w = bt >> 5;
    // with 128 dims chunks 4 (w % 2) .. and every second eight rows from 8 (w / 2), with 64 every fourth from 8 w
    const int chunk = (HD == 128 ? 4 * (w & 1) : 0) + c4, row0 = HD == 128 ? 8 * (w >> 1) : 8 * w;
    constexpr int kStep = HD == 128 ? 16 : 32;
    raw += (row0 + r8) * HD + (HD == 128 ? chunk ^ r8 : chunk ^ (r8 >> 1)) * 16;
    to += row0 / 8 * (HD / 8 * 128) + chunk * 256 + r8 * 16;
    uint4 x[kMine];
#pragma unroll
    for (int i = 0; i < kMine; ++i) x[i] = *reinterpret_cast<const uint4*>(raw + i * kStep * HD);
#pragma unroll
    for (int i = 0; i < kMine; ++i) widen(x[i], to + i * (kStep / 8) * (HD / 8 * 128));
}
__device__ __forceinline__ void tma_tile(uint32_t to, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(to),
                 "l"(map), "r"(x), "r"(y), "r"(bar)
                 : "memory");
}

// The query block of a piece as F16 terms, and the factors that undo the rows'
// powers of two: eight rows by a warp, four lanes to a row, which take its units
// of eight values in turn.
template <class T, int HD, int NT>
__device__ __noinline__ void stage_queries(const TreeArgs& a, const Piece& p, int row0, uint8_t* qt, float* fac) {
    constexpr int V = 16 / sizeof(T), kSteps = HD / 32, kPacks = 8 / V;
    const int lane = threadIdx.x & 31, r8 = lane & 7, c4 = lane >> 3, row = row0 + r8, r = p.row0 + row;
    const bool real = row < p.have;
    const int node = real ? (int)a.per_group(r) : 0;
    const T* src = (const T*)a.q.p + p.s * a.q.seq + node * a.q.node +
                   (size_t)(p.g * a.group + (real ? r - node * a.group : 0)) * a.q.head + c4 * 8;
    float big = 0.f;
    auto largest = [&](T v) {
        const float y = fabsf(to_f32(v));
        big = fmaxf(big, y <= 3.402823466e38f ? y : 0.f);
    };
    Pack<T, V> all[kSteps][kPacks] = {};
    if (real && a.wide) {
#pragma unroll
        for (int i = 0; i < kSteps; ++i)
#pragma unroll
            for (int k = 0; k < kPacks; ++k) all[i][k] = *reinterpret_cast<const Pack<T, V>*>(src + 32 * i + V * k);
#pragma unroll
        for (int i = 0; i < kSteps; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) largest(all[i][e / V].v[e % V]);
    } else if (real) {
#pragma unroll 1
        for (int i = 0; i < kSteps; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) largest(src[32 * i + e]);
    }
    big = fmaxf(big, __shfl_xor_sync(~0u, big, 8));
    big = fmaxf(big, __shfl_xor_sync(~0u, big, 16));
    const RowScale rs(big);
    uint8_t* to = qt + (row >> 3) * (HD / 8 * 128) + r8 * 16 + c4 * 128;
    auto store = [&](int i, const Pack<T, V> (&x)[kPacks]) {
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = to_f32(x[e / V].v[e % V]) * rs.f0 * rs.f1;
        const uint4 hi = make_uint4(pack_half(y[0], y[1]), pack_half(y[2], y[3]), pack_half(y[4], y[5]), pack_half(y[6], y[7]));
        *reinterpret_cast<uint4*>(to + i * 512) = hi;
        if (NT == 2)
            *reinterpret_cast<uint4*>(to + Shape<HD, NT>::kQBytes + i * 512) =
                make_uint4(rest_half(y[0], y[1], hi.x), rest_half(y[2], y[3], hi.y), rest_half(y[4], y[5], hi.z),
                           rest_half(y[6], y[7], hi.w));
    };
    // Queries of two bytes are read a second time, from L1, in a loop that is a quarter of the code to fetch (64 x 16
    // nodes 154 -> 151 us); F32 ones would not all be there still (174 -> 181 us).
    if (NT == 2 && (a.wide || !real)) {
#pragma unroll
        for (int i = 0; i < kSteps; ++i) store(i, all[i]);
    } else {
#pragma unroll 1
        for (int i = 0; i < kSteps; ++i) {
            Pack<T, V> x[kPacks] = {};
            if (real && a.wide) {
#pragma unroll
                for (int k = 0; k < kPacks; ++k) x[k] = *reinterpret_cast<const Pack<T, V>*>(src + 32 * i + V * k);
            } else if (real) {
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e / V].v[e % V] = src[32 * i + e];
            }
            store(i, x);
        }
    }
    if (c4 == 0) fac[row] = rs.undo(a.scale);
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

// ---- the kernel ----------------------------------------------------------------

struct Maps {
    CUtensorMap k, v;
};

// Tiles count through all lists: tile t is softmax group t % 2's, its S in
// buffer t % 4, its operands in stages t % 2 (K) and t % 4 (V, and the columns'
// constants).  Pieces (those with tiles) likewise.
template <class T, int HD, int NT>
__global__ void __launch_bounds__(kTcThreads, 1) k_tree_tc(const __grid_constant__ TreeArgs a, const __grid_constant__ Maps maps) {
    using S = Shape<HD, NT>;
    extern __shared__ uint8_t dyn[];
    __shared__ Bars bars;
    __shared__ Columns cols[kVs];
    __shared__ float fac_s[kFacs][kRows], m_s[2][2][kRows], l_s[2][2][kRows];
    __shared__ PieceList list;
    __shared__ uint32_t tmem_s;
    __shared__ int gave_up;
    uint8_t* raw_s = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(dyn) + 1023) & ~(uintptr_t)1023);   // [ahead][K, V]
    uint8_t* q_s = raw_s + S::kQAt;                              // [block][term]
    uint8_t* k_s = raw_s + S::kKvAt;                             // [stage]
    uint8_t* v_s = k_s + kKs * S::kTileBytes;                    // [stage]
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    list_pieces(a, list, 0);
    if (!list.count) return;                                     // whole CTA
    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_s)), "n"(S::kTmem)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (tid == 0) {
        gave_up = 0;
        for (int i = 0; i < 4; ++i) bar_init(&bars.raw[i], 1), bar_init(&bars.raw_free[i], kTeam / 32);
        for (int i = 0; i < kKs; ++i) bar_init(&bars.k_full[i], kTeam / 32), bar_init(&bars.k_free[i], 1);
        for (int i = 0; i < kVs; ++i) bar_init(&bars.v_full[i], kTeam / 32), bar_init(&bars.v_free[i], 1), bar_init(&bars.c_full[i], 1);
        for (int i = 0; i < kScores; ++i) bar_init(&bars.s_ready[i], 1), bar_init(&bars.p_ready[i], kGroup / 32);
        for (int i = 0; i < 2; ++i) bar_init(&bars.o_done[i], 1), bar_init(&bars.q_free[i], 1);
        for (int i = 0; i < kFacs; ++i) bar_init(&bars.q_full[i], kTeam / 32);
        bar_init(&bars.both, 2 * kGroup / 32);
        bar_init(&bars.o_free, 2 * kGroup / 32);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    // the first piece's queries, if it has tiles (a part may lie past what its rows see)
    const bool eager = list.piece[0].tile1 > list.piece[0].tile0;
    if (eager) stage_queries<T, HD, NT>(a, list.piece[0], warp * 8, q_s, fac_s[0]);
    fence_before();
    __syncthreads();
    fence_after();
    if (eager && tid < kTeam / 32) bar_arrive(&bars.q_full[0]);
    const uint32_t tmem = tmem_s;
    unsigned t = 0, pc = 0;                                      // tiles and pieces of the lists before
    for (int batch = 0;; ++batch) {
        const int count = list.count;
        if (warp < 8) {
            // ---- softmax ----
            const int w = warp >> 2, row = tid & 127;
            const uint32_t lanes = tmem + ((uint32_t)(32 * (warp & 3)) << 16), to = lanes + S::kO + HD * w;
            bool ok = !gave_up;
            for (int i = 0; ok && i < count; ++i) {
                const Piece& p = list.piece[i];
                const int nt = max(0, p.tile1 - p.tile0), j0 = (w ^ t) & 1;
                const int node = row < p.have ? (p.row0 + row) / a.group : -1;
                float m = -INFINITY, top = -INFINITY, fac = 0.f;
                float2 l2 = make_float2(0.f, 0.f);
                for (int j = j0; j < nt; j += 2) {
                    const unsigned tt = t + j, st = tt % kVs;
                    const uint32_t ts = lanes + kTile * (tt % kScores);
                    ok = (j != j0 || bar_wait(&bars.q_full[pc % kFacs], (pc / kFacs) & 1, &gave_up)) &&
                         bar_wait(&bars.c_full[st], (tt / kVs) & 1, &gave_up) &&
                         bar_wait(&bars.s_ready[tt % kScores], (tt / kScores) & 1, &gave_up);
                    ok = __all_sync(~0u, ok);                    // and the warp is one again for what follows
                    if (!ok) break;
                    fence_after();
                    if (j == j0) fac = fac_s[pc % kFacs][row];
                    const Columns& col = cols[st];
                    const float2 fac2 = make_float2(fac, fac);
                    const int t0 = (p.tile0 + j) * kTile;
                    const bool edge = t0 + kTile > p.len;
                    unsigned long long see = 0ull;
                    if (edge) {
                        if (node >= 0)
                            see = sees64(a.mask ? a.mask + ((size_t)p.s * a.d.max_nodes + node) * a.words : nullptr, a.words, node, t0, p.len, p.n);
                        __syncwarp();                            // the loads below are the whole warp's
                    }
                    // 32 columns at a time, in a loop: half the registers, and half the code to fetch
#pragma unroll 1
                    for (int h = 0; h < 2; ++h) {
                        float2 x[16];
                        tmem_ld32(ts + 32 * h, reinterpret_cast<uint32_t*>(x));
                        wait_ld();
                        loaded(x);
#pragma unroll
                        for (int c = 0; c < 16; c += 2) {
                            const float4 k = *reinterpret_cast<const float4*>(&col.ks[32 * h + 2 * c]),
                                         v = *reinterpret_cast<const float4*>(&col.lv[32 * h + 2 * c]);
                            x[c] = fma2(mul2(x[c], fac2), make_float2(k.x, k.y), make_float2(v.x, v.y));
                            x[c + 1] = fma2(mul2(x[c + 1], fac2), make_float2(k.z, k.w), make_float2(v.z, v.w));
                        }
                        if (edge) {
                            const uint32_t bits = (uint32_t)(see >> (32 * h));
#pragma unroll
                            for (int c = 0; c < 16; ++c) {
                                if (!(bits >> (2 * c) & 1u)) x[c].x = -INFINITY;
                                if (!(bits >> (2 * c + 1) & 1u)) x[c].y = -INFINITY;
                            }
                        }
                        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                        for (int c = 0; c < 16; ++c) mx[c & 3] = fmaxf(mx[c & 3], fmaxf(x[c].x, x[c].y));
                        const float big = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
                        top = fmaxf(top, big);
                        const bool raise = big > m + kSlack || (m == -INFINITY && big > -INFINITY);
                        if (__any_sync(~0u, raise)) {
                            // Every row of the warp goes up to the largest score it has seen, so that this is rare from then on;
                            // by a whole number of powers of two, so that what is rescaled loses no bits: m1's own rounding,
                            // 2^-24 of it, is far below half a step of the F16 weights, whose second rounding takes it back.
                            // (Weights that are subnormal by then, 2^-22 of the largest and less, do lose bits.)
                            const float m1 = m == -INFINITY ? top : m + fmaxf(ceilf(top - m), 0.f);
                            const float f = m == -INFINITY ? 0.f : exp2_fast(m - m1);
                            m = m1;
                            l2 = mul2(l2, make_float2(f, f));
                            if (j != j0) {                       // the accumulator, once its last product is in
                                ok = bar_wait(&bars.o_done[w], ((tt - 2) >> 1) & 1, &gave_up);
                                ok = __all_sync(~0u, ok);
                                if (!ok) break;
                                fence_after();
#pragma unroll 1
                                for (int c = 0; c < HD; c += 32) {
                                    float2 o[8], u[8];
                                    tmem_ld16(to + c, reinterpret_cast<uint32_t*>(o));
                                    tmem_ld16(to + c + 16, reinterpret_cast<uint32_t*>(u));
                                    wait_ld();
                                    loaded(o);
                                    loaded(u);
#pragma unroll
                                    for (int e = 0; e < 8; ++e) o[e] = mul2(o[e], make_float2(f, f)), u[e] = mul2(u[e], make_float2(f, f));
                                    tmem_st16(to + c, reinterpret_cast<const uint32_t*>(o));
                                    tmem_st16(to + c + 16, reinterpret_cast<const uint32_t*>(u));
                                }
                            }
                            if (h) {                             // and the weights of the first half
#pragma unroll 1
                                for (int q = 0; q < NT; ++q) {
                                    float2 w2[8];
                                    uint32_t* u = reinterpret_cast<uint32_t*>(w2);
                                    wait_st();
                                    tmem_ld16(ts + 16 * q, u);
                                    wait_ld();
                                    loaded(w2);
#pragma unroll
                                    for (int e = 0; e < 16; ++e) {
                                        const float2 g = __half22float2(*reinterpret_cast<const __half2*>(u + e));
                                        u[e] = pack_half(g.x * f, g.y * f);
                                    }
                                    tmem_st16(ts + 16 * q, u);
                                }
                            }
                        }
                        const float up = kPBias - (m == -INFINITY ? 0.f : m);
                        const float2 up2 = make_float2(up, up);
                        uint32_t ph[16], pl[16];
#pragma unroll
                        for (int c = 0; c < 16; c += 2) {
                            const float4 iv = *reinterpret_cast<const float4*>(&col.iv[32 * h + 2 * c]);
#pragma unroll
                            for (int u = 0; u < 2; ++u) {
                                float2 e = add2(x[c + u], up2);
                                e.x = exp2_fast(e.x);
                                e.y = exp2_fast(e.y);
                                l2 = fma2(e, u ? make_float2(iv.z, iv.w) : make_float2(iv.x, iv.y), l2);
                                ph[c + u] = pack_half(e.x, e.y);
                                if (NT == 2) pl[c + u] = rest_half(e.x, e.y, ph[c + u]);
                            }
                        }
                        // P of 32 columns over their S: 16 registers of the first term, 16 of the rest
                        tmem_st16(ts + 32 * h, ph);
                        if (NT == 2) tmem_st16(ts + 32 * h + 16, pl);
                    }
                    if (!ok) break;
                    wait_st();
                    // The group's products before this one, each in its turn: a wait tells a phase from the next only, so
                    // none may be passed over.  Long done, as a rule.
                    if (tt >= 2) ok = bar_wait(&bars.o_done[w], ((tt - 2) >> 1) & 1, &gave_up);
                    ok = __all_sync(~0u, ok);
                    if (!ok) break;
                    fence_before();
                    warp_arrive(&bars.p_ready[tt % kScores]);
                }
                if (!ok) break;
                // both groups' references and sums, then half of the dims each
                float* part = part_of(a, blockIdx.x, p.begins) + (size_t)row * (kPartHead + HD);
                if (nt > 0) {
                    const int by = pc & 1;
                    m_s[by][w][row] = m;
                    l_s[by][w][row] = l2.x + l2.y;
                    if (j0 < nt) {                               // this group's last tile
                        const unsigned last = t + nt - 1 - ((nt - 1 - j0) & 1);
                        ok = bar_wait(&bars.o_done[w], (last >> 1) & 1, &gave_up);
                    }
                    warp_arrive(&bars.both);
                    ok = bar_wait(&bars.both, pc & 1, &gave_up) && ok;
                    ok = __all_sync(~0u, ok);
                    if (!ok) break;
                    fence_after();
                    const float ma = m_s[by][0][row], mb = m_s[by][1][row], la = l_s[by][0][row], lb = l_s[by][1][row];
                    const float top = fmaxf(ma, mb);
                    // a group without a tile has m -infinity and sum 0: factor 0, and its O is not read
                    const bool has_a = nt > 1 || (t & 1) == 0, has_b = nt > 1 || (t & 1) == 1;
                    const float fa = part_weight(ma, la, top), fb = part_weight(mb, lb, top);
                    const float sum = fmaf(fa, la, fb * lb);
                    const float by_sum = p.whole ? (sum == 0.f ? 0.f : 1.f / sum) : 1.f;
                    const float2 a2 = make_float2(fa * by_sum, fa * by_sum), b2 = make_float2(fb * by_sum, fb * by_sum);
                    const int h = p.g * a.group + (p.row0 + row) % a.group;
                    T* dst = (T*)a.out.p + p.s * a.out.seq + node * a.out.node + h * a.out.head;
#pragma unroll 1
                    for (int c = w * (HD / 2); c < (w + 1) * (HD / 2); c += 16) {
                        float2 oa[8] = {}, ob[8] = {};
                        __syncwarp();                            // lanes without a row went on early
                        if (has_a) tmem_ld16(lanes + S::kO + c, reinterpret_cast<uint32_t*>(oa));
                        if (has_b) tmem_ld16(lanes + S::kO + HD + c, reinterpret_cast<uint32_t*>(ob));
                        wait_ld();
                        loaded(oa);
                        loaded(ob);
#pragma unroll
                        for (int e = 0; e < 8; ++e) oa[e] = fma2(ob[e], b2, mul2(oa[e], a2));
                        if (node < 0) continue;
                        if (!p.whole) {
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                *reinterpret_cast<float4*>(part + kPartHead + c + 4 * e) =
                                    make_float4(oa[2 * e].x, oa[2 * e].y, oa[2 * e + 1].x, oa[2 * e + 1].y);
                        } else {
                            constexpr int V = 16 / sizeof(T);
                            const float* y = reinterpret_cast<const float*>(oa);
#pragma unroll
                            for (int e = 0; e < 16; e += V) {
                                Pack<T, V> z;
#pragma unroll
                                for (int u = 0; u < V; ++u) z.v[u] = from_f32<T>(y[e + u]);
                                if (a.wide) {
                                    *reinterpret_cast<Pack<T, V>*>(dst + c + e) = z;
                                } else {
#pragma unroll
                                    for (int u = 0; u < V; ++u) dst[c + e + u] = z.v[u];
                                }
                            }
                        }
                    }
                    if (node >= 0 && w == 0) {
                        if (p.whole) write_lse(a, p.s, node, h, top, sum);
                        else part[0] = top, part[1] = sum;
                    }
                    fence_before();
                    warp_arrive(&bars.o_free);
                    ++pc;
                } else if (node >= 0) {                          // no row of the block sees these tiles
#pragma unroll 1
                    for (int c = w * (HD / 2); c < (w + 1) * (HD / 2); c += 4)
                        *reinterpret_cast<float4*>(part + kPartHead + c) = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (w == 0) part[0] = -INFINITY, part[1] = 0.f;
                }
                t += nt;
            }
        } else if (warp >= 12) {
            // ---- widen the codes, bring the queries ----
            const int bt = tid - 384;
            bool ok = !gave_up;
            unsigned qc = pc;                                    // query blocks staged
            int q_at = -1;                                       // the piece of the last
            auto stage = [&]() {                                 // the next piece's, if there is one
                do ++q_at;
                while (q_at < count && list.piece[q_at].tile1 <= list.piece[q_at].tile0);
                if (q_at >= count) return;
                if (qc || !eager) {
                    const unsigned b = qc % S::kQs, use = qc / S::kQs;
                    if (use) ok = bar_wait(&bars.q_free[b], (use - 1) & 1, &gave_up) && ok;
                    ok = __all_sync(~0u, ok);
                    if (!ok) return;
#pragma unroll 1
                    for (int r = 0; r < kRows; r += 8 * (kTeam / 32))
                        stage_queries<T, HD, NT>(a, list.piece[q_at], r + 8 * (bt >> 5), q_s + b * NT * S::kQBytes, fac_s[qc % kFacs]);
                    warp_arrive(&bars.q_full[qc % kFacs]);
                }
                ++qc;
            };
            stage();
            for (int i = 0; ok && i < count; ++i) {
                const int nt = list.piece[i].tile1 - list.piece[i].tile0;
                for (int j = 0; j < nt; ++j, ++t) {
                    const unsigned ks = t % kKs, vs = t % kVs, slot = t % S::kAhead;
                    const uint8_t* raw = raw_s + slot * 2 * S::kRawBytes;
                    ok = bar_wait(&bars.raw[slot], (t / S::kAhead) & 1, &gave_up);
                    if (ok && t >= kKs) ok = bar_wait(&bars.k_free[ks], (t / kKs - 1) & 1, &gave_up);
                    ok = __all_sync(~0u, ok);
                    if (!ok) break;
                    widen_tile<HD>(raw, bt, k_s + ks * S::kTileBytes);
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    warp_arrive(&bars.k_full[ks]);
                    if (t >= kVs) ok = bar_wait(&bars.v_free[vs], (t / kVs - 1) & 1, &gave_up);
                    ok = __all_sync(~0u, ok);
                    if (!ok) break;
                    widen_tile<HD>(raw + S::kRawBytes, bt, v_s + vs * S::kTileBytes);
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    warp_arrive(&bars.v_full[vs]);
                    warp_arrive(&bars.raw_free[slot]);
                    // with two blocks, while the softmax still has tiles of this piece before it; with one, behind its last S
                    if (j == (S::kQs == 2 ? min(nt, kVs) : nt) - 1) stage();
                    if (!ok) {
                        ++t;
                        break;
                    }
                }
            }
            pc = qc;                                             // every piece of the list with tiles has its queries
        } else if (warp == 10) {
            // ---- ask for the codes ----
            const uint32_t raw_a = smem_addr(raw_s);
            const unsigned t0 = t;
            bool ok = !gave_up;
            for (int i = 0; ok && i < count; ++i) {
                const Piece& p = list.piece[i];
                const int x = p.g * HD;
                int y = (int)p.base_row + p.tile0 * kTile;
                for (int left = p.tile1 - p.tile0; left > 0; --left, ++t, y += kTile) {
                    const unsigned slot = t % S::kAhead, use = t / S::kAhead;
                    if (use) ok = bar_wait(&bars.raw_free[slot], (use - 1) & 1, &gave_up);   // the codes before have been read
                    ok = __all_sync(~0u, ok);
                    if (!ok) break;
                    if (lane == 0) {
                        const uint32_t bar = smem_addr(&bars.raw[slot]), to = raw_a + slot * 2 * S::kRawBytes;
                        asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(2 * S::kRawBytes) : "memory");
                        tma_tile(to, &maps.k, x, y, bar);
                        tma_tile(to + S::kRawBytes, &maps.v, x, y, bar);
                    }
                    __syncwarp();
                }
            }
            // copies still on their way, if a wait gave up
            if (!ok)
                for (unsigned i = t > t0 + S::kAhead ? t - S::kAhead : t0; i < t; ++i)
                    bar_wait(&bars.raw[i % S::kAhead], (i / S::kAhead) & 1, &gave_up, true);
        } else if (warp == 9) {
            // ---- make the columns' constants ----
            bool ok = !gave_up;
            for (int i = 0; ok && i < count; ++i) {
                const Piece& p = list.piece[i];
                const int last = p.len + p.n - 1, end = p.tile1;
                int tile = p.tile0;
                if (tile >= end) continue;
                // the scales of rows 2 lane and 2 lane + 1, a tile ahead
                const float *ks = a.c.ks + p.base_row, *vs = a.c.vs + p.base_row;
                auto scales = [&](int at) {
                    const int r0 = min(at * kTile + 2 * lane, last), r1 = min(at * kTile + 2 * lane + 1, last);
                    return make_float4(__ldg(ks + r0), __ldg(ks + r1), __ldg(vs + r0), __ldg(vs + r1));
                };
                float4 sc = scales(tile);
                for (; tile < end; ++tile, ++t) {
                    const unsigned st = t % kVs;
                    const float4 now = sc;
                    if (tile + 1 < end) sc = scales(tile + 1);
                    if (t >= kVs) ok = bar_wait(&bars.v_free[st], (t / kVs - 1) & 1, &gave_up);
                    ok = __all_sync(~0u, ok);
                    if (!ok) break;
                    *reinterpret_cast<float2*>(&cols[st].ks[2 * lane]) = make_float2(now.x, now.y);
                    *reinterpret_cast<float2*>(&cols[st].lv[2 * lane]) = make_float2(log_vs(now.z), log_vs(now.w));
                    *reinterpret_cast<float2*>(&cols[st].iv[2 * lane]) = make_float2(inv_vs(now.z), inv_vs(now.w));
                    warp_arrive(&bars.c_full[st]);
                }
            }
        } else {
            // ---- issue the products ----
            // The whole warp goes along, so that what the instructions take is uniform; one lane issues.
            constexpr uint32_t kGroupStride = HD / 8 * 128;       // eight rows
            const bool issues = elected();
            const unsigned t0 = t;
            bool ok = !gave_up;
            if (warp == 8) {
                constexpr uint32_t id = idesc_f16(kRows, kTile, false);
                // descriptors of the operands' first blocks; others are so many 16-byte units further
                const uint64_t qd = umma_desc(smem_addr(q_s), 128, kGroupStride), kd = umma_desc(smem_addr(k_s), 128, kGroupStride);
                for (int i = 0; ok && i < count; ++i) {
                    int left = list.piece[i].tile1 - list.piece[i].tile0;
                    if (left <= 0) continue;
                    const uint64_t q0 = qd + (pc % S::kQs) * (NT * S::kQBytes / 16);
                    ok = __all_sync(~0u, bar_wait(&bars.q_full[pc % kFacs], (pc / kFacs) & 1, &gave_up));
                    for (; ok && left > 0; --left, ++t) {
                        const unsigned ks = t % kKs, sb = t % kScores;
                        // the keys; and the buffer: P of four tiles before has been used
                        ok = bar_wait(&bars.k_full[ks], (t / kKs) & 1, &gave_up) &&
                             (t < kScores || bar_wait(&bars.v_free[t % kVs], (t / kVs - 1) & 1, &gave_up));
                        ok = __all_sync(~0u, ok);
                        if (!ok) break;
                        fence_after();
                        if (issues) {
                            const uint64_t k0 = kd + ks * (S::kTileBytes / 16);
                            const uint32_t d = tmem + kTile * sb;
                            // the smaller term first (qx_tree.cuh)
#pragma unroll
                            for (int q = NT - 1; q >= 0; --q)
#pragma unroll
                                for (int k = 0; k < HD / 16; ++k)
                                    mma_ss(d, q0 + q * (S::kQBytes / 16) + k * 16, k0 + k * 16, id, q < NT - 1 || k > 0);
                            mma_commit(&bars.s_ready[sb]);
                            mma_commit(&bars.k_free[ks]);
                            if (left == 1) mma_commit(&bars.q_free[pc % S::kQs]);
                        }
                        __syncwarp();
                    }
                    ++pc;
                }
                // what this warp has in flight, if a wait gave up
                if (!ok)
                    for (unsigned i = t > t0 + kScores ? t - kScores : t0; i < t; ++i)
                        bar_wait(&bars.s_ready[i % kScores], (i / kScores) & 1, &gave_up, true);
            } else {
                constexpr uint32_t id = idesc_f16(kRows, HD, true);
                const uint64_t vd = umma_desc(smem_addr(v_s), kGroupStride, 128);
                for (int i = 0; ok && i < count; ++i) {
                    const int nt = list.piece[i].tile1 - list.piece[i].tile0;
                    if (nt <= 0) continue;
                    if (pc) ok = __all_sync(~0u, bar_wait(&bars.o_free, (pc - 1) & 1, &gave_up));
                    for (int j = 0; ok && j < nt; ++j, ++t) {
                        const unsigned vs = t % kVs, sb = t % kScores;
                        ok = bar_wait(&bars.p_ready[sb], (t / kScores) & 1, &gave_up) &&
                             bar_wait(&bars.v_full[vs], (t / kVs) & 1, &gave_up);
                        ok = __all_sync(~0u, ok);
                        if (!ok) break;
                        fence_after();
                        if (issues) {
                            const uint64_t v0 = vd + vs * (S::kTileBytes / 16);
                            const uint32_t d = tmem + S::kO + HD * (t & 1), ap = tmem + kTile * sb, add = j >= 2;
#pragma unroll
                            for (int q = 0; q < NT; ++q)
#pragma unroll
                                for (int k = 0; k < kTile / 16; ++k)
                                    mma_ts(d, ap + 32 * (k >> 1) + 16 * q + 8 * (k & 1), v0 + k * (2 * kGroupStride / 16), id,
                                           q + k > 0 ? 1u : add);
                            mma_commit(&bars.v_free[vs]);
                            mma_commit(&bars.o_done[t & 1]);
                        }
                        __syncwarp();
                    }
                    ++pc;
                }
                if (!ok)
                    for (unsigned i = t > t0 + 2 ? t - 2 : t0; i < t; ++i)
                        bar_wait(&bars.o_done[i & 1], (i >> 1) & 1, &gave_up, true);
            }
        }
        __syncwarp();
        __syncthreads();                                         // every role is done with the list
        const bool again = !gave_up && list.more;
        __syncthreads();                                         // and has seen whether there is another
        if (!again) break;
        list_pieces(a, list, batch + 1);
    }
    fence_before();
    __syncthreads();
    fence_after();
    if (tid == 0 && gave_up && a.status) atomicOr(a.status, QX_CUDA_STATUS_TIMEOUT);
    if (warp == 8) {
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(S::kTmem) : "memory");
    }
}

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                 const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled encoder() {
    static const EncodeTiled fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult r{};
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &r) != cudaSuccess ||
            r != cudaDriverEntryPointSuccess)
            p = nullptr;
        return (EncodeTiled)p;
    }();
    return fn;
}

// The whole cache as rows of codes; boxes of 64 rows of one KV head.  Rows past
// the last are filled with zeros, so a tile may run over the end.
cudaError_t cache_maps(const Cache& c, Maps& m) {
    const EncodeTiled encode = encoder();
    if (!encode) return cudaErrorNotSupported;
    const cuuint64_t row = (cuuint64_t)c.kv_heads * c.head_dim;
    const cuuint64_t dims[2] = {row, (cuuint64_t)cache_rows(c)}, strides[1] = {row};
    const cuuint32_t box[2] = {(cuuint32_t)c.head_dim, (cuuint32_t)kTile}, steps[2] = {1, 1};
    const CUtensorMapSwizzle sw = c.head_dim == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B;
    for (int i = 0; i < 2; ++i)
        if (encode(i ? &m.v : &m.k, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, i ? c.v : c.k, dims, strides, box, steps,
                   CU_TENSOR_MAP_INTERLEAVE_NONE, sw, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
            return cudaErrorInvalidValue;
    return cudaSuccess;
}

template <class T, int HD, int NT>
cudaError_t run(TreeArgs& a, int sms, cudaStream_t st) {
    a.ctas = sms < kMaxCtas / 8 ? sms : kMaxCtas / 8;
    a.per_cta = Over((uint32_t)a.ctas);
    Maps maps;
    cudaError_t e = cache_maps(a.c, maps);
    if (e != cudaSuccess) return e;
    e = cudaFuncSetAttribute((const void*)k_tree_tc<T, HD, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<HD, NT>::kSmem);
    if (e != cudaSuccess) return e;
    k_tree_tc<T, HD, NT><<<a.ctas, kTcThreads, Shape<HD, NT>::kSmem, st>>>(a, maps);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_tree_tc(TreeArgs& a, uint32_t type, int sms, cudaStream_t st) {
    if (a.c.head_dim == 128) {
        if (type == QX_CUDA_F32) return run<float, 128, 2>(a, sms, st);
        return type == QX_CUDA_F16 ? run<__half, 128, 1>(a, sms, st) : run<__nv_bfloat16, 128, 1>(a, sms, st);
    }
    if (type == QX_CUDA_F32) return run<float, 64, 2>(a, sms, st);
    return type == QX_CUDA_F16 ? run<__half, 64, 1>(a, sms, st) : run<__nv_bfloat16, 64, 1>(a, sms, st);
}

}  // namespace ops
}  // namespace qx
