// Tree attention on the tcgen05 tensor cores (qx_tree.cuh has the mathematics
// and the cut of the work): blocks of 128 query rows against tiles of 64 cache
// rows, one persistent CTA per SM.
//
// Roles, by warp:
//   0-3, 4-7   two softmax groups, which take a piece's tiles in turn; a thread
//              has one query row (TMEM lane), and each group its own scores,
//              reference, sum and output accumulator
//   8-11       bring the cache: INT8 codes from global memory into registers
//              two tiles ahead, to F16 in shared memory, and the per-row
//              constants of the scores; also the query block of each piece
//   12         issues the MMAs: S = Q K^T (128 x 64), then O += P V with P read
//              from TMEM, where it overwrites the S it came from
// S of one group is computed while the other group is in its softmax.
//
// Shared memory operands are in the no-swizzle core-matrix layout: 8 rows x 16
// bytes each, [row / 8][dim / 8][row % 8].  That one layout is K-major for
// K (rows = N, dims = K) and for Q, and MN-major for V (dims = N, rows = K), so
// nothing is transposed.
#include <cmath>

#include "qx_tree.cuh"

namespace qx {
namespace ops {
namespace {

constexpr int kRows = 128, kGroup = 128, kBring = 128, kTcThreads = 2 * kGroup + kBring + 32;
constexpr int kStages = 4, kAhead = 2;

template <int HD, int NT>
struct Shape {
    static constexpr int kTileBytes = kTile * HD * 2;          // K or V of a tile
    static constexpr int kQBytes = kRows * HD * 2;             // one term of Q
    static constexpr int kSmem = NT * kQBytes + kStages * 2 * kTileBytes + 128;
    static constexpr int kTmem = HD == 128 ? 512 : 256;        // S of both groups, then O of both (a power of two)
};

struct Bars {
    unsigned long long full[kStages], empty[kStages], s_ready[2], p_ready[2], o_done[2], q_full, q_free, both, o_free;
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
// Bounded wait for a phase (2 s; a healthy one takes microseconds).  Gives up
// at once where another role has.
__device__ __forceinline__ bool bar_wait(unsigned long long* b, unsigned parity, volatile int* gave_up) {
    unsigned long long t0 = 0;
    for (unsigned i = 0;; ++i) {
        uint32_t done;
        asm volatile(
            "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
            : "=r"(done)
            : "r"(smem_addr(b)), "r"(parity)
            : "memory");
        if (done) return true;
        if ((i & 255u) == 255u) {
            unsigned long long t;
            asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
            if (!t0) t0 = t;
            if (*gave_up || t - t0 > 2000000000ull) {
                *gave_up = 1;
                return false;
            }
        }
    }
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

// The tiles of a CTA, one after another over its pieces.
struct TileCursor {
    Cursor c;
    Piece p;
    int tile;
    bool more;
    __device__ __forceinline__ void find(const TreeArgs& a) {
        do more = c.next(a, p);
        while (more && p.tile1 <= p.tile0);
        tile = p.tile0;
    }
    __device__ __forceinline__ void next(const TreeArgs& a) {
        if (++tile >= p.tile1) find(a);
    }
};

// A bringing thread's share of a tile's bytes.  Eight lanes take eight rows of
// one 16-byte chunk (their F16 stores then fill 128 consecutive bytes), the
// four groups of eight lanes four chunks.
template <int HD>
struct Raw {
    static constexpr int kLoads = kTile * HD / 16 / kBring;    // of K, and of V
    uint4 k[kLoads], v[kLoads];
    float ks, vs;
};
template <int HD>
__device__ __forceinline__ void where(int bt, int i, int& row, int& chunk) {
    const int w = bt >> 5, lane = bt & 31, slot = w + 4 * i;   // warp-wide accesses: [chunk / 4][row / 8]
    row = (slot & 7) * 8 + (lane & 7);
    chunk = (slot >> 3) * 4 + (lane >> 3);
}
template <int HD>
__device__ __forceinline__ void load_raw(const TreeArgs& a, const TileCursor& t, int bt, Raw<HD>& r) {
    const int last = t.p.len + t.p.n - 1, row0 = t.tile * kTile;
    const size_t KV = (size_t)a.c.kv_heads * HD;
#pragma unroll
    for (int i = 0; i < Raw<HD>::kLoads; ++i) {
        int row, chunk;
        where<HD>(bt, i, row, chunk);
        const size_t at = (t.p.base_row + min(row0 + row, last)) * KV + (size_t)t.p.g * HD + 16 * chunk;
        r.k[i] = __ldg(reinterpret_cast<const uint4*>(a.c.k + at));
        r.v[i] = __ldg(reinterpret_cast<const uint4*>(a.c.v + at));
    }
    if (bt < kTile) {
        const size_t row = t.p.base_row + min(row0 + bt, last);
        r.ks = __ldg(a.c.ks + row);
        r.vs = __ldg(a.c.vs + row);
    }
}
// 16 codes as F16: two 16-byte units of an operand tile.
__device__ __forceinline__ void widen(const uint4& w, uint8_t* to) {
    const uint32_t c[4] = {w.x ^ 0x80808080u, w.y ^ 0x80808080u, w.z ^ 0x80808080u, w.w ^ 0x80808080u};
    *reinterpret_cast<uint4*>(to) = make_uint4(low_pair(c[0]), high_pair(c[0]), low_pair(c[1]), high_pair(c[1]));
    *reinterpret_cast<uint4*>(to + 128) = make_uint4(low_pair(c[2]), high_pair(c[2]), low_pair(c[3]), high_pair(c[3]));
}
template <int HD>
__device__ __forceinline__ void store_raw(const Raw<HD>& r, int bt, uint8_t* kt, uint8_t* vt, Columns& col) {
#pragma unroll
    for (int i = 0; i < Raw<HD>::kLoads; ++i) {
        int row, chunk;
        where<HD>(bt, i, row, chunk);
        const int o = (row >> 3) * (HD / 8 * 128) + 2 * chunk * 128 + (row & 7) * 16;
        widen(r.k[i], kt + o);
        widen(r.v[i], vt + o);
    }
    if (bt < kTile) {
        col.ks[bt] = r.ks;
        col.lv[bt] = log_vs(r.vs);
        col.iv[bt] = inv_vs(r.vs);
    }
}

// Query row bt of a piece: F16 terms into the operand, the undoing factor to fac.
template <class T, int HD, int NT>
__device__ __forceinline__ void stage_row(const TreeArgs& a, const Piece& p, int bt, uint8_t* qt, float* fac) {
    constexpr int V = 16 / sizeof(T), U = 8;
    const int r = p.row0 + bt;
    const bool real = bt < p.have;
    const T* src = (const T*)a.q.p + p.s * a.q.seq + (real ? r / a.group : 0) * a.q.node +
                   (size_t)(p.g * a.group + (real ? r % a.group : 0)) * a.q.head;
    auto read = [&](int i) {
        Pack<T, V> x;
        if (a.wide) {
            x = *reinterpret_cast<const Pack<T, V>*>(src + i);
        } else {
#pragma unroll
            for (int u = 0; u < V; ++u) x.v[u] = src[i + u];
        }
        return x;
    };
    float big = 0.f;
    if (real)
        for (int i = 0; i < HD; i += U * V) {
            Pack<T, V> x[U];
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (i + u * V < HD) x[u] = read(i + u * V);
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (i + u * V < HD)
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        const float y = to_f32(x[u].v[e]);
                        big = fmaxf(big, isfinite(y) ? fabsf(y) : 0.f);
                    }
        }
    const RowScale rs(big);
    uint8_t* to = qt + (bt >> 3) * (HD / 8 * 128) + (bt & 7) * 16;
#pragma unroll 2
    for (int d = 0; d < HD; d += 8) {
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; e += V) {
            if (real) {
                const Pack<T, V> x = read(d + e);
#pragma unroll
                for (int u = 0; u < V; ++u) y[e + u] = to_f32(x.v[u]) * rs.f0 * rs.f1;
            } else {
#pragma unroll
                for (int u = 0; u < V; ++u) y[e + u] = 0.f;
            }
        }
        const uint4 hi = make_uint4(pack_half(y[0], y[1]), pack_half(y[2], y[3]), pack_half(y[4], y[5]), pack_half(y[6], y[7]));
        *reinterpret_cast<uint4*>(to + d / 8 * 128) = hi;
        if (NT == 2)
            *reinterpret_cast<uint4*>(to + Shape<HD, NT>::kQBytes + d / 8 * 128) =
                make_uint4(rest_half(y[0], y[1], hi.x), rest_half(y[2], y[3], hi.y), rest_half(y[4], y[5], hi.z),
                           rest_half(y[6], y[7], hi.w));
    }
    fac[bt] = rs.undo(a.scale);
}

// ---- the kernel ----------------------------------------------------------------

template <class T, int HD, int NT>
__global__ void __launch_bounds__(kTcThreads, 1) k_tree_tc(TreeArgs a) {
    using S = Shape<HD, NT>;
    extern __shared__ uint8_t dyn[];
    __shared__ Bars bars;
    __shared__ Columns cols[kStages];
    __shared__ float fac_s[2][kRows], m_s[2][2][kRows], l_s[2][2][kRows];
    __shared__ ScanShared scan;
    __shared__ uint32_t tmem_s;
    __shared__ int gave_up;
    uint8_t* q_s = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(dyn) + 127) & ~(uintptr_t)127);
    uint8_t* kv_s = q_s + NT * S::kQBytes;                       // [stage][K, V]
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    Cursor cur;
    if (!begin_share(a, scan, cur)) return;                      // whole CTA
    if (warp == 12) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_s)), "n"(S::kTmem)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (tid == 0) {
        gave_up = 0;
        for (int i = 0; i < kStages; ++i) bar_init(&bars.full[i], kBring), bar_init(&bars.empty[i], 1);
        for (int w = 0; w < 2; ++w) bar_init(&bars.s_ready[w], 1), bar_init(&bars.p_ready[w], kGroup), bar_init(&bars.o_done[w], 1);
        bar_init(&bars.q_full, kBring);
        bar_init(&bars.q_free, 1);
        bar_init(&bars.both, 2 * kGroup);
        bar_init(&bars.o_free, 2 * kGroup);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = tmem_s;
    // columns: S of group w at 64 w (P over it), O of group w at 128 + HD w
    if (warp < 8) {
        // ---- softmax ----
        const int w = warp >> 2, row = tid & 127;
        const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
        const uint32_t ts = tmem + lanes + 64 * w, to = tmem + lanes + 128 + HD * w;
        unsigned tiles = 0, mine = 0, pieces = 0;                // tiles before this piece, of this group, pieces with tiles
        Piece p;
        bool ok = true;
        while (ok && cur.next(a, p)) {
            const int nt = max(0, p.tile1 - p.tile0);
            float m = -INFINITY;
            float2 l2 = make_float2(0.f, 0.f);
            const bool real = row < p.have;
            const int node = real ? (p.row0 + row) / a.group : 0;
            const unsigned long long* mrow = a.mask ? a.mask + ((size_t)p.s * a.d.max_nodes + node) * a.words : nullptr;
            float fac = 0.f;
            for (int j = w; j < nt; j += 2) {
                const unsigned t = tiles + j, st = t % kStages;
                ok = bar_wait(&bars.full[st], (t / kStages) & 1, &gave_up) && bar_wait(&bars.s_ready[w], mine & 1, &gave_up);
                ok = __all_sync(~0u, ok);                        // and the warp is one again for what follows
                if (!ok) break;
                fence_after();
                if (j == w) fac = fac_s[pieces & 1][row];
                float2 x[32];
                tmem_ld32(ts, reinterpret_cast<uint32_t*>(x));
                tmem_ld32(ts + 32, reinterpret_cast<uint32_t*>(x + 16));
                wait_ld();
                const Columns& col = cols[st];
                const float2 fac2 = make_float2(fac, fac);
#pragma unroll
                for (int i = 0; i < 32; i += 2) {
                    const float4 k = *reinterpret_cast<const float4*>(&col.ks[2 * i]), v = *reinterpret_cast<const float4*>(&col.lv[2 * i]);
                    x[i] = fma2(mul2(x[i], fac2), make_float2(k.x, k.y), make_float2(v.x, v.y));
                    x[i + 1] = fma2(mul2(x[i + 1], fac2), make_float2(k.z, k.w), make_float2(v.z, v.w));
                }
                const int t0 = (p.tile0 + j) * kTile;
                if (t0 + kTile > p.len) {
                    const unsigned long long see = real ? sees64(mrow, a.words, node, t0, p.len, p.n) : 0ull;
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        if (!(see >> (2 * i) & 1ull)) x[i].x = -INFINITY;
                        if (!(see >> (2 * i + 1) & 1ull)) x[i].y = -INFINITY;
                    }
                }
                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int i = 0; i < 32; ++i) mx[i & 3] = fmaxf(mx[i & 3], fmaxf(x[i].x, x[i].y));
                const float big = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
                const bool raise = big > m + kSlack || (m == -INFINITY && big > -INFINITY);
                if (__any_sync(~0u, raise)) {
                    const float f = raise ? exp2_fast(m - big) : 1.f;
                    if (raise) m = big;
                    l2 = mul2(l2, make_float2(f, f));
                    if (j != w) {                                // an accumulator to rescale, once its last product is in
                        ok = bar_wait(&bars.o_done[w], (mine - 1) & 1, &gave_up);
                        ok = __all_sync(~0u, ok);
                        if (!ok) break;
                        fence_after();
                        for (int c = 0; c < HD; c += 16) {
                            float2 o[8];
                            tmem_ld16(to + c, reinterpret_cast<uint32_t*>(o));
                            wait_ld();
#pragma unroll
                            for (int i = 0; i < 8; ++i) o[i] = mul2(o[i], make_float2(f, f));
                            tmem_st16(to + c, reinterpret_cast<const uint32_t*>(o));
                        }
                    }
                }
                const float up = kPBias - (m == -INFINITY ? 0.f : m);
                const float2 up2 = make_float2(up, up);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t ph[16], pl[16];
#pragma unroll
                    for (int i = 0; i < 16; i += 2) {
                        const float4 iv = *reinterpret_cast<const float4*>(&col.iv[32 * h + 2 * i]);
#pragma unroll
                        for (int u = 0; u < 2; ++u) {
                            float2 e = add2(x[16 * h + i + u], up2);
                            e.x = exp2_fast(e.x);
                            e.y = exp2_fast(e.y);
                            l2 = fma2(e, u ? make_float2(iv.z, iv.w) : make_float2(iv.x, iv.y), l2);
                            ph[i + u] = pack_half(e.x, e.y);
                            if (NT == 2) pl[i + u] = rest_half(e.x, e.y, ph[i + u]);
                        }
                    }
                    tmem_st16(ts + 16 * h, ph);
                    if (NT == 2) tmem_st16(ts + 32 + 16 * h, pl);
                }
                wait_st();
                fence_before();
                bar_arrive(&bars.p_ready[w]);
                ++mine;
            }
            if (!ok) break;
            // both groups' references and sums, then half of the dims each
            const int by = pieces & 1;
            float* part = part_of(a, blockIdx.x, p.begins) + (size_t)row * (kPartHead + HD);
            if (nt > 0) {
                m_s[by][w][row] = m;
                l_s[by][w][row] = l2.x + l2.y;
                if (w < nt) ok = bar_wait(&bars.o_done[w], (mine - 1) & 1, &gave_up);
                bar_arrive(&bars.both);
                ok = bar_wait(&bars.both, pieces & 1, &gave_up) && ok;
                ok = __all_sync(~0u, ok);
                if (!ok) break;
                fence_after();
                const float ma = m_s[by][0][row], mb = m_s[by][1][row], la = l_s[by][0][row], lb = l_s[by][1][row];
                const float top = fmaxf(ma, mb);
                const float fa = part_weight(ma, la, top), fb = nt > 1 ? part_weight(mb, lb, top) : 0.f;
                const float sum = fmaf(fa, la, fb * lb);
                const float by_sum = p.whole ? (sum == 0.f ? 0.f : 1.f / sum) : 1.f;
                const float2 a2 = make_float2(fa * by_sum, fa * by_sum), b2 = make_float2(fb * by_sum, fb * by_sum);
                const int h = p.g * a.group + (p.row0 + row) % a.group;
                T* dst = (T*)a.out.p + p.s * a.out.seq + node * a.out.node + h * a.out.head;
                for (int c = w * (HD / 2); c < (w + 1) * (HD / 2); c += 16) {
                    float2 oa[8], ob[8];
                    tmem_ld16(tmem + lanes + 128 + c, reinterpret_cast<uint32_t*>(oa));
                    if (nt > 1) tmem_ld16(tmem + lanes + 128 + HD + c, reinterpret_cast<uint32_t*>(ob));
                    wait_ld();
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        oa[i] = mul2(oa[i], a2);
                        if (nt > 1) oa[i] = fma2(ob[i], b2, oa[i]);
                    }
                    if (!real) continue;
                    if (!p.whole) {
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            *reinterpret_cast<float4*>(part + kPartHead + c + 4 * i) =
                                make_float4(oa[2 * i].x, oa[2 * i].y, oa[2 * i + 1].x, oa[2 * i + 1].y);
                    } else {
                        constexpr int V = 16 / sizeof(T);
                        const float* y = reinterpret_cast<const float*>(oa);
#pragma unroll
                        for (int i = 0; i < 16; i += V) {
                            Pack<T, V> z;
#pragma unroll
                            for (int u = 0; u < V; ++u) z.v[u] = from_f32<T>(y[i + u]);
                            if (a.wide) {
                                *reinterpret_cast<Pack<T, V>*>(dst + c + i) = z;
                            } else {
#pragma unroll
                                for (int u = 0; u < V; ++u) dst[c + i + u] = z.v[u];
                            }
                        }
                    }
                }
                if (real && w == 0) {
                    if (p.whole) write_lse(a, p.s, node, h, top, sum);
                    else part[0] = top, part[1] = sum;
                }
                fence_before();
                bar_arrive(&bars.o_free);
                ++pieces;
            } else if (real) {                                   // no row of the block sees these tiles
                for (int c = w * (HD / 2); c < (w + 1) * (HD / 2); c += 4)
                    *reinterpret_cast<float4*>(part + kPartHead + c) = make_float4(0.f, 0.f, 0.f, 0.f);
                if (w == 0) part[0] = -INFINITY, part[1] = 0.f;
            }
            tiles += nt;
        }
    } else if (warp < 12) {
        // ---- bring the cache ----
        const int bt = tid - 2 * kGroup;
        TileCursor ld, cv;
        ld.c = cv.c = cur;
        ld.find(a);
        cv.find(a);
        Raw<HD> raw[kAhead];
#pragma unroll
        for (int d = 0; d < kAhead; ++d)
            if (ld.more) load_raw<HD>(a, ld, bt, raw[d]), ld.next(a);
        unsigned t = 0, pieces = 0;
        bool ok = true, fresh = true;
        while (ok && cv.more) {
#pragma unroll
            for (int d = 0; d < kAhead; ++d) {
                if (!ok || !cv.more) break;
                if (fresh) {
                    if (pieces) ok = bar_wait(&bars.q_free, (pieces - 1) & 1, &gave_up);
                    if (!ok) break;
                    stage_row<T, HD, NT>(a, cv.p, bt, q_s, fac_s[pieces & 1]);
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    bar_arrive(&bars.q_full);
                    ++pieces;
                }
                const unsigned st = t % kStages, use = t / kStages;
                if (use) ok = bar_wait(&bars.empty[st], (use - 1) & 1, &gave_up);
                if (!ok) break;
                uint8_t* kt = kv_s + (size_t)st * 2 * S::kTileBytes;
                store_raw<HD>(raw[d], bt, kt, kt + S::kTileBytes, cols[st]);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                bar_arrive(&bars.full[st]);
                ++t;
                fresh = cv.tile + 1 >= cv.p.tile1;
                cv.next(a);
                if (ld.more) load_raw<HD>(a, ld, bt, raw[d]), ld.next(a);
            }
        }
    } else if (lane == 0) {
        // ---- issue the products ----
        const uint32_t qa = smem_addr(q_s), kva = smem_addr(kv_s);
        constexpr uint32_t kGroupStride = HD / 8 * 128;           // eight rows
        constexpr uint32_t id_s = idesc_f16(kRows, kTile, false), id_o = idesc_f16(kRows, HD, true);
        unsigned t = 0, mine[2] = {0, 0}, pieces = 0;
        Piece p;
        bool ok = true;
        while (ok && cur.next(a, p)) {
            const int nt = max(0, p.tile1 - p.tile0);
            if (!nt) continue;
            ok = bar_wait(&bars.q_full, pieces & 1, &gave_up);
            bool fresh_o = true;
            for (int j = 0; ok && j <= nt; ++j) {
                if (j < nt) {                                    // S of tile j
                    const unsigned st = (t + j) % kStages;
                    ok = bar_wait(&bars.full[st], ((t + j) / kStages) & 1, &gave_up);
                    if (!ok) break;
                    fence_after();
                    const uint32_t kt = kva + st * 2 * S::kTileBytes, d = tmem + 64 * (j & 1);
#pragma unroll
                    for (int q = 0; q < NT; ++q)
#pragma unroll
                        for (int k = 0; k < HD / 16; ++k)
                            mma_ss(d, umma_desc(qa + q * S::kQBytes + k * 256, 128, kGroupStride),
                                   umma_desc(kt + k * 256, 128, kGroupStride), id_s, q + k > 0);
                    mma_commit(&bars.s_ready[j & 1]);
                    if (j == nt - 1) mma_commit(&bars.q_free);
                }
                if (j > 0) {                                     // O of tile j - 1
                    const int w = (j - 1) & 1;
                    const unsigned st = (t + j - 1) % kStages;
                    if (fresh_o && pieces) ok = bar_wait(&bars.o_free, (pieces - 1) & 1, &gave_up);
                    fresh_o = false;
                    ok = ok && bar_wait(&bars.p_ready[w], mine[w] & 1, &gave_up);
                    if (!ok) break;
                    ++mine[w];
                    fence_after();
                    const uint32_t vt = kva + st * 2 * S::kTileBytes + S::kTileBytes, d = tmem + 128 + HD * w, ap = tmem + 64 * w;
#pragma unroll
                    for (int q = 0; q < NT; ++q)
#pragma unroll
                        for (int k = 0; k < kTile / 16; ++k)
                            mma_ts(d, ap + 32 * q + 8 * k, umma_desc(vt + k * 2 * kGroupStride, kGroupStride, 128), id_o,
                                   j - 1 >= 2 || q + k > 0);
                    mma_commit(&bars.empty[st]);
                    mma_commit(&bars.o_done[w]);
                }
            }
            t += nt;
            ++pieces;
        }
        // the last products are in before TMEM goes (the softmax groups waited for them, unless a wait gave up)
        if (!ok)
            for (int w = 0; w < 2; ++w)
                if (mine[w]) bar_wait(&bars.o_done[w], (mine[w] - 1) & 1, &gave_up);
    }
    __syncwarp();
    fence_before();
    __syncthreads();
    fence_after();
    if (tid == 0 && gave_up && a.status) atomicOr(a.status, QX_CUDA_STATUS_TIMEOUT);
    if (warp == 12) {
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(S::kTmem) : "memory");
    }
}

template <class T, int HD, int NT>
cudaError_t run(TreeArgs& a, int sms, cudaStream_t st) {
    a.ctas = sms < kMaxCtas / 8 ? sms : kMaxCtas / 8;
    const cudaError_t e = cudaFuncSetAttribute((const void*)k_tree_tc<T, HD, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               Shape<HD, NT>::kSmem);
    if (e != cudaSuccess) return e;
    k_tree_tc<T, HD, NT><<<a.ctas, kTcThreads, Shape<HD, NT>::kSmem, st>>>(a);
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
