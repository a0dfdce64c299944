// What the kernels of qx_cuda_tree_attention share (qx_tree.cu, qx_tree_tc.cu):
// the mathematics, how the work is cut and shared out, and F16 operands.
//
// For a query row q (one node, one head) and cache row t with codes k_t, v_t
// and scales ks_t, vs_t:
//     s_t = scale ks_t (q . k_t),   o = sum_t e^(s_t) vs_t v_t / sum_t e^(s_t).
// In base 2 and with the value scale inside the exponent,
//     x_t = s_t log2(e) + log2(vs_t),   P_t = 2^(x_t - m + 8),   m >= max x_t - 7,
//     o = sum_t P_t v_t / sum_t (P_t / vs_t):
// what meets the codes v_t in the second product is one F16 number in
// (0, 2^15] per (row, t) whatever the scales are, and the running reference m
// is the only thing the accumulators are ever rescaled by.  The price: P_t / vs_t
// is lost where P_t is below 2^-126, x_t more than 133 below the largest, so
// value scales may lie 2^100 apart (what is lost then has a share of 2^-33).
// And P_t below 2^-25, 2^-32 of the largest, rounds to 0 in F16: such rows add
// nothing to o, which shows only in dims where all larger rows hold zeros.
//
// INT8 codes are exact in F16, so both products run on the tensor cores as F16
// with F32 accumulation.  F16 and BF16 queries are one F16 term: a row is
// multiplied by a power of two that puts its largest value in [2^13, 2^14)
// (BF16 values more than 2^38 below it lose bits).  F32 queries, and P_t then
// too, are two F16 terms (hi + the rest, 22 bits).  Everything else is F32.
// (The tensor cores' sums are F32 numbers that are cut off, not rounded, at each
// step of 16: the smaller term of the queries comes first, which halved the
// error of F32 calls, and outputs come out small by up to 3e-6 of themselves
// where a CTA has a hundred tiles of a unit: 64 x 16 nodes over 4096 rows 3.9e-6
// against 1.6e-6 for F32 sums that are rounded.)
// That P_t is one F16 term for half types is a choice: its 2^-11 is the size of
// an F16 output's own rounding (16 nodes over 4096 random rows: error 2.9e-4
// against 2.1e-4 with P_t in F32) and an eighth of a BF16 output's (1.68e-3
// against 1.66e-3), while a second term takes as long as F32 queries do (64 x 16
// nodes 173 against 151 us).
//
// Work is cut into units (sequence, KV head, block of rows) and those into
// tiles of 64 cache rows; the tiles of all units, laid end to end, are shared
// out evenly over the CTAs.  A CTA that has all of a unit's tiles writes its
// rows; parts of a unit go to the workspace as (m, sum, o) and k_tree_join
// adds them in the order of their tiles.
#pragma once
#include "qx_ops.cuh"

namespace qx {
namespace ops {

constexpr int kTile = 64;                 // cache rows
constexpr int kScanThreads = 128;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kPBias = 8.f;
constexpr float kSlack = 7.f;             // how far x_t may pass the reference: P_t <= 2^15, and F16 ends at 2^16
constexpr float kMinLogVs = -90.f;        // value scales below 2^-90 count as that: 2^15 2^90 times 65536 rows still fits the F32 sum
constexpr int kPartHead = 4;              // floats of a part's row before its o: m, sum, two unused (16-byte rows)
constexpr int kMaxCtas = 148 * 8;

struct Tensor {
    void* p;
    size_t seq, node, head;
};

// Parts to join: those of CTAs c - 1 .. c - 1 + parts - 1 (none: nothing to do), c the record's index.
struct Join {
    int parts, s, g, row0, have;
};

struct TreeArgs {
    Cache c;
    Drafts d;
    int layer, q_heads, group, block_rows, row_blocks;   // row_blocks: of max_nodes * group rows
    Tensor q, out;
    int wide;                                             // q and out allow 16-byte accesses
    const unsigned long long* mask;
    int words;
    float scale;
    float* lse;                                           // caller's, or null
    float* lse2;                                          // workspace: base-2 log sums, for the mass
    float* mass;
    float* parts;                                         // [2 * ctas][block_rows][kPartHead + head_dim]
    Join* joins;                                          // [ctas]
    int ctas;
    Over per_block, per_heads, per_group, per_cta;        // division by block_rows, kv_heads, group, ctas
    uint32_t* status;
};

// The tensor-core kernel for blocks of 128 query rows (qx_tree_tc.cu).
// type: QX_CUDA_F32, F16 or BF16; sets a.ctas.
cudaError_t launch_tree_tc(TreeArgs& a, uint32_t type, int sms, cudaStream_t st);

#ifdef __CUDACC__
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// ---- which tiles are whose -----------------------------------------------------

// A sequence's share of the work: `units` units of `tiles` tiles each.  (The
// host refuses calls whose tiles could pass 2^31.)
struct SeqWork {
    int tiles, units, slot, len, n;
    __device__ __forceinline__ int all() const { return tiles * units; }
};
__device__ __forceinline__ SeqWork seq_work(const TreeArgs& a, int s, bool report) {
    const int slot = a.d.slots[s], len = a.d.lens[s], n = a.d.count(s);
    if (!fits(a.c, a.d, slot, len, n)) {
        if (report && a.status) atomicOr(a.status, QX_CUDA_STATUS_RANGE);
        return {};
    }
    if (n == 0) return {};
    return {(len + n + kTile - 1) / kTile, a.c.kv_heads * (int)a.per_block(n * a.group + a.block_rows - 1), slot, len, n};
}

// The tiles of all units laid end to end, cut into shares that differ by one
// tile at most; never more CTAs than tiles.
struct Shares {
    int busy, each, extra;
    __device__ __forceinline__ Shares(const TreeArgs& a, int total) {
        busy = min(a.ctas, total);
        each = total < a.ctas ? 1 : (int)a.per_cta(total);
        extra = total < a.ctas ? 0 : total - each * busy;
    }
    __device__ __forceinline__ int begin(int c) const { return each * c + min(c, extra); }
    // the CTA that has tile t
    __device__ __forceinline__ int of(int t) const {
        const int longer = extra * (each + 1);
        return each == 1 && t >= longer ? extra + t - longer : t < longer ? t / (each + 1) : extra + (t - longer) / each;
    }
};

// One unit's tiles that a CTA has.
struct Piece {
    size_t base_row;                       // the sequence's row 0 in the layer
    int s, len, n, g, row0, have;          // query rows row0 .. row0 + have of KV head g
    int tile0, tile1;                      // tiles; none (tile1 <= tile0) where no row of the block sees them
    int begins, whole;
};
// The pieces of a CTA, kList at a time: every thread of the first 128 looks at
// its own sequences and writes down those units of theirs that the CTA's share
// of the tiles meets, so that no one follows a chain of loads.
constexpr int kList = 32;
struct PieceList {
    Piece piece[kList];
    int tile_sum[kScanThreads / 32], unit_sum[kScanThreads / 32], first_unit;
    int count, more;
};
// Fills the list with pieces batch * kList and on; whole CTA, and it must be
// done with the pieces before.  The first batch also writes the CTA's join
// record.  (Not inlined: instruction fetch is what kernels with several roles
// run short of.)
static __device__ __noinline__ void list_pieces(const TreeArgs& a, PieceList& sh, int batch) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, per = (a.d.seqs + kScanThreads - 1) / kScanThreads;
    const bool scans = threadIdx.x < kScanThreads;
    const int s0 = scans ? min(a.d.seqs, (int)threadIdx.x * per) : 0, s1 = scans ? min(a.d.seqs, s0 + per) : 0;
    int tiles = 0, units = 0;
    SeqWork one{};                                        // kept where a thread has one sequence
    for (int s = s0; s < s1; ++s) {
        one = seq_work(a, s, blockIdx.x == 0 && batch == 0);
        tiles += one.all();
        units += one.units;
    }
    auto work = [&](int s) { return per == 1 ? one : seq_work(a, s, false); };
    int tl = tiles, un = units;
    if (scans) {
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int t = __shfl_up_sync(~0u, tl, o), u = __shfl_up_sync(~0u, un, o);
            if (lane >= o) tl += t, un += u;
        }
        if (lane == 31) sh.tile_sum[w] = tl, sh.unit_sum[w] = un;
    }
    if (threadIdx.x == 0) {
        sh.count = sh.more = 0;
        if (batch == 0) a.joins[blockIdx.x].parts = 0;
    }
    __syncthreads();
    int first = tl - tiles, unit0 = un - units, total = 0;
#pragma unroll
    for (int i = 0; i < kScanThreads / 32; ++i) {
        if (i < w) first += sh.tile_sum[i], unit0 += sh.unit_sum[i];
        total += sh.tile_sum[i];
    }
    const Shares cut(a, total);
    const int c = blockIdx.x, begin = c < cut.busy ? cut.begin(c) : 0, end = c < cut.busy ? cut.begin(c + 1) : 0;
    const bool meets = begin < end && first < end && first + tiles > begin;
    if (meets && begin >= first) {                        // the unit that holds the share's first tile
        int f = first, u = unit0;
        for (int s = s0; s < s1; ++s) {
            const SeqWork k = work(s);
            if (begin >= f && begin < f + k.all()) sh.first_unit = u + (begin - f) / k.tiles;
            f += k.all();
            u += k.units;
        }
    }
    __syncthreads();
    if (meets)
        for (int s = s0; s < s1; ++s) {
            const SeqWork k = work(s);
            if (k.units && first < end && first + k.all() > begin) {
                const int u0 = begin > first ? (begin - first) / k.tiles : 0;
                const int u1 = end < first + k.all() ? (end - first + k.tiles - 1) / k.tiles : k.units;
                for (int u = u0; u < u1; ++u) {
                    const int at = unit0 + u - sh.first_unit - batch * kList;
                    if (at < 0) continue;
                    if (at >= kList) {
                        sh.more = 1;
                        break;
                    }
                    const int f = first + u * k.tiles;
                    Piece& p = sh.piece[at];
                    p.s = s;
                    p.len = k.len, p.n = k.n;
                    const int block = (int)a.per_heads(u);
                    p.g = u - block * a.c.kv_heads;
                    p.row0 = block * a.block_rows;
                    p.have = min(a.block_rows, p.n * a.group - p.row0);
                    p.tile0 = max(begin, f) - f;
                    p.tile1 = min(k.tiles, end - f);
                    p.begins = p.tile0 == 0;
                    p.whole = p.begins && p.tile1 == k.tiles;
                    p.base_row = (size_t)k.slot * a.c.slot_rows + (size_t)a.layer * a.c.layer_rows;
                    // of the CTAs that share a unit, the second sees to its joining
                    if (at == 0 && batch == 0 && !p.begins && cut.begin(c - 1) <= f)
                        a.joins[c] = {cut.of(f + k.tiles - 1) - c + 2, s, p.g, p.row0, p.have};
                    // in a chain no row of the block sees past its last node
                    const int limit = a.mask ? p.len + p.n : min(p.len + p.n, p.len + (p.row0 + p.have - 1) / a.group + 1);
                    p.tile1 = min(p.tile1, (limit + kTile - 1) / kTile);
                    atomicAdd(&sh.count, 1);
                }
            }
            first += k.all();
            unit0 += k.units;
        }
    __syncthreads();
}
// Where the part of a piece goes: a CTA has at most one that ends a unit
// begun elsewhere, and one that begins a unit.
__device__ __forceinline__ float* part_of(const TreeArgs& a, int cta, bool begins) {
    return a.parts + (size_t)(2 * cta + (begins ? 1 : 0)) * a.block_rows * (kPartHead + a.c.head_dim);
}

// ---- parts -----------------------------------------------------------------------

// The factor of a part whose reference is m when parts are joined at mx; a
// part that saw nothing has none, and one that met a NaN keeps it.
__device__ __forceinline__ float part_weight(float m, float l, float mx) {
    return m == -INFINITY ? (l == 0.f ? 0.f : 1.f) : exp2_fast(m - mx);
}
__device__ __forceinline__ void write_lse(const TreeArgs& a, int s, int node, int h, float m, float sum) {
    const float lg = sum == 0.f ? -INFINITY : m - kPBias + log2f(sum);
    const size_t li = ((size_t)s * a.d.max_nodes + node) * a.q_heads + h;
    if (a.lse) a.lse[li] = lg * 0.69314718055994531f;
    if (a.lse2) a.lse2[li] = lg;
}

// ---- operands ------------------------------------------------------------------

// Four INT8 codes as F16: b + 128 as the low byte of 0x64xx is 1024 + b + 128,
// and subtracting 1152 is exact.  `biased` holds b + 128 (b ^ 0x80).
__device__ __forceinline__ uint32_t sub1152(uint32_t x) {
    const __half2 r = __hsub2(*reinterpret_cast<__half2*>(&x), __half2half2(__ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t low_pair(uint32_t biased) { return sub1152(__byte_perm(biased, 0x64646464u, 0x4140)); }
__device__ __forceinline__ uint32_t high_pair(uint32_t biased) { return sub1152(__byte_perm(biased, 0x64646464u, 0x4342)); }

__device__ __forceinline__ uint32_t pack_half(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// The pair minus its F16 rounding, as F16.
__device__ __forceinline__ uint32_t rest_half(float a, float b, uint32_t hi) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hi));
    return pack_half(a - f.x, b - f.y);
}
// The power of two 2^up that puts `big` (the largest finite magnitude of a
// row) in [2^13, 2^14), as two factors that are normal numbers.
struct RowScale {
    int up;
    float f0, f1;
    __device__ __forceinline__ explicit RowScale(float big) {
        const int b = __float_as_int(big);
        const int e = b < 0x00800000 ? b ? 31 - __clz(b) - 149 : 0 : (b >> 23) - 127;
        up = 13 - e;
        const int u0 = up / 2;
        f0 = pow2(u0);
        f1 = pow2(up - u0);
    }
    __device__ __forceinline__ static float pow2(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }
    // what turns the integer dot product of scaled queries and codes into a base-2 score, but for ks_t
    __device__ __forceinline__ float undo(float scale) const { return scale * kLog2e * pow2(-(up / 2)) * pow2(up / 2 - up); }
};

// log2(vs) for the exponent, and 1 / vs for the sum of weights.
__device__ __forceinline__ float log_vs(float vs) {
    return vs >= 0.f ? fmaxf(__log2f(vs), kMinLogVs) : __int_as_float(0x7fc00000);
}
__device__ __forceinline__ float inv_vs(float vs) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(vs));   // one ulp
    return vs > 0x1p-90f ? r : 0x1p90f;
}

// ---- visibility ----------------------------------------------------------------

// Which of the 64 rows from t0 on a node sees, as bits (mrow: its mask words, or null).
__device__ __forceinline__ unsigned long long sees64(const unsigned long long* mrow, int words, int node, int t0, int len,
                                                     int n) {
    const unsigned long long all = ~0ull;
    auto first = [&](int c) { return c <= 0 ? 0ull : c >= 64 ? all : (1ull << c) - 1ull; };   // bits 0 .. c - 1
    if (!mrow) return first(min(len + n, len + node + 1) - t0);
    unsigned long long w;
    if (t0 >= len) {
        const int b = t0 - len, i = b >> 6, sh = b & 63;
        w = i < words ? mrow[i] >> sh : 0ull;
        if (sh && i + 1 < words) w |= mrow[i + 1] << (64 - sh);
    } else {
        const int c = len - t0;
        w = c >= 64 ? all : first(c) | mrow[0] << c;
    }
    return w & first(len + n - t0);
}
#endif  // __CUDACC__

}  // namespace ops
}  // namespace qx
