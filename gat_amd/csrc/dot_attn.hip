// Scaled dot-product attention on [B, N, heads, D] rows with the framework's additive mask, and its gradients.
//
//   z_ij = scale <q_i, k_j> + bias_ij,   P_ij = exp(z_ij - lse_i) over the attended keys of row i,   out_i = sum_j P_ij v_j
//   dv_j = sum_i P_ij do_i,   dz_ij = P_ij (<do_i, v_j> - delta_i),   delta_i = <do_i, out_i>,
//   dq_i = scale sum_j dz_ij k_j,   dk_j = scale sum_i dz_ij q_i
//
// A key is attended when j < key_sizes[b] and its bias is above kAttended (masks are written with -1e9; a NaN in a bias masks its
// entry).  A row without an attended key, or behind query_sizes[b], has out = 0 and no gradients.  Query heads h share the
// key/value head h / (H / Hkv): a "row" below is a pair (query i, head of the group), i * group + g, so that
// the rows of all sharing heads walk the same staged keys.
//
// The forward keeps the running maximum and sum of each row (one pass over the keys) and saves lse; the backward
// forms P again from lse in two passes without atomics: one per query tile for dq (and delta), one per key tile for dk, dv
// (which adds up the sharing heads as it walks their rows).
//
// Matrix instructions: v_mfma_f32_16x16x4_f32 and v_mfma_f32_16x16x32_bf16, sums in fp32.  The scores are formed transposed (keys down, queries
// across the lanes): a lane then holds four consecutive keys of ONE query, the softmax statistics are one register each,
// and the probabilities sit in the operand layout of the second product as they are: they never go through LDS.  For that
// product bf16 rows have P and dz as two bf16 each, high and low (Wide16), or, beyond 1024 nodes without a mask, rounded to one (uint16_t: half a step of 2^-8, as its
// other operand has and its result is stored with; see dot_wide16).
//
// A mask with few entries is walked entry by entry (dot_entries_*), a denser one in tiles, without the 16 x 16 parts that it leaves empty.
//
// What the tiles measure, forward / dq / dk, dv: 4 graphs of 2048 to 4096 nodes, 16 heads on 4 of 128, bf16: 520 / 655 / 1180 us, 594 / 708 / 524
// TFLOP/s of products (a large bf16 product reaches 1140).  Matrix units 37 / 45 / 29 % busy, vector units 49 / 41 / 22 %, LDS 28 / 30 / 24 %: none is
// full, 1.6 waves a SIMD wait for their own reads (33 / 34 / 64 % of their time), most of all in dk, dv with two operands that are read column-wise.  16 x 1024 nodes, 4 heads of 64, fp32: 92 / 121 / 164 us, 187 / 213 / 210 TFLOP/s of fp32 accuracy (a
// large fp32 product: 153).  1024 graphs of 246 nodes, 8 heads of 8, 10 % attended: 375 / 419 / 589 us for 2 / 3 / 4 products of 8 wide operands each:
// matrix instructions (45 to 58 % of the cycles) and exponentials, masks and the bits' tests (51 to 36 %) share the SIMDs and nearly fill them.
// One query on 98000 keys, 8 heads on 2 of 64, two graphs: 20.2 us in bf16, 5.0 TB/s (a large copy: 4.7), with the join 24; 51 in fp32 with the join, 4.0 TB/s.
//
// fp32 rows are computed in one of two ways.  A few rows: on v_mfma_f32_16x16x4_f32 (256 flop / clock / CU, which the vector units cannot use
// meanwhile).  Otherwise (Split3): every number x is split exactly into three bf16, h + m + l with 8 bits each, and a product is the six
// terms hh + hm + mh + mm + hl + lh on the bf16 instructions (16 times the rate, beside the vector units; what is left out is below 2^-23
// of the product).  q, k, v and dout are split once into rows of three parts, probabilities and dz in registers.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "common.h"
#include "device_common.h"

namespace gatmi {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef short i16x8 __attribute__((ext_vector_type(8)));
struct __attribute__((packed, aligned(4))) f32x4_u { float v[4]; };       // a 16-byte access at 4-byte alignment

constexpr float kAttended = -1e8f;
// two numbers as h + m + l, bf16 each (exact: what is left of 24 bits after two roundings to 8 has 8 at most), packed pairwise
__device__ __forceinline__ void split3_pack(float a, float b, uint32_t &h, uint32_t &m, uint32_t &l) {
    h = pack_bf16x2(a, b);
    a -= __uint_as_float(h << 16);
    b -= __uint_as_float(h & 0xffff0000u);
    m = pack_bf16x2(a, b);
    l = pack_bf16x2(a - __uint_as_float(m << 16), b - __uint_as_float(m & 0xffff0000u));
}

constexpr int kSplitsMax = 256;

// ---- rows in LDS and operand fragments -----------------------------------------------------------------------------------
// Staged rows are DP elements wide and lie in LDS without padding, because the loads go straight from memory to LDS (64 lanes
// write 1 KB in lane order).  Instead the 16-byte pieces of row r are permuted by an exclusive or with a number made of r, so that the lanes of
// one LDS read, which want the same piece of many rows, find them in different banks.
// A fragment is what a lane holds of 16 rows x KD elements: lane (n = l & 15, q = l >> 4) the PIECE bytes at q * PIECE of the
// fragment's part of row n.
struct Split3 {};                                        // fp32 as three bf16
struct Wide16 {};                                        // bf16, P and dz as two bf16
template <typename T> struct ElemOf { using type = T; };
template <> struct ElemOf<Split3> { using type = float; };
template <> struct ElemOf<Wide16> { using type = uint16_t; };
template <typename T> using Elem = typename ElemOf<T>::type;              // what results are stored as
template <typename T> constexpr bool kSplit = std::is_same_v<T, Split3>;

template <typename T, int DP> struct Shape {
    static constexpr int PLANES = 1;
    static constexpr int SIZE = (int)sizeof(T), ROW = DP * SIZE, CPR = ROW / 16;         // bytes and 16-byte pieces of a row
    static constexpr bool NARROW = ROW == 32;                                              // one fragment of 8 bytes a lane
    static constexpr int PIECE = NARROW ? 8 : 16, FRAGS = ROW / (4 * PIECE), ELEMS = PIECE / SIZE, KD = 4 * ELEMS, GROUPS = FRAGS;
    static constexpr int CHUNK = SIZE == 4 ? 16 : 32;                                      // rows that one fragment of the second product covers
    static constexpr int KT = (SIZE == 4 && DP == 128) ? 32 : 64;                         // rows of a staged tile
    static constexpr int DT = (DP + 15) / 16;                                            // 16-wide tiles of a result row
    static constexpr int KTW = ROW >= 512 ? 16 : (ROW >= 128 ? 32 : 64);               // where each wave stages tiles of its own
    static constexpr int PLANE = KT * ROW, TILE = PLANE;
    // 16-row tiles of a wave: two where the accumulators and operands of two fit the 256 registers that leave two waves on a SIMD
    static constexpr int NQ = SIZE == 4 && DP >= 64 ? 1 : 2;
    static constexpr int nk(bool) { return SIZE == 4 && DP >= 64 ? 1 : 2; }
    __device__ static __forceinline__ int swizzle(int r) {      // the same for r and r + 16
        if constexpr (CPR >= 16) return r & 15;
        else return (r / (16 / CPR)) & (CPR - 1);
    }
    __device__ static __forceinline__ int at(int r, int byte) { return r * ROW + (((byte >> 4) ^ swizzle(r)) << 4) + (byte & 15); }
};

// Rows of three parts: planes of their own (h of the whole row, then m, then l), and the six terms are six instructions over the same fragments.
template <int DP> struct Shape<Split3, DP> : Shape<uint16_t, DP> {
    using H = Shape<uint16_t, DP>;
    static constexpr int PLANES = 3, COLS = 3 * DP, FRAGS = 3 * H::GROUPS, KT = DP >= 64 ? 32 : 64, PLANE = KT * H::ROW, TILE = 3 * PLANE;
    static constexpr int NQ = 2;
    static constexpr int nk(bool masked) { return DP == 32 || (DP == 128 && !masked) ? 2 : 1; }
};

template <int DP> struct Shape<Wide16, DP> : Shape<uint16_t, DP> {
    static constexpr int NQ = DP == 128 ? 1 : 2;
    static constexpr int nk(bool masked) { return DP == 128 || (DP == 64 && masked) ? 1 : 2; }
};

struct FragF { float v[4]; };
struct FragH { uint4 v; };
template <typename T> struct FragOf;
template <> struct FragOf<float> { using type = FragF; };
template <> struct FragOf<uint16_t> { using type = FragH; };
template <> struct FragOf<Split3> { using type = FragH; };
template <> struct FragOf<Wide16> { using type = FragH; };
template <typename T> using Frag = typename FragOf<T>::type;
// operands of the second product: one fragment, or one of each part
template <typename T> struct ManyOf { Frag<T> p[1]; };
template <> struct ManyOf<Split3> { FragH p[3]; };
template <> struct ManyOf<Wide16> { FragH p[2]; };

template <typename T, int DP>
__device__ __forceinline__ Frag<T> frag_load(const char *p) {
    if constexpr (std::is_same_v<T, float>) {
        if constexpr (Shape<T, DP>::NARROW) {
            const float2 u = *reinterpret_cast<const float2 *>(p);
            return FragF{{u.x, u.y, 0.f, 0.f}};
        } else {
            const float4 u = *reinterpret_cast<const float4 *>(p);
            return FragF{{u.x, u.y, u.z, u.w}};
        }
    } else {
        if constexpr (Shape<T, DP>::NARROW) {
            const uint2 u = *reinterpret_cast<const uint2 *>(p);
            return FragH{make_uint4(u.x, u.y, 0, 0)};
        } else {
            return FragH{*reinterpret_cast<const uint4 *>(p)};
        }
    }
}
// the fragments of one row in memory: zeros behind its D elements and where there is no row
template <typename T, int DP>
__device__ __forceinline__ void row_frags(const char *row, int D, bool ok, Frag<T> (&f)[Shape<T, DP>::FRAGS]) {
    using S = Shape<T, DP>;
    const int q = (threadIdx.x & 63) >> 4;
#pragma unroll
    for (int c = 0; c < S::FRAGS; ++c) {
        if constexpr (kSplit<T>) {                                      // the parts come padded with zeros
            const int byte = (c / S::GROUPS) * S::ROW + (c % S::GROUPS) * 64 + q * 16;
            if (ok) f[c] = frag_load<T, DP>(row + byte);
            else f[c] = Frag<T>{};
        } else {
            const int e = c * S::KD + q * S::ELEMS;
            if (ok && e < D) f[c] = frag_load<T, DP>(row + e * S::SIZE);
            else f[c] = Frag<T>{};
        }
    }
}
template <typename T>
__device__ __forceinline__ Frag<T> frag_negated(Frag<T> f) {
    if constexpr (std::is_same_v<T, float>) return FragF{{-f.v[0], -f.v[1], -f.v[2], -f.v[3]}};
    else return FragH{make_uint4(f.v.x ^ 0x80008000u, f.v.y ^ 0x80008000u, f.v.z ^ 0x80008000u, f.v.w ^ 0x80008000u)};
}

// acc += A B over the KD elements of one fragment
template <typename T, int DP>
__device__ __forceinline__ void mma(const Frag<T> &a, const Frag<T> &b, f32x4 &acc) {
    if constexpr (std::is_same_v<T, float>) {
#pragma unroll
        for (int t = 0; t < Shape<T, DP>::ELEMS; ++t) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[t], b.v[t], acc, 0, 0, 0);
    } else if constexpr (Shape<T, DP>::NARROW) {
        acc = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(i16x4, make_uint2(a.v.x, a.v.y)), __builtin_bit_cast(i16x4, make_uint2(b.v.x, b.v.y)), acc, 0, 0, 0);
    } else {
        acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a.v), __builtin_bit_cast(bf16x8, b.v), acc, 0, 0, 0);
    }
}
// the terms of a product of parts, small ones first: part of A, part of B
constexpr int kTerms = 6;
constexpr int kTermA[kTerms] = {2, 0, 1, 1, 0, 0}, kTermB[kTerms] = {0, 2, 1, 0, 1, 0};

// Results of matrix instructions that a branch stands between them and their first other reader: hipcc (ROCm 7.2) counts the wait states such a
// reader needs (10 at most here) along straight code and can miss them behind a branch, and the hardware does not wait by itself.  The
// wait is therefore taken here, next to the matrix instructions, and the values pass through it.
__device__ __forceinline__ void settle(f32x4 &a) { asm volatile("s_nop 10" : "+v"(a)); }
__device__ __forceinline__ void settle(f32x4 &a, f32x4 &b) { asm volatile("s_nop 10" : "+v"(a), "+v"(b)); }
__device__ __forceinline__ void settle(f32x4 &a, f32x4 &b, f32x4 &c, f32x4 &d) { asm volatile("s_nop 10" : "+v"(a), "+v"(b), "+v"(c), "+v"(d)); }
// the same for sums that stay where they are (the end of a loop's body)
__device__ __forceinline__ void settle_sums() {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_nop 10" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}
template <int N>
__device__ __forceinline__ void settle(f32x4 (&z)[N]) {
    static_assert(N == 1 || N == 2 || N == 4, "tiles of a lane");
    if constexpr (N == 1) settle(z[0]);
    else if constexpr (N == 2) settle(z[0], z[1]);
    else settle(z[0], z[1], z[2], z[3]);
}
template <int M, int N>
__device__ __forceinline__ void settle(f32x4 (&z)[M][N]) {
    static_assert(M == 1 || M == 2, "tiles of a lane");
    if constexpr (M == 1) settle(z[0]);
    else if constexpr (N == 1) settle(z[0][0], z[1][0]);
    else if constexpr (N == 2) settle(z[0][0], z[0][1], z[1][0], z[1][1]);
    else asm volatile("s_nop 10" : "+v"(z[0][0]), "+v"(z[0][1]), "+v"(z[0][2]), "+v"(z[0][3]), "+v"(z[1][0]), "+v"(z[1][1]), "+v"(z[1][2]), "+v"(z[1][3]));
}

// The second product sums over CHUNK staged rows.  Its B operand is made of score tiles (C layout: row 4 q + r of a
// tile in register r), its A operand reads the staged rows column-wise in the same order of rows.
template <typename T>
__device__ __forceinline__ ManyOf<T> frag_scores(const f32x4 *tile) {
    if constexpr (std::is_same_v<T, float>) {
        return {FragF{{tile[0][0], tile[0][1], tile[0][2], tile[0][3]}}};
    } else if constexpr (std::is_same_v<T, Wide16>) {
        uint32_t h[4], l[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float x = tile[i >> 1][2 * (i & 1)], y = tile[i >> 1][2 * (i & 1) + 1];
            h[i] = pack_bf16x2(x, y);
            l[i] = pack_bf16x2(x - __uint_as_float(h[i] << 16), y - __uint_as_float(h[i] & 0xffff0000u));
        }
        return {FragH{make_uint4(h[0], h[1], h[2], h[3])}, FragH{make_uint4(l[0], l[1], l[2], l[3])}};
    } else if constexpr (!kSplit<T>) {
        return {FragH{make_uint4(pack_bf16x2(tile[0][0], tile[0][1]), pack_bf16x2(tile[0][2], tile[0][3]), pack_bf16x2(tile[1][0], tile[1][1]), pack_bf16x2(tile[1][2], tile[1][3]))}};
    } else {
        ManyOf<T> f;
        uint32_t w[3][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) split3_pack(tile[i >> 1][2 * (i & 1)], tile[i >> 1][2 * (i & 1) + 1], w[0][i], w[1][i], w[2][i]);
#pragma unroll
        for (int k = 0; k < 3; ++k) f.p[k] = FragH{make_uint4(w[k][0], w[k][1], w[k][2], w[k][3])};
        return f;
    }
}
// the 16 columns from byte `col` on of CHUNK staged 16-bit rows: ds_read_b64_tr_b16, in which 16 lanes give the addresses of a 4 x 16 block
// (lane i: row i / 4, columns 4 (i % 4) ..) and each gets a column of it
template <typename S>
__device__ __forceinline__ FragH turned_h(const char *plane, int row0, int col) {
    const int lane = threadIdx.x & 63;
    const char *p = plane + S::at(row0 + 4 * (lane >> 4) + ((lane & 15) >> 2), col + (lane & 3) * 8);
    using lds4 = __attribute__((address_space(3))) i16x4;
    const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4 *)p);
    const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4 *)(p + 16 * S::ROW));
    return FragH{__builtin_bit_cast(uint4, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7))};
}
// row0 a multiple of CHUNK; result columns 16 t ..
template <typename T, int DP>
__device__ __forceinline__ ManyOf<T> frag_turned(const char *tile, int row0, int t) {
    using S = Shape<T, DP>;
    if constexpr (std::is_same_v<T, float>) {
        const int lane = threadIdx.x & 63, n = DP == 8 ? lane & 7 : lane & 15;                  // DP = 8: the upper eight columns are not used
        FragF f;
#pragma unroll
        for (int r = 0; r < 4; ++r) f.v[r] = *reinterpret_cast<const float *>(tile + S::at(row0 + 4 * (lane >> 4) + r, (16 * t + n) * 4));
        return {f};
    } else if constexpr (!kSplit<T>) {
        return {turned_h<S>(tile, row0, 32 * t)};
    } else {
        return {turned_h<S>(tile, row0, 32 * t), turned_h<S>(tile + S::PLANE, row0, 32 * t), turned_h<S>(tile + 2 * S::PLANE, row0, 32 * t)};
    }
}
// acc[u] += A B[u] over CHUNK rows
template <typename T, int DP, int N, bool SKIP>
__device__ __forceinline__ void mma_rows(const ManyOf<T> &a, const ManyOf<T> (&b)[N], const bool (&use)[N], f32x4 *const (&acc)[N]) {
    if constexpr (!kSplit<T>) {
#pragma unroll
        for (int u = 0; u < N; ++u)
            if (use[u]) {
                if constexpr (std::is_same_v<T, Wide16>) mma<T, 64>(a.p[0], b[u].p[1], *acc[u]);
                mma<T, 64>(a.p[0], b[u].p[0], *acc[u]);
            }
    } else {
#pragma unroll
        for (int u = 0; u < N; ++u)
            if (use[u]) {
#pragma unroll
                for (int k = 0; k < kTerms; ++k) mma<T, 64>(a.p[kTermA[k]], b[u].p[kTermB[k]], *acc[u]);
            }
        if constexpr (SKIP) settle_sums();                              // branches stand between: see settle
    }
}
template <typename T, int DP>
__device__ __forceinline__ Frag<T> frag_row(const char *tile, int row0, int c) {
    using S = Shape<T, DP>;
    const int lane = threadIdx.x & 63, q = lane >> 4, row = row0 + (lane & 15);
    return frag_load<T, DP>(tile + (c / S::GROUPS) * S::PLANE + S::at(row, (c % S::GROUPS) * 4 * S::PIECE + q * S::PIECE));
}
// acc[u] += (16 staged rows from row0) . (row in registers b[u]), over the whole width
template <typename T, int DP, int N, bool SKIP>
__device__ __forceinline__ void mma_scores(const char *tile, int row0, const Frag<T> (&b)[N][Shape<T, DP>::FRAGS], const bool (&use)[N], f32x4 *const (&acc)[N]) {
    using S = Shape<T, DP>;
#pragma unroll
    for (int c = 0; c < S::GROUPS; ++c) {
        Frag<T> a[S::PLANES];
#pragma unroll
        for (int k = 0; k < S::PLANES; ++k) a[k] = frag_row<T, DP>(tile, row0, k * S::GROUPS + c);
        if constexpr (S::PLANES == 1) {
#pragma unroll
            for (int u = 0; u < N; ++u)
                if (use[u]) mma<T, DP>(a[0], b[u][c], *acc[u]);
        } else {
#pragma unroll
            for (int u = 0; u < N; ++u)
                if (use[u]) {
#pragma unroll
                    for (int k = 0; k < kTerms; ++k) mma<T, DP>(a[kTermA[k]], b[u][kTermB[k] * S::GROUPS + c], *acc[u]);
                }
        }
    }
    if constexpr (SKIP && kSplit<T>) settle_sums();
}

// how a kernel gets the mask: there is none; as floats (the few rows of KEYW); as bits
constexpr int kNoMask = 0, kFloats = 1, kBits = 2;

// ---- arguments ---------------------------------------------------------------------------------------------------------
struct DotRows {              // [B, N, heads, D] rows: element strides, D contiguous
    const void *p;
    int64_t batch, node, head;
};

struct DotArgs {
    DotRows q, k, v, o, d_o;
    void *out, *dq, *dk, *dv;           // contiguous [B, N, heads, D]
    uint16_t *out_low;                  // what rounding to bf16 took from out, rows as it; or null
    float *lse, *delta;                 // [B, H, Nq]: log2 of the row's sum of exponentials; <do, out>
    const float *bias;
    int64_t bias_batch, bias_row;
    const ulonglong2 *row_words, *col_words;      // the mask as bits (dot_mask_kernel), or null
    int64_t row_words_batch, col_words_batch;     // of one graph; 0: one mask for all
    const int32_t *sparse;                        // per mask: 1 where the kernels that walk single entries do the work; or null
    int sparse_batch;                             // 1, or 0: one mask for all
    const int32_t *key_sizes, *query_sizes;
    int64_t b0;                         // first graph of this launch
    int B, Nq, Nk, H, Hkv, group, D;    // B: graphs of this launch
    int tiles, splits;                  // row (or key) tiles, key ranges
    float scale, scale2;                // scale2 = |scale| log2 e; the sign is carried by q
    float *part_o, *part_ml;            // split forward: [rows of the launch][splits][D], [..][2]
};

__device__ __forceinline__ bool by_entries(const DotArgs &a, int64_t b) { return a.sparse && a.sparse[b * a.sparse_batch] != 0; }
// row i of a head of graph b
template <typename S>
__device__ __forceinline__ const char *row_of(const DotRows &x, int64_t b, int64_t i, int head) {
    return reinterpret_cast<const char *>(x.p) + (b * x.batch + i * x.node + head * x.head) * S::SIZE;
}
__device__ __forceinline__ int graph_size(const int32_t *sizes, int64_t b, int n) { return sizes ? max(0, min(sizes[b], n)) : n; }

// Which (graph, key/value head, tile, split) a block of the 1-d grid works on.  Blocks go to the eight dies in turn and each die has an
// L2 of its own.  What shares data forms a group whose blocks go to one die, next to each other: without a mask the tiles of one
// (graph, head), which read the same keys and values; with a mask the heads of one (graph, tile, split), which read the same part of it.
// Groups are dealt to the dies in turn (so that graphs of unequal sizes spread), the last groups that do not fill a round are cut into eight equal pieces.
struct DotBlock { int64_t b; int hk, tile, split; bool ok; };
template <int MASK>
__device__ __forceinline__ DotBlock dot_block(const DotArgs &a) {
    const uint32_t inner = MASK ? a.Hkv : a.tiles * a.splits, groups = MASK ? (uint32_t)a.B * a.tiles * a.splits : (uint32_t)a.B * a.Hkv;
    const uint32_t die = blockIdx.x & 7, at = blockIdx.x >> 3, whole = groups / 8 * inner;       // blocks of a die that belong to whole rounds
    uint32_t group = at / inner * 8 + die, i = at % inner;
    DotBlock r;
    r.ok = true;
    if (at >= whole) {
        const uint32_t rest = groups % 8 * inner, per = (rest + 7) / 8, item = die * per + (at - whole);
        r.ok = at - whole < per && item < rest;
        group = groups / 8 * 8 + item / inner;
        i = item % inner;
    }
    if constexpr (MASK != kNoMask) {
        r.hk = i;
        r.split = group % a.splits; group /= a.splits;
        r.tile = group % a.tiles;
        r.b = a.b0 + group / a.tiles;
    } else {
        r.split = i % a.splits;
        r.tile = i / a.splits;
        r.hk = group % a.Hkv;
        r.b = a.b0 + group / a.Hkv;
    }
    return r;
}

// ---- staging: tiles of KT rows of two tensors, straight from memory to LDS by WAVES waves ------------------------------------
// A load is 1 KB: 64 / CPR rows.  Loads whose rows are a multiple of 16 apart share the permutation of their pieces, hence an address that
// differs by whole rows: a wave keeps one address per tensor for each of BASES such sets and moves them on from tile to tile.
// Only the last tile looks at every row: rows behind the last one are replaced by it (what is computed from them is masked or not
// stored; memory behind a graph's own rows is not read).  Pieces behind D are replaced by the row's first: the other operand has zeros there.
template <typename T, int DP, int KT, int WAVES>
struct Stager {
    using S = Shape<T, DP>;
    static constexpr int ROWS = 64 / S::CPR, LOADS = KT / ROWS;             // of a load; of one tensor's tile
    static constexpr bool APART = LOADS < WAVES;                            // a wave has loads of one tensor only
    static constexpr int LANES = APART ? WAVES / 2 : WAVES;                 // waves that share a tensor's loads
    static constexpr int OWN = LOADS / LANES;                               // loads of a wave and tensor: rows (u * LANES + w) * ROWS ..
    static constexpr int BASES = LANES * ROWS >= 16 ? 1 : 16 / (LANES * ROWS), APARTS = OWN / BASES;
    static_assert(LOADS % LANES == 0 && OWN % BASES == 0 && (LANES * ROWS >= 16 ? LANES * ROWS % 16 == 0 : 16 % (LANES * ROWS) == 0), "loads do not divide");
    const char *base[2][BASES];
    int64_t node[2];                                                        // bytes
    int w, tensor;                                                          // this wave's place, and its tensor if APART
    __device__ __forceinline__ int row_of(int set, int lane) const { return (set * LANES + w) * ROWS + lane / S::CPR; }
    __device__ __forceinline__ int byte_of(int r, int lane, int D) const {
        const int c = (lane % S::CPR) ^ S::swizzle(r);
        return kSplit<T> || c * (16 / S::SIZE) < D ? c * 16 : 0;
    }
    // x0, y0: element offsets of the first row
    __device__ __forceinline__ void init(const DotRows &x, const DotRows &y, int64_t x0, int64_t y0, int D, int wave) {
        const int lane = threadIdx.x & 63;
        w = wave % LANES;
        tensor = wave / LANES;
        node[0] = x.node * S::SIZE;
        node[1] = y.node * S::SIZE;
#pragma unroll
        for (int s = 0; s < BASES; ++s) {
            const int r = row_of(s, lane), byte = byte_of(r, lane, D);
            base[0][s] = reinterpret_cast<const char *>(x.p) + x0 * S::SIZE + r * node[0] + byte;
            base[1][s] = reinterpret_cast<const char *>(y.p) + y0 * S::SIZE + r * node[1] + byte;
        }
    }
    __device__ __forceinline__ void move(int64_t bx, int64_t by) {
#pragma unroll
        for (int s = 0; s < BASES; ++s) {
            base[0][s] += bx;
            base[1][s] += by;
        }
    }
    // the tile at the present place, `count` rows of it, into lds (the first tensor's, then the second's); then on to the next
    __device__ __forceinline__ void load(char *lds, int count) {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int z = 0; z < 2; ++z) {
            if (APART && z != tensor) continue;
#pragma unroll
            for (int s = 0; s < BASES; ++s)
#pragma unroll
                for (int u = 0; u < APARTS; ++u) {
                    const int set = u * BASES + s, apart = u * BASES * LANES * ROWS;        // rows from this set's base
                    const char *src = base[z][s] + apart * node[z];
                    if (count < KT) {
                        const int r = row_of(set, lane);
                        src -= max(0, r - (count - 1)) * node[z];
                    }
#pragma unroll
                    for (int k = 0; k < S::PLANES; ++k)
                        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)(src + k * S::ROW),
                                                         (__attribute__((address_space(3))) void *)(lds + ((z * S::PLANES + k) * LOADS + set * LANES + w) * 1024), 16, 0, 0);
                }
        }
        move(KT * node[0], KT * node[1]);
    }
};
// what this wave (BLOCK: every wave) has asked for is in LDS; nobody reads the other buffer any more
template <bool BLOCK>
__device__ __forceinline__ void arrived() {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if constexpr (BLOCK) __syncthreads();
    else __builtin_amdgcn_wave_barrier();
}

// ---- the mask as bits --------------------------------------------------------------------------------------------------------
// Every head of every pass reads the mask of a row; as floats that was most of the bytes of small heads.  Read once, it becomes 64 entries
// a word, along the rows and along the columns: {attended, attended with a bias other than 0}.  Hard masks need the first only; where a tile has a
// bit in the second, the kernels read the floats too.  1024 masks of 246 x 246: 76 us, 3.3 TB/s.
__global__ __launch_bounds__(256) void dot_mask_kernel(const float *bias, int64_t bias_batch, int64_t bias_row, int Nq, int Nk, ulonglong2 *row_words, ulonglong2 *col_words, int32_t *counts) {
    __shared__ uint16_t part[2][4][64];
    __shared__ int count[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int rw = (Nk + 63) / 64, cw = (Nq + 63) / 64;
    const uint32_t tj = blockIdx.x % rw, ti = blockIdx.x / rw % cw;
    const int64_t b = blockIdx.x / rw / cw;
    const int j = tj * 64 + lane;
    const float *p = bias + b * bias_batch + j;
    uint32_t seen = 0, soft = 0;
    int entries = 0;
    float v[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const int i = ti * 64 + wave * 16 + r;
        v[r] = i < Nq && j < Nk ? p[i * bias_row] : -INFINITY;
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const int i = ti * 64 + wave * 16 + r;
        const bool a = v[r] > kAttended, s = a && v[r] != 0.f;
        const uint64_t wa = __ballot(a), ws = __ballot(s);
        if (lane == 0 && i < Nq) row_words[(b * Nq + i) * rw + tj] = make_ulonglong2(wa, ws);
        entries += __popcll(wa);
        seen |= (uint32_t)a << r;
        soft |= (uint32_t)s << r;
    }
    part[0][wave][lane] = (uint16_t)seen;
    part[1][wave][lane] = (uint16_t)soft;
    if (lane == 0) count[wave] = entries;
    __syncthreads();
    if (counts && threadIdx.x == 0) counts[blockIdx.x] = (count[0] + count[1]) + (count[2] + count[3]);
    if (wave == 0 && j < Nk) {
        uint64_t w[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) w[k] = (uint64_t)part[k][0][lane] | (uint64_t)part[k][1][lane] << 16 | (uint64_t)part[k][2][lane] << 32 | (uint64_t)part[k][3][lane] << 48;
        col_words[(b * Nk + j) * cw + ti] = make_ulonglong2(w[0], w[1]);
    }
}
// flags[b] = few of the mask's entries are attended
__global__ __launch_bounds__(256) void dot_mask_count_kernel(const int32_t *counts, int per, int64_t limit, int32_t *flags) {
    __shared__ int64_t part[4];
    int64_t n = 0;
    for (int i = threadIdx.x; i < per; i += 256) n += counts[(int64_t)blockIdx.x * per + i];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o, 64);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = n;
    __syncthreads();
    if (threadIdx.x == 0) flags[blockIdx.x] = (part[0] + part[1]) + (part[2] + part[3]) <= limit;
}
// the first `n` of 64 entries
__device__ __forceinline__ uint64_t first_bits(int n) { return n >= 64 ? ~0ull : (n <= 0 ? 0 : (1ull << n) - 1); }
// z where bit `pos` of w is set, -inf elsewhere
__device__ __forceinline__ float where_bit(uint32_t w, int pos, float z) {
    const uint32_t m = (uint32_t)__builtin_amdgcn_sbfe((int)w, pos, 1);
    return __uint_as_float((__float_as_uint(z) & m) | (0xff800000u & ~m));
}

// biases of four consecutive keys of one query, -inf behind the row
__device__ __forceinline__ f32x4 bias4(const float *row, int j, int nk) {
    f32x4 v;
    if (j + 3 < nk) {
        const f32x4_u u = *reinterpret_cast<const f32x4_u *>(row + j);
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = u.v[r];
    } else {
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = j + r < nk ? row[j + r] : -INFINITY;
    }
    return v;
}
// The mask of one lane's row over a tile of KT keys.  In a lane only the bits of its own keys (16 t + 4 q .. + 3) count.
template <int MASK, int KT>
struct RowMask {
    const float *bias;                  // the row's floats and words
    const ulonglong2 *words;
    ulonglong2 next;                    // of the tile to come
    f32x4 floats[MASK == kFloats ? KT / 16 : 1];
    uint32_t lo, hi;                    // attended keys of the present tile, shifted by 4 q
    bool soft;                          // some attended entry of the wave's tile has a bias other than 0
    __device__ __forceinline__ void init(const DotArgs &a, int64_t b, int64_t i) {
        if constexpr (MASK != kNoMask) bias = a.bias + b * a.bias_batch + i * a.bias_row;
        if constexpr (MASK == kBits) words = a.row_words + b * a.row_words_batch + i * ((a.Nk + 63) / 64);
    }
    __device__ __forceinline__ void fetch(int j, int nk) {
        const int q = (threadIdx.x & 63) >> 4;
        if constexpr (MASK == kBits) next = words[j >> 6];
        if constexpr (MASK == kFloats) {
#pragma unroll
            for (int t = 0; t < KT / 16; ++t) floats[t] = bias4(bias, j + 16 * t + 4 * q, nk);
        }
    }
    // takes what was fetched for the tile at j; keys from `end` on are not attended
    __device__ __forceinline__ void take(int j, int end) {
        const int q = (threadIdx.x & 63) >> 4;
        uint64_t w = first_bits(end - j);
        soft = false;
        if constexpr (MASK == kBits) {
            w &= next.x >> (j & 63);
            soft = __ballot((next.y >> (j & 63) & w) != 0) != 0;
        }
        w >>= 4 * q;
        lo = (uint32_t)w;
        hi = (uint32_t)(w >> 32);
        if constexpr (MASK == kFloats) {
            soft = true;
#pragma unroll
            for (int t = 0; t < KT / 16; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (!(floats[t][r] > kAttended)) (t < 2 ? lo : hi) &= ~(1u << (16 * (t & 1) + r));
        }
    }
    __device__ __forceinline__ bool some(int t) const { return __ballot(((t < 2 ? lo : hi) >> (16 * (t & 1)) & 15u) != 0) != 0; }
    // raw products of tile t -> what exp2(fma(z, factor(), -base)) takes
    __device__ __forceinline__ void apply(f32x4 &z, int t, int j, int nk, float scale2) const {
        if (MASK != kNoMask && soft) {
            const f32x4 f = MASK == kFloats ? floats[t] : bias4(bias, j + 16 * t + 4 * ((threadIdx.x & 63) >> 4), nk);
#pragma unroll
            for (int r = 0; r < 4; ++r) z[r] = fmaf(z[r], scale2, f[r] * kLog2e);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) z[r] = where_bit(t < 2 ? lo : hi, 16 * (t & 1) + r, z[r]);
    }
    __device__ __forceinline__ float factor(float scale2) const { return MASK != kNoMask && soft ? 1.f : scale2; }
};

__device__ __forceinline__ float over_groups_max(float v) {
    v = fmaxf(v, __shfl_xor(v, 16, 64));
    return fmaxf(v, __shfl_xor(v, 32, 64));
}
__device__ __forceinline__ float over_groups_sum(float v) {
    v += __shfl_xor(v, 16, 64);
    return v + __shfl_xor(v, 32, 64);
}

// four consecutive elements of a result row
template <typename T>
__device__ __forceinline__ void store4(T *p, f32x4 v) {
    if constexpr (sizeof(T) == 4) *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
    else *reinterpret_cast<uint2 *>(p) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
}

// what rounding to bf16 takes from v
__device__ __forceinline__ f32x4 low_part(f32x4 v) {
    const uint32_t a = pack_bf16x2(v[0], v[1]), b = pack_bf16x2(v[2], v[3]);
    return (f32x4){v[0] - __uint_as_float(a << 16), v[1] - __uint_as_float(a & 0xffff0000u), v[2] - __uint_as_float(b << 16), v[3] - __uint_as_float(b & 0xffff0000u)};
}

// ---- forward -------------------------------------------------------------------------------------------------------------
// A wave owns NQ x 16 rows.  KEYW = false: four waves with rows of their own walk the staged tiles together.  KEYW = true: for 16 rows or
// fewer, the four waves have the same rows and walk different tiles, each staging its own, and join at the end.
// SPLIT: the block covers one range of the keys and leaves its unnormalised sums.
template <typename T, int DP, bool KEYW, int NQ, bool SPLIT, int MASK>
__global__ __launch_bounds__(256, (Shape<T, DP>::TILE > 20480 ? 1 : 2)) void dot_fwd_kernel(DotArgs a) {
    using S = Shape<T, DP>;
    constexpr int KT = KEYW ? S::KTW : S::KT, TILE = KT * S::ROW * S::PLANES, KS = KT / 16, DT = S::DT, ROWS = KEYW ? 16 : 64 * NQ, OWNERS = KEYW ? 4 : 1, STEP = OWNERS * KT;
    constexpr bool ONES = DP == 8 && std::is_same_v<T, float>;              // eight columns of the last product are free: one of them sums the probabilities
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const DotBlock blk = dot_block<MASK>(a);
    if (!blk.ok) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 15, q4 = lane >> 4;
    const int64_t b = blk.b;
    if (MASK != kNoMask && by_entries(a, b)) return;
    const int keys = graph_size(a.key_sizes, b, a.Nk), queries = graph_size(a.query_sizes, b, a.Nq);
    const int share = SPLIT ? ((keys + a.splits - 1) / a.splits + 63) / 64 * 64 : keys;           // of this graph's own keys
    const int j0 = SPLIT ? blk.split * share : 0, j1 = min(keys, j0 + share);
    char *const mine = lds + (KEYW ? wave * 4 * TILE : 0);
    auto buf = [&](int at) { return mine + at * 2 * TILE; };
    int row[NQ], qi[NQ], head[NQ];
    bool live[NQ];
    Frag<T> qf[NQ][S::FRAGS];
    RowMask<MASK, KT> mask[NQ];
#pragma unroll
    for (int u = 0; u < NQ; ++u) {
        row[u] = blk.tile * ROWS + ((KEYW ? 0 : wave) * NQ + u) * 16 + n;
        qi[u] = row[u] / a.group;
        head[u] = blk.hk * a.group + row[u] - qi[u] * a.group;
        live[u] = qi[u] < queries;
        const int64_t i = live[u] ? qi[u] : 0;
        row_frags<T, DP>(row_of<S>(a.q, b, i, head[u]), a.D, live[u], qf[u]);
        if (a.scale < 0.f) {
#pragma unroll
            for (int c = 0; c < S::FRAGS; ++c) qf[u][c] = frag_negated<T>(qf[u][c]);
        }
        mask[u].init(a, b, i);
    }
    f32x4 o[NQ][DT];
    float m[NQ], l[NQ];                 // every term of a row is formed against the same m, which follows the maximum only when that has grown by 8 (in log2): see below
#pragma unroll
    for (int u = 0; u < NQ; ++u) {
        m[u] = -INFINITY;
        l[u] = 0.f;
#pragma unroll
        for (int t = 0; t < DT; ++t) o[u][t] = (f32x4){0.f, 0.f, 0.f, 0.f};
    }
    int j = j0 + (KEYW ? wave * KT : 0), at = 0;
    Stager<T, DP, KT, KEYW ? 1 : 4> rows;
    rows.init(a.k, a.v, b * a.k.batch + blk.hk * a.k.head + j * a.k.node, b * a.v.batch + blk.hk * a.v.head + j * a.v.node, a.D, KEYW ? 0 : wave);
    auto fetch = [&](char *to, int from) {
        rows.load(to, j1 - from);
        if constexpr (KEYW) rows.move((STEP - KT) * rows.node[0], (STEP - KT) * rows.node[1]);
    };
    if (j < j1) {
        fetch(buf(0), j);
#pragma unroll
        for (int u = 0; u < NQ; ++u) mask[u].fetch(j, a.Nk);
    }
    for (; j < j1; j += STEP, at ^= 1) {
        arrived<!KEYW>();
        const char *ks = buf(at), *vs = ks + TILE;
        if (j + STEP < j1) fetch(buf(at ^ 1), j + STEP);
        const bool plain = MASK == kNoMask && j + KT <= j1;           // no entry of this tile is masked
        bool has[NQ][KS], full = true;   // tiles with an attended key, the same for the whole wave
#pragma unroll
        for (int u = 0; u < NQ; ++u) {
            if (!plain) mask[u].take(j, j1);
#pragma unroll
            for (int t = 0; t < KS; ++t) {
                has[u][t] = MASK == kNoMask || mask[u].some(t);
                full &= has[u][t];
            }
        }
        // Straight code where no tile is empty: its reads and matrix instructions run ahead of each other.
        auto walk = [&](auto skip) __attribute__((always_inline)) {
            constexpr bool SKIP = decltype(skip)::value;
            f32x4 z[NQ][KS];
            float top[NQ];
#pragma unroll
            for (int t = 0; t < KS; ++t) {
                bool any = !SKIP;
#pragma unroll
                for (int u = 0; u < NQ; ++u) {
                    any |= has[u][t];
                    z[u][t] = (f32x4){0.f, 0.f, 0.f, 0.f};
                }
                if (any) {
                    bool use[NQ];
                    f32x4 *to[NQ];
#pragma unroll
                    for (int u = 0; u < NQ; ++u) {
                        use[u] = !SKIP || has[u][t];
                        to[u] = &z[u][t];
                    }
                    mma_scores<T, DP, NQ, SKIP>(ks, 16 * t, qf, use, to);
                    if constexpr (SKIP) {
                        if constexpr (NQ == 1) settle(z[0][t]);
                        else settle(z[0][t], z[1][t]);
                    }
                }
            }
            if constexpr (!SKIP) settle(z);
#pragma unroll
            for (int u = 0; u < NQ; ++u) {
                float factor = a.scale2;
                if (!plain) {
                    factor = mask[u].factor(a.scale2);
#pragma unroll
                    for (int t = 0; t < KS; ++t)
                        if (!SKIP || has[u][t]) mask[u].apply(z[u][t], t, j, a.Nk, a.scale2);
                }
                top[u] = -INFINITY;
#pragma unroll
                for (int t = 0; t < KS; ++t)
                    if (!SKIP || has[u][t]) top[u] = fmaxf(top[u], fmaxf(fmaxf(z[u][t][0], z[u][t][1]), fmaxf(z[u][t][2], z[u][t][3])));
                top[u] *= factor;
                // The running maximum only has to keep the exponentials in range.  It is raised, and the sums shrunk, when some row's
                // maximum has passed it by 8: after the first tiles hardly ever.  Terms up to 2^8 lose nothing in fp32 or bf16.
                if (__ballot(top[u] > m[u] + 8.f)) {
                    top[u] = over_groups_max(top[u]);
                    const float now = fmaxf(m[u], top[u]), shrink = now == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m[u] - now);
                    m[u] = now;
                    l[u] *= shrink;
#pragma unroll
                    for (int t = 0; t < DT; ++t)
#pragma unroll
                        for (int r = 0; r < 4; ++r) o[u][t][r] *= shrink;
                }
                const float base = m[u] == -INFINITY ? 0.f : m[u];
#pragma unroll
                for (int t = 0; t < KS; ++t) {
                    if (!SKIP || has[u][t]) {
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            z[u][t][r] = __builtin_amdgcn_exp2f(fmaf(z[u][t][r], factor, -base));
                            if constexpr (!ONES) l[u] += z[u][t][r];
                        }
                    }
                }
            }
#pragma unroll
            for (int c = 0; c < KT / S::CHUNK; ++c) {
                constexpr int PER = S::CHUNK / 16;
                bool any = !SKIP, use[NQ];
#pragma unroll
                for (int u = 0; u < NQ; ++u) {
                    use[u] = has[u][c * PER] || has[u][c * PER + PER - 1];
                    any |= use[u];
                }
                if (!any) continue;
                ManyOf<T> pf[NQ];
#pragma unroll
                for (int u = 0; u < NQ; ++u) {
                    pf[u] = frag_scores<T>(&z[u][c * PER]);       // a tile without attended keys holds zeros
                    use[u] |= !SKIP;
                }
#pragma unroll
                for (int t = 0; t < DT; ++t) {
                    ManyOf<T> vf = frag_turned<T, DP>(vs, c * S::CHUNK, t);
                    if constexpr (ONES) {
#pragma unroll
                        for (int r = 0; r < 4; ++r) vf.p[0].v[r] = n == 8 ? 1.f : vf.p[0].v[r];
                    }
                    f32x4 *to[NQ];
#pragma unroll
                    for (int u = 0; u < NQ; ++u) to[u] = &o[u][t];
                    mma_rows<T, DP, NQ, SKIP>(vf, pf, use, to);
                }
            }
            settle_sums();
        };
        if (MASK == kNoMask || full) walk(std::false_type{});
        else walk(std::true_type{});
        if (j + STEP < j1) {
#pragma unroll
            for (int u = 0; u < NQ; ++u) mask[u].fetch(j + STEP, a.Nk);
        }
    }
    float sum[NQ];
#pragma unroll
    for (int u = 0; u < NQ; ++u) {
        if constexpr (ONES) sum[u] = __shfl(o[u][0][0], 32 + n, 64);              // row 8 of the transposed result
        else sum[u] = over_groups_sum(l[u]);
    }
    if constexpr (KEYW) {                                                            // NQ = 1: join the four waves
        __syncthreads();
        float *ml = reinterpret_cast<float *>(lds), *po = ml + 128;
        if (q4 == 0) {
            ml[wave * 16 + n] = m[0];
            ml[64 + wave * 16 + n] = sum[0];
        }
        __syncthreads();
        const float now = fmaxf(fmaxf(ml[n], ml[16 + n]), fmaxf(ml[32 + n], ml[48 + n]));
        float total = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) total += now == -INFINITY ? 0.f : ml[64 + w * 16 + n] * __builtin_amdgcn_exp2f(ml[w * 16 + n] - now);
        const float part = now == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[0] - now);
        m[0] = now;
        sum[0] = total;
#pragma unroll
        for (int t = 0; t < DT; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) po[(wave * DT + t) * 256 + r * 64 + lane] = o[0][t][r] * part;
        __syncthreads();
        if (wave != 0) return;
#pragma unroll
        for (int t = 0; t < DT; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                float v = 0.f;
#pragma unroll
                for (int w = 0; w < 4; ++w) v += po[(w * DT + t) * 256 + r * 64 + lane];
                o[0][t][r] = v;
            }
    }
#pragma unroll
    for (int u = 0; u < NQ; ++u) {
        if (qi[u] >= a.Nq) continue;
        if constexpr (SPLIT) {
            const int64_t slot = ((((b - a.b0) * a.Hkv + blk.hk) * (int64_t)a.Nq * a.group + row[u]) * a.splits + blk.split);
#pragma unroll
            for (int t = 0; t < DT; ++t)
                if (16 * t + 4 * q4 < a.D) store4<float>(a.part_o + slot * a.D + 16 * t + 4 * q4, o[u][t]);
            if (q4 == 0) {
                a.part_ml[2 * slot] = m[u];
                a.part_ml[2 * slot + 1] = sum[u];
            }
        } else {
            const float inv = !live[u] || sum[u] == 0.f ? 0.f : 1.0f / sum[u];
            const int64_t oat = ((b * a.Nq + qi[u]) * a.H + head[u]) * (int64_t)a.D;
            Elem<T> *orow = reinterpret_cast<Elem<T> *>(a.out) + oat;
#pragma unroll
            for (int t = 0; t < DT; ++t)
                if (16 * t + 4 * q4 < a.D) {
                    f32x4 v = o[u][t];
#pragma unroll
                    for (int r = 0; r < 4; ++r) v[r] = inv == 0.f ? 0.f : v[r] * inv;
                    store4<Elem<T>>(orow + 16 * t + 4 * q4, v);
                    if constexpr (S::SIZE == 2 && !kSplit<T>)
                        if (a.out_low) store4<uint16_t>(a.out_low + oat + 16 * t + 4 * q4, low_part(v));
                }
            if (a.lse && q4 == 0) a.lse[(b * a.H + head[u]) * a.Nq + qi[u]] = inv == 0.f ? INFINITY : m[u] + log2f(sum[u]);
        }
    }
}

template <typename T>
__device__ __forceinline__ void store_joined(const DotArgs &a, int64_t b, int qi, int head, int d, float top, float sum, float4 acc) {
    const bool live = qi < graph_size(a.query_sizes, b, a.Nq);
    const float inv = !live || sum == 0.f ? 0.f : 1.0f / sum;
    f32x4 v = {acc.x, acc.y, acc.z, acc.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = inv == 0.f ? 0.f : v[k] * inv;
    const int64_t at = ((b * a.Nq + qi) * a.H + head) * (int64_t)a.D + d;
    store4<T>(reinterpret_cast<T *>(a.out) + at, v);
    if constexpr (sizeof(T) == 2)
        if (a.out_low) store4<uint16_t>(a.out_low + at, low_part(v));
    if (a.lse && d == 0) a.lse[(b * a.H + head) * a.Nq + qi] = inv == 0.f ? INFINITY : top + log2f(sum);
}

// Joins the key ranges of a row where there are few of them: D / 4 lanes a row.
template <typename T>
__global__ __launch_bounds__(256) void dot_join_few_kernel(DotArgs a, int64_t rows) {
    const int lanes = a.D / 4, groups = 256 / lanes, g = threadIdx.x / lanes, d = (threadIdx.x - g * lanes) * 4;
    const int64_t rr = blockIdx.x * (int64_t)groups + g, per = (int64_t)a.Nq * a.group;
    if (g >= groups || rr >= rows) return;
    const int r = (int)(rr % per), hk = (int)(rr / per % a.Hkv), qi = r / a.group, head = hk * a.group + r % a.group;
    const int64_t b = a.b0 + rr / per / a.Hkv;
    if (by_entries(a, b)) return;
    const float *ml = a.part_ml + 2 * rr * a.splits, *po = a.part_o + rr * a.splits * a.D + d;
    float top = -INFINITY, sum = 0.f;
    for (int s = 0; s < a.splits; ++s) top = fmaxf(top, ml[2 * s]);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s = 0; s < a.splits; ++s) {
        const float w = top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml[2 * s] - top);
        sum = fmaf(ml[2 * s + 1], w, sum);
        acc = f4_fma(w, *reinterpret_cast<const float4 *>(po + (int64_t)s * a.D), acc);
    }
    store_joined<T>(a, b, qi, head, d, top, sum, acc);
}

// Joins the key ranges of a row where there are many (one block a row): the weights of the ranges first, then groups of lanes add up every so many ranges, four elements
// a lane, and their sums are added in order.
template <typename T>
__global__ __launch_bounds__(256) void dot_join_kernel(DotArgs a, int64_t rows) {
    __shared__ float weight[kSplitsMax], red[8];
    __shared__ __attribute__((aligned(16))) float part[256 * 4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int64_t rr = blockIdx.x; rr < rows; rr += gridDim.x) {
        const int64_t per = (int64_t)a.Nq * a.group;
        const int r = (int)(rr % per), hk = (int)(rr / per % a.Hkv), qi = r / a.group, head = hk * a.group + r % a.group;
        const int64_t b = a.b0 + rr / per / a.Hkv;
        if (by_entries(a, b)) continue;
        const bool has = (int)threadIdx.x < a.splits;
        const float *ml = a.part_ml + 2 * (rr * a.splits + (has ? threadIdx.x : 0));
        const float ms = has ? ml[0] : -INFINITY, ls = has ? ml[1] : 0.f;
        const float wtop = wave_max(ms);
        if (lane == 0) red[wave] = wtop;
        __syncthreads();
        const float top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
        const float w = top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ms - top);
        if (has) weight[threadIdx.x] = w;
        const float ws = group_sum<64>(ls * w);
        if (lane == 0) red[4 + wave] = ws;
        __syncthreads();
        const float sum = (red[4] + red[5]) + (red[6] + red[7]);
        const int lanes = a.D / 4, groups = 256 / lanes, g = threadIdx.x / lanes, d = (threadIdx.x - g * lanes) * 4;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        if (g < groups) {
            const float *po = a.part_o + rr * a.splits * a.D + d;
#pragma unroll 4
            for (int s = g; s < a.splits; s += groups) acc = f4_fma(weight[s], *reinterpret_cast<const float4 *>(po + (int64_t)s * a.D), acc);
            *reinterpret_cast<float4 *>(&part[4 * threadIdx.x]) = acc;
        }
        __syncthreads();
        if (g == 0) {
            for (int k = 1; k < groups; ++k) acc = f4_add(acc, *reinterpret_cast<const float4 *>(&part[4 * (threadIdx.x + k * lanes)]));
            store_joined<T>(a, b, qi, head, d, top, sum, acc);
        }
        __syncthreads();
    }
}

// ---- backward: dq and delta ------------------------------------------------------------------------------------------------
template <typename T, int DP, int NQ, int MASK>
__global__ __launch_bounds__(256, (Shape<T, DP>::TILE > 20480 ? 1 : 2)) void dot_bwd_q_kernel(DotArgs a) {
    using S = Shape<T, DP>;
    constexpr int KT = S::KT, DT = S::DT, ROWS = 64 * NQ, PER = S::CHUNK / 16;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const DotBlock blk = dot_block<MASK>(a);
    if (!blk.ok) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 15, q4 = lane >> 4;
    const int64_t b = blk.b;
    if (MASK != kNoMask && by_entries(a, b)) return;
    const int keys = graph_size(a.key_sizes, b, a.Nk), queries = graph_size(a.query_sizes, b, a.Nq);
    auto buf = [&](int at) { return lds + at * 2 * S::TILE; };
    Stager<T, DP, KT, 4> rows;
    rows.init(a.k, a.v, b * a.k.batch + blk.hk * a.k.head, b * a.v.batch + blk.hk * a.v.head, a.D, wave);
    auto fetch = [&](char *to, int from) { rows.load(to, keys - from); };
    if (keys > 0) fetch(buf(0), 0);
    int qi[NQ], head[NQ];
    float lse[NQ], delta[NQ];
    Frag<T> qf[NQ][S::FRAGS], df[NQ][S::FRAGS];
    RowMask<MASK, KT> mask[NQ];
#pragma unroll
    for (int u = 0; u < NQ; ++u) {
        const int row = blk.tile * ROWS + (wave * NQ + u) * 16 + n;
        qi[u] = row / a.group;
        head[u] = blk.hk * a.group + row - qi[u] * a.group;
        const bool live = qi[u] < queries;
        const int64_t i = live ? qi[u] : 0;
        row_frags<T, DP>(row_of<S>(a.q, b, i, head[u]), a.D, live, qf[u]);
        row_frags<T, DP>(row_of<S>(a.d_o, b, i, head[u]), a.D, live, df[u]);
        const int64_t at = (b * a.H + head[u]) * a.Nq + min(qi[u], a.Nq - 1);
        lse[u] = live ? a.lse[at] : INFINITY;
        if constexpr (kSplit<T>) {                                       // formed where dout was split
            delta[u] = live ? a.delta[at] : 0.f;
        } else {
            Frag<T> of[S::FRAGS];
            row_frags<T, DP>(row_of<S>(a.o, b, i, head[u]), a.D, live, of);
            float dot = 0.f;
#pragma unroll
            for (int c = 0; c < S::FRAGS; ++c) {
                if constexpr (S::SIZE == 4) {
#pragma unroll
                    for (int t = 0; t < S::ELEMS; ++t) dot = fmaf(df[u][c].v[t], of[c].v[t], dot);
                } else {
                    const uint32_t x[4] = {df[u][c].v.x, df[u][c].v.y, df[u][c].v.z, df[u][c].v.w}, y[4] = {of[c].v.x, of[c].v.y, of[c].v.z, of[c].v.w};
#pragma unroll
                    for (int t = 0; t < S::ELEMS / 2; ++t) {
                        dot = fmaf(__uint_as_float(x[t] << 16), __uint_as_float(y[t] << 16), dot);
                        dot = fmaf(__uint_as_float(x[t] & 0xffff0000u), __uint_as_float(y[t] & 0xffff0000u), dot);
                    }
                }
            }
            if constexpr (S::SIZE == 2) {
                if (a.out_low) {                                             // rows as those of out
                    Frag<T> low[S::FRAGS];
                    row_frags<T, DP>(row_of<S>(DotRows{a.out_low, a.o.batch, a.o.node, a.o.head}, b, i, head[u]), a.D, live, low);
#pragma unroll
                    for (int c = 0; c < S::FRAGS; ++c) {
                        const uint32_t x[4] = {df[u][c].v.x, df[u][c].v.y, df[u][c].v.z, df[u][c].v.w}, y[4] = {low[c].v.x, low[c].v.y, low[c].v.z, low[c].v.w};
#pragma unroll
                        for (int t = 0; t < S::ELEMS / 2; ++t) {
                            dot = fmaf(__uint_as_float(x[t] << 16), __uint_as_float(y[t] << 16), dot);
                            dot = fmaf(__uint_as_float(x[t] & 0xffff0000u), __uint_as_float(y[t] & 0xffff0000u), dot);
                        }
                    }
                }
            }
            delta[u] = over_groups_sum(dot);
            if (q4 == 0 && qi[u] < a.Nq) a.delta[at] = delta[u];
        }
        if (a.scale < 0.f) {
#pragma unroll
            for (int c = 0; c < S::FRAGS; ++c) qf[u][c] = frag_negated<T>(qf[u][c]);
        }
        mask[u].init(a, b, i);
    }
    if (keys > 0) {
#pragma unroll
        for (int u = 0; u < NQ; ++u) mask[u].fetch(0, a.Nk);
    }
    f32x4 acc[NQ][DT];
#pragma unroll
    for (int u = 0; u < NQ; ++u)
#pragma unroll
        for (int t = 0; t < DT; ++t) acc[u][t] = (f32x4){0.f, 0.f, 0.f, 0.f};
    for (int j = 0, at = 0; j < keys; j += KT, at ^= 1) {
        arrived<true>();
        const char *ks = buf(at), *vs = ks + S::TILE;
        if (j + KT < keys) fetch(buf(at ^ 1), j + KT);
        const bool plain = MASK == kNoMask && j + KT <= keys;
        float factor[NQ];
#pragma unroll
        for (int u = 0; u < NQ; ++u) {
            factor[u] = a.scale2;
            if (!plain) {
                mask[u].take(j, keys);
                factor[u] = mask[u].factor(a.scale2);
            }
        }
        bool has[NQ][KT / 16], full = true;
#pragma unroll
        for (int u = 0; u < NQ; ++u)
#pragma unroll
            for (int t = 0; t < KT / 16; ++t) {
                has[u][t] = MASK == kNoMask || mask[u].some(t);
                full &= has[u][t];
            }
        auto walk = [&](auto skip) __attribute__((always_inline)) {
            constexpr bool SKIP = decltype(skip)::value;
#pragma unroll
            for (int c = 0; c < KT / S::CHUNK; ++c) {
                f32x4 z[NQ][PER];
                bool use[NQ], any = !SKIP;
#pragma unroll
                for (int u = 0; u < NQ; ++u) use[u] = false;
#pragma unroll
                for (int t = 0; t < PER; ++t) {
                    const int r0 = c * S::CHUNK + 16 * t;
                    f32x4 dp[NQ];
                    bool here = !SKIP;
#pragma unroll
                    for (int u = 0; u < NQ; ++u) {
                        z[u][t] = dp[u] = (f32x4){0.f, 0.f, 0.f, 0.f};
                        use[u] |= has[u][r0 / 16];
                        here |= has[u][r0 / 16];
                    }
                    any |= here;
                    if (!here) continue;
                    bool some[NQ];
                    f32x4 *zt[NQ], *dt[NQ];
#pragma unroll
                    for (int u = 0; u < NQ; ++u) {
                        some[u] = !SKIP || has[u][r0 / 16];
                        zt[u] = &z[u][t];
                        dt[u] = &dp[u];
                    }
                    mma_scores<T, DP, NQ, SKIP>(ks, r0, qf, some, zt);
                    mma_scores<T, DP, NQ, SKIP>(vs, r0, df, some, dt);
                    if constexpr (NQ == 1) settle(z[0][t], dp[0]);
                    else settle(z[0][t], dp[0], z[1][t], dp[1]);
#pragma unroll
                    for (int u = 0; u < NQ; ++u)
                        if (!SKIP || has[u][r0 / 16]) {
                            if (!plain) mask[u].apply(z[u][t], r0 / 16, j, a.Nk, a.scale2);
#pragma unroll
                            for (int r = 0; r < 4; ++r) z[u][t][r] = __builtin_amdgcn_exp2f(fmaf(z[u][t][r], factor[u], -lse[u])) * (dp[u][r] - delta[u]);
                        }
                }
                if (!any) continue;
                ManyOf<T> zf[NQ];
#pragma unroll
                for (int u = 0; u < NQ; ++u) {
                    zf[u] = frag_scores<T>(z[u]);
                    use[u] |= !SKIP;
                }
#pragma unroll
                for (int t = 0; t < DT; ++t) {
                    f32x4 *to[NQ];
#pragma unroll
                    for (int u = 0; u < NQ; ++u) to[u] = &acc[u][t];
                    mma_rows<T, DP, NQ, SKIP>(frag_turned<T, DP>(ks, c * S::CHUNK, t), zf, use, to);
                }
            }
            settle_sums();
        };
        if (MASK == kNoMask || full) walk(std::false_type{});
        else walk(std::true_type{});
        if (j + KT < keys) {
#pragma unroll
            for (int u = 0; u < NQ; ++u) mask[u].fetch(j + KT, a.Nk);
        }
    }
#pragma unroll
    for (int u = 0; u < NQ; ++u) {
        if (qi[u] >= a.Nq) continue;
        Elem<T> *row = reinterpret_cast<Elem<T> *>(a.dq) + ((b * a.Nq + qi[u]) * a.H + head[u]) * (int64_t)a.D;
#pragma unroll
        for (int t = 0; t < DT; ++t)
            if (16 * t + 4 * q4 < a.D) {
                f32x4 v = acc[u][t];
#pragma unroll
                for (int r = 0; r < 4; ++r) v[r] *= a.scale;
                store4<Elem<T>>(row + 16 * t + 4 * q4, v);
            }
    }
}

// ---- backward: dk and dv -----------------------------------------------------------------------------------------------------
// A wave owns NK x 16 keys (one per lane of a row of 16) and walks the queries of each sharing head in turn.  Rows behind the last
// one come with lse = inf: their probabilities are zero.
template <typename T, int DP, int NK, int MASK>
__global__ __launch_bounds__(256, (Shape<T, DP>::ROW == 512 || Shape<T, DP>::TILE > 20480 ? 1 : 2)) void dot_bwd_kv_kernel(DotArgs a) {
    using S = Shape<T, DP>;
    constexpr int QT = S::KT, DT = S::DT, KEYS = 64 * NK, PER = S::CHUNK / 16;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    __shared__ __attribute__((aligned(16))) float lses[2][QT], deltas[2][QT];
    const DotBlock blk = dot_block<MASK>(a);
    if (!blk.ok) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 15, q4 = lane >> 4;
    const int64_t b = blk.b;
    if (MASK != kNoMask && by_entries(a, b)) return;
    const int keys = graph_size(a.key_sizes, b, a.Nk), queries = graph_size(a.query_sizes, b, a.Nq);
    auto buf = [&](int at) { return lds + at * 2 * S::TILE; };
    const int head0 = blk.hk * a.group;
    Stager<T, DP, QT, 4> rows;
    rows.init(a.q, a.d_o, b * a.q.batch + head0 * a.q.head, b * a.d_o.batch + head0 * a.d_o.head, a.D, wave);
    const int tiles = (queries + QT - 1) / QT;
    // of the tile that is fetched next: its head in the group and its first query
    int next_head = 0, next_i = 0;
    auto fetch = [&](int to) {
        rows.load(buf(to), queries - next_i);
        if (threadIdx.x < QT) {
            const int i = next_i + (int)threadIdx.x;
            const int64_t at = (b * a.H + head0 + next_head) * a.Nq + min(i, queries - 1);
            lses[to][threadIdx.x] = i < queries ? a.lse[at] : INFINITY;
            deltas[to][threadIdx.x] = a.delta[at];
        }
        next_i += QT;
        if (next_i >= queries) {                      // on to the next head: back to its first row
            rows.move(a.q.head * S::SIZE - (int64_t)tiles * QT * rows.node[0], a.d_o.head * S::SIZE - (int64_t)tiles * QT * rows.node[1]);
            next_i = 0;
            ++next_head;
        }
    };
    if (queries > 0) fetch(0);
    int key[NK], col[NK];
    const ulonglong2 *words[NK];          // the mask of this lane's key over the queries
    ulonglong2 next[NK];
    Frag<T> kf[NK][S::FRAGS], vf[NK][S::FRAGS];
    f32x4 dk[NK][DT], dv[NK][DT];
#pragma unroll
    for (int u = 0; u < NK; ++u) {
        key[u] = blk.tile * KEYS + (wave * NK + u) * 16 + n;
        const bool live = key[u] < keys;
        col[u] = live ? key[u] : 0;
        row_frags<T, DP>(row_of<S>(a.k, b, col[u], blk.hk), a.D, live, kf[u]);
        row_frags<T, DP>(row_of<S>(a.v, b, col[u], blk.hk), a.D, live, vf[u]);
        if (a.scale < 0.f) {
#pragma unroll
            for (int c = 0; c < S::FRAGS; ++c) kf[u][c] = frag_negated<T>(kf[u][c]);
        }
        if constexpr (MASK == kBits) {
            words[u] = a.col_words + b * a.col_words_batch + (int64_t)col[u] * ((a.Nq + 63) / 64);
            if (queries > 0) next[u] = words[u][0];
        }
#pragma unroll
        for (int t = 0; t < DT; ++t) dk[u][t] = dv[u][t] = (f32x4){0.f, 0.f, 0.f, 0.f};
    }
    for (int it = 0, i0 = 0, at = 0; it < tiles * a.group; ++it, at ^= 1) {
        arrived<true>();
        const char *qs = buf(at), *ds = qs + S::TILE;
        if (it + 1 < tiles * a.group) fetch(at ^ 1);
        uint32_t lo[NK], hi[NK];
        bool soft[NK];
        const int here0 = i0;                         // the tile's first query
        i0 = i0 + QT >= queries ? 0 : i0 + QT;
#pragma unroll
        for (int u = 0; u < NK; ++u) {
            soft[u] = false;
            if constexpr (MASK == kBits) {
                const uint64_t w = next[u].x >> (here0 & 63);
                soft[u] = __ballot(next[u].y >> (here0 & 63) != 0) != 0;
                lo[u] = (uint32_t)(w >> (4 * q4));
                hi[u] = (uint32_t)(w >> (4 * q4) >> 32);
                next[u] = words[u][i0 >> 6];
            }
        }
        bool has[NK][QT / 16], full = true;
#pragma unroll
        for (int u = 0; u < NK; ++u)
#pragma unroll
            for (int t = 0; t < QT / 16; ++t) {
                has[u][t] = MASK != kBits || __ballot(((t < 2 ? lo[u] : hi[u]) >> (16 * (t & 1)) & 15u) != 0) != 0;
                full &= has[u][t];
            }
        auto walk = [&](auto skip) __attribute__((always_inline)) {
            constexpr bool SKIP = decltype(skip)::value;
#pragma unroll
            for (int c = 0; c < QT / S::CHUNK; ++c) {
                f32x4 p[NK][PER], z[NK][PER];
                bool use[NK], any = !SKIP;
#pragma unroll
                for (int u = 0; u < NK; ++u) use[u] = false;
#pragma unroll
                for (int t = 0; t < PER; ++t) {
                    const int s0 = c * S::CHUNK + 16 * t;
                    f32x4 dp[NK], bias[NK];
                    bool some[NK], here = !SKIP;
#pragma unroll
                    for (int u = 0; u < NK; ++u) {
                        z[u][t] = dp[u] = p[u][t] = (f32x4){0.f, 0.f, 0.f, 0.f};
                        some[u] = has[u][s0 / 16];
                        if constexpr (MASK == kBits) {
                            if (soft[u]) {
#pragma unroll
                                for (int r = 0; r < 4; ++r) bias[u][r] = a.bias[b * a.bias_batch + (int64_t)min(here0 + s0 + 4 * q4 + r, queries - 1) * a.bias_row + col[u]];
                            }
                        }
                        use[u] |= some[u];
                        here |= some[u];
                    }
                    any |= here;
                    if (!here) continue;
                    f32x4 *zt[NK], *dt[NK];
#pragma unroll
                    for (int u = 0; u < NK; ++u) {
                        some[u] |= !SKIP;
                        zt[u] = &z[u][t];
                        dt[u] = &dp[u];
                    }
                    mma_scores<T, DP, NK, SKIP>(qs, s0, kf, some, zt);
                    mma_scores<T, DP, NK, SKIP>(ds, s0, vf, some, dt);
                    if constexpr (NK == 1) settle(z[0][t], dp[0]);
                    else settle(z[0][t], dp[0], z[1][t], dp[1]);
                    const f32x4 lse = *reinterpret_cast<const f32x4 *>(&lses[at][s0 + 4 * q4]), delta = *reinterpret_cast<const f32x4 *>(&deltas[at][s0 + 4 * q4]);
#pragma unroll
                    for (int u = 0; u < NK; ++u)
                        if (!SKIP || some[u]) {
                            float factor = a.scale2;
                            if constexpr (MASK == kBits) {
                                if (soft[u]) {
                                    factor = 1.f;
#pragma unroll
                                    for (int r = 0; r < 4; ++r) z[u][t][r] = fmaf(z[u][t][r], a.scale2, bias[u][r] * kLog2e);
                                }
#pragma unroll
                                for (int r = 0; r < 4; ++r) z[u][t][r] = where_bit(s0 < 32 ? lo[u] : hi[u], (s0 & 31) + r, z[u][t][r]);
                            }
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                p[u][t][r] = __builtin_amdgcn_exp2f(fmaf(z[u][t][r], factor, -lse[r]));
                                z[u][t][r] = p[u][t][r] * (dp[u][r] - delta[r]);
                            }
                        }
                }
                if (!any) continue;
                ManyOf<T> pf[NK], zf[NK];
#pragma unroll
                for (int u = 0; u < NK; ++u) {
                    pf[u] = frag_scores<T>(p[u]);
                    zf[u] = frag_scores<T>(z[u]);
                    use[u] |= !SKIP;
                }
#pragma unroll
                for (int t = 0; t < DT; ++t) {
                    f32x4 *vt[NK], *kt[NK];
#pragma unroll
                    for (int u = 0; u < NK; ++u) {
                        vt[u] = &dv[u][t];
                        kt[u] = &dk[u][t];
                    }
                    mma_rows<T, DP, NK, SKIP>(frag_turned<T, DP>(ds, c * S::CHUNK, t), pf, use, vt);
                    mma_rows<T, DP, NK, SKIP>(frag_turned<T, DP>(qs, c * S::CHUNK, t), zf, use, kt);
                }
            }
            settle_sums();
        };
        if (MASK == kNoMask || full) walk(std::false_type{});
        else walk(std::true_type{});
    }
#pragma unroll
    for (int u = 0; u < NK; ++u) {
        if (key[u] >= a.Nk) continue;
        const float keep = key[u] < keys ? 1.f : 0.f;                  // a key behind the graph's own has been walked as a row of zeros
        const int64_t at = ((b * a.Nk + key[u]) * a.Hkv + blk.hk) * (int64_t)a.D;
#pragma unroll
        for (int t = 0; t < DT; ++t)
            if (16 * t + 4 * q4 < a.D) {
                f32x4 x = dk[u][t], y = dv[u][t];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    x[r] = keep == 0.f ? 0.f : x[r] * a.scale;
                    y[r] = keep == 0.f ? 0.f : y[r];
                }
                store4<Elem<T>>(reinterpret_cast<Elem<T> *>(a.dk) + at + 16 * t + 4 * q4, x);
                store4<Elem<T>>(reinterpret_cast<Elem<T> *>(a.dv) + at + 16 * t + 4 * q4, y);
            }
    }
}

// ---- masks with few entries ------------------------------------------------------------------------------------------------------
// A 16 x 16 tile with one attended entry costs what a full one costs.  Where a mask has few entries they are walked one by one: a group of lanes
// has a row (a query, or a key for dk and dv), DL lanes eight elements each of its width, WS of these sets different words of the mask; their results
// are added in a fixed order.  Probabilities stay in fp32 for bf16, too.  Bound by the latency of scattered rows; Cora's mask (2708 nodes, 0.15 %), 8 heads of 8,
// forward / dq / dk, dv: 13 / 11 / 12 us, in tiles 44 / 95 / 117.
template <int DP> struct Entries {
    static constexpr int DL = DP / 8, WS = DL <= 2 ? 4 : (DL <= 8 ? 2 : 1), LANES = DL * WS, ROWS = 256 / LANES;
};
template <typename T>
__device__ __forceinline__ void load8(const T *p, int e, int D, float (&f)[8]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int k = 0; k < 8; k += 4) {
            const float4 u = e + k < D ? *reinterpret_cast<const float4 *>(p + e + k) : make_float4(0.f, 0.f, 0.f, 0.f);
            f[k] = u.x; f[k + 1] = u.y; f[k + 2] = u.z; f[k + 3] = u.w;
        }
    } else {
        const uint4 u = e < D ? *reinterpret_cast<const uint4 *>(p + e) : make_uint4(0, 0, 0, 0);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            f[2 * k] = __uint_as_float(w[k] << 16);
            f[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
        }
    }
}
template <typename T>
__device__ __forceinline__ void store8(T *p, int e, int D, const float (&f)[8]) {
#pragma unroll
    for (int k = 0; k < 8; k += 4)
        if (e + k < D) store4<T>(p + e + k, (f32x4){f[k], f[k + 1], f[k + 2], f[k + 3]});
}
template <typename T>
__device__ __forceinline__ const T *entry_row(const DotRows &x, int64_t b, int64_t i, int head) {
    return reinterpret_cast<const T *>(x.p) + b * x.batch + i * x.node + head * x.head;
}
template <int DL>
__device__ __forceinline__ float dot8(const float (&x)[8], const float (&y)[8]) {
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) s = fmaf(x[k], y[k], s);
    return group_sum<DL>(s);
}
// each(entry, whether its bias is other than 0) for the attended ones among the first n, every WS-th word from `first` on.
// The entry's bit of the second word is taken with the lowest bit of `bits`, not with a shift: hipcc (ROCm 7.2) put the amount of that 64-bit shift into
// the last register of the wave, from where the hardware reads it wrong in all but a SIMD's first wave (tests/test_shift_amounts.py).
template <int WS, typename F>
__device__ __forceinline__ void walk_entries(const ulonglong2 *words, int n, int first, F each) {
    const int count = (n + 63) / 64;
    for (int w0 = first; w0 < count; w0 += 4 * WS) {
        ulonglong2 x[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) x[u] = w0 + u * WS < count ? words[w0 + u * WS] : make_ulonglong2(0, 0);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int base = (w0 + u * WS) * 64;
            for (uint64_t bits = x[u].x & first_bits(n - base); bits; bits &= bits - 1)
                each(base + __builtin_ctzll(bits), (x[u].y & bits & -bits) != 0);
        }
    }
}
template <int DL, int LANES>
__device__ __forceinline__ void over_sets(float (&f)[8]) {
#pragma unroll
    for (int o = DL; o < LANES; o <<= 1)
#pragma unroll
        for (int k = 0; k < 8; ++k) f[k] += __shfl_xor(f[k], o, 64);
}

// The heads of a query lie next to each other, among the lanes as in memory.
template <typename T, int DP>
__global__ __launch_bounds__(256) void dot_entries_fwd_kernel(DotArgs a, int64_t rows) {
    using E = Entries<DP>;
    const int e = threadIdx.x % E::DL * 8, set = threadIdx.x / E::DL % E::WS;
    for (int64_t rr = blockIdx.x * (int64_t)E::ROWS + threadIdx.x / E::LANES; rr < rows; rr += (int64_t)gridDim.x * E::ROWS) {
        const int64_t bi = rr / a.H, b = bi / a.Nq;
        if (!by_entries(a, b)) continue;
        const int head = (int)(rr - bi * a.H), hk = head / a.group, i = (int)(bi - b * a.Nq);
        const bool live = i < graph_size(a.query_sizes, b, a.Nq);
        float q[8], o[8] = {0.f}, m = -INFINITY, l = 0.f;
        load8<T>(entry_row<T>(a.q, b, i, head), e, live ? a.D : 0, q);
        walk_entries<E::WS>(a.row_words + b * a.row_words_batch + (int64_t)i * ((a.Nk + 63) / 64), live ? graph_size(a.key_sizes, b, a.Nk) : 0, set, [&](int j, bool soft) {
            float k[8], v[8];
            load8<T>(entry_row<T>(a.k, b, j, hk), e, a.D, k);
            load8<T>(entry_row<T>(a.v, b, j, hk), e, a.D, v);
            float z = dot8<E::DL>(q, k) * (a.scale * kLog2e);
            if (soft) z = fmaf(a.bias[b * a.bias_batch + i * a.bias_row + j], kLog2e, z);
            const float top = fmaxf(m, z), base = top == -INFINITY ? 0.f : top, shrink = __builtin_amdgcn_exp2f(m - base), p = __builtin_amdgcn_exp2f(z - base);
            m = top;
            l = fmaf(l, shrink, p);
#pragma unroll
            for (int r = 0; r < 8; ++r) o[r] = fmaf(o[r], shrink, p * v[r]);
        });
        float top = m;
#pragma unroll
        for (int w = E::DL; w < E::LANES; w <<= 1) top = fmaxf(top, __shfl_xor(top, w, 64));
        const float part = __builtin_amdgcn_exp2f(m - (top == -INFINITY ? 0.f : top));
        l *= part;
#pragma unroll
        for (int w = E::DL; w < E::LANES; w <<= 1) l += __shfl_xor(l, w, 64);
#pragma unroll
        for (int r = 0; r < 8; ++r) o[r] *= part;
        over_sets<E::DL, E::LANES>(o);
        if (set != 0) continue;
        const float inv = l == 0.f ? 0.f : 1.0f / l;
#pragma unroll
        for (int r = 0; r < 8; ++r) o[r] = inv == 0.f ? 0.f : o[r] * inv;
        store8<T>(reinterpret_cast<T *>(a.out) + rr * a.D, e, a.D, o);
        if constexpr (sizeof(T) == 2)
            if (a.out_low) {
#pragma unroll
                for (int r = 0; r < 8; r += 4)
                    if (e < a.D) store4<uint16_t>(a.out_low + rr * a.D + e + r, low_part((f32x4){o[r], o[r + 1], o[r + 2], o[r + 3]}));
            }
        if (a.lse && e == 0) a.lse[(b * a.H + head) * a.Nq + i] = inv == 0.f ? INFINITY : top + log2f(l);
    }
}

template <typename T, int DP>
__global__ __launch_bounds__(256) void dot_entries_q_kernel(DotArgs a, int64_t rows) {
    using E = Entries<DP>;
    const int e = threadIdx.x % E::DL * 8, set = threadIdx.x / E::DL % E::WS;
    for (int64_t rr = blockIdx.x * (int64_t)E::ROWS + threadIdx.x / E::LANES; rr < rows; rr += (int64_t)gridDim.x * E::ROWS) {
        const int64_t bi = rr / a.H, b = bi / a.Nq;
        if (!by_entries(a, b)) continue;
        const int head = (int)(rr - bi * a.H), hk = head / a.group, i = (int)(bi - b * a.Nq);
        const bool live = i < graph_size(a.query_sizes, b, a.Nq);
        const int64_t at = (b * a.H + head) * a.Nq + i;
        float q[8], d[8], o[8], dq[8] = {0.f};
        load8<T>(entry_row<T>(a.q, b, i, head), e, live ? a.D : 0, q);
        load8<T>(entry_row<T>(a.d_o, b, i, head), e, live ? a.D : 0, d);
        load8<T>(entry_row<T>(a.o, b, i, head), e, live ? a.D : 0, o);
        if constexpr (sizeof(T) == 2)
            if (a.out_low) {
                float low[8];
                load8<T>(a.out_low + rr * a.D, e, live ? a.D : 0, low);
#pragma unroll
                for (int r = 0; r < 8; ++r) o[r] += low[r];
            }
        const float delta = dot8<E::DL>(d, o), lse = a.lse[at];
        walk_entries<E::WS>(a.row_words + b * a.row_words_batch + (int64_t)i * ((a.Nk + 63) / 64), live ? graph_size(a.key_sizes, b, a.Nk) : 0, set, [&](int j, bool soft) {
            float k[8], v[8];
            load8<T>(entry_row<T>(a.k, b, j, hk), e, a.D, k);
            load8<T>(entry_row<T>(a.v, b, j, hk), e, a.D, v);
            float z = dot8<E::DL>(q, k) * (a.scale * kLog2e);
            if (soft) z = fmaf(a.bias[b * a.bias_batch + i * a.bias_row + j], kLog2e, z);
            const float dz = __builtin_amdgcn_exp2f(z - lse) * (dot8<E::DL>(d, v) - delta);
#pragma unroll
            for (int r = 0; r < 8; ++r) dq[r] = fmaf(dz, k[r], dq[r]);
        });
        over_sets<E::DL, E::LANES>(dq);
        if (set != 0) continue;
#pragma unroll
        for (int r = 0; r < 8; ++r) dq[r] *= a.scale;
        store8<T>(reinterpret_cast<T *>(a.dq) + rr * a.D, e, a.D, dq);
        if (e == 0) a.delta[at] = delta;
    }
}

template <typename T, int DP>
__global__ __launch_bounds__(256) void dot_entries_kv_kernel(DotArgs a, int64_t rows) {
    using E = Entries<DP>;
    const int e = threadIdx.x % E::DL * 8, set = threadIdx.x / E::DL % E::WS;
    for (int64_t rr = blockIdx.x * (int64_t)E::ROWS + threadIdx.x / E::LANES; rr < rows; rr += (int64_t)gridDim.x * E::ROWS) {
        const int64_t bj = rr / a.Hkv, b = bj / a.Nk;
        if (!by_entries(a, b)) continue;
        const int hk = (int)(rr - bj * a.Hkv), j = (int)(bj - b * a.Nk);
        const bool live = j < graph_size(a.key_sizes, b, a.Nk);
        float k[8], v[8], dk[8] = {0.f}, dv[8] = {0.f};
        load8<T>(entry_row<T>(a.k, b, j, hk), e, live ? a.D : 0, k);
        load8<T>(entry_row<T>(a.v, b, j, hk), e, live ? a.D : 0, v);
        walk_entries<E::WS>(a.col_words + b * a.col_words_batch + (int64_t)j * ((a.Nq + 63) / 64), live ? graph_size(a.query_sizes, b, a.Nq) : 0, set, [&](int i, bool soft) {
            const float bias = soft ? a.bias[b * a.bias_batch + i * a.bias_row + j] * kLog2e : 0.f;
            for (int g = 0; g < a.group; ++g) {
                const int head = hk * a.group + g;
                const int64_t at = (b * a.H + head) * a.Nq + i;
                float q[8], d[8];
                load8<T>(entry_row<T>(a.q, b, i, head), e, a.D, q);
                load8<T>(entry_row<T>(a.d_o, b, i, head), e, a.D, d);
                const float p = __builtin_amdgcn_exp2f(fmaf(dot8<E::DL>(q, k), a.scale * kLog2e, bias) - a.lse[at]), dz = p * (dot8<E::DL>(d, v) - a.delta[at]);
#pragma unroll
                for (int r = 0; r < 8; ++r) {
                    dk[r] = fmaf(dz, q[r], dk[r]);
                    dv[r] = fmaf(p, d[r], dv[r]);
                }
            }
        });
        over_sets<E::DL, E::LANES>(dk);
        over_sets<E::DL, E::LANES>(dv);
        if (set != 0) continue;
#pragma unroll
        for (int r = 0; r < 8; ++r) dk[r] *= a.scale;
        store8<T>(reinterpret_cast<T *>(a.dk) + rr * a.D, e, a.D, dk);
        store8<T>(reinterpret_cast<T *>(a.dv) + rr * a.D, e, a.D, dv);
    }
}

// ---- rows of three parts -------------------------------------------------------------------------------------------------------
struct SplitArgs {
    DotRows x[3];                       // fp32 rows of up to three tensors, one to a blockIdx.y
    void *out[3];                       // their [B, N, heads] rows of 3 x DP bf16
    int64_t rows[3];                    // B * N * heads
    int N[3], heads[3], D;
    DotRows o;                          // DELTA: the forward's result, rows as x[0]
    float *delta;                       // [B, heads, N]: <x, o>
};

// DP / 8 lanes a row, eight elements a lane: 4 bytes read and 6 written per element (5.2 TB/s for 26 M elements)
template <int DP, bool DELTA>
__global__ __launch_bounds__(256) void dot_split_kernel(SplitArgs a) {
    constexpr int LANES = DP / 8;
    const int lane = threadIdx.x % LANES, e = lane * 8, z = blockIdx.y, heads = a.heads[z], N = a.N[z];
    const DotRows x = a.x[z];
    // whole lane groups leave the loop together
    for (int64_t rr = blockIdx.x * (int64_t)(256 / LANES) + threadIdx.x / LANES; rr < a.rows[z]; rr += (int64_t)gridDim.x * (256 / LANES)) {
        const int64_t bi = rr / heads, b = bi / N;
        const int h = (int)(rr - bi * heads), i = (int)(bi - b * N);
        auto load = [&](const DotRows &r, float (&f)[8]) {
            const float *p = reinterpret_cast<const float *>(r.p) + b * r.batch + i * r.node + h * r.head + e;
#pragma unroll
            for (int k = 0; k < 8; k += 4) {
                const float4 u = e + k < a.D ? *reinterpret_cast<const float4 *>(p + k) : make_float4(0.f, 0.f, 0.f, 0.f);      // D is a multiple of 4
                f[k] = u.x; f[k + 1] = u.y; f[k + 2] = u.z; f[k + 3] = u.w;
            }
        };
        float v[8], o[8];
        load(x, v);
        if constexpr (DELTA) load(a.o, o);
        uint32_t w[3][4];
#pragma unroll
        for (int k = 0; k < 4; ++k) split3_pack(v[2 * k], v[2 * k + 1], w[0][k], w[1][k], w[2][k]);
        uint16_t *out = reinterpret_cast<uint16_t *>(a.out[z]) + rr * (3 * DP) + e;
#pragma unroll
        for (int k = 0; k < 3; ++k) *reinterpret_cast<uint4 *>(out + k * DP) = make_uint4(w[k][0], w[k][1], w[k][2], w[k][3]);
        if constexpr (DELTA) {
            float dot = 0.f;
#pragma unroll
            for (int k = 0; k < 8; ++k) dot = fmaf(v[k], o[k], dot);
            dot = group_sum<LANES>(dot);
            if (lane == 0) a.delta[(b * heads + h) * N + i] = dot;
        }
    }
}

// ---- host --------------------------------------------------------------------------------------------------------------------
static int dot_check(const char *what, int64_t B, int32_t Nq, int32_t Nk, int32_t H, int32_t Hkv, int32_t D, int32_t dtype) {
    GATMI_REQUIRE(B >= 0 && Nq >= 0 && Nk >= 0, GATMI_EINVAL, "%s: B = %lld, Nq = %d, Nk = %d", what, (long long)B, Nq, Nk);
    GATMI_REQUIRE(H >= 1 && Hkv >= 1 && H % Hkv == 0, GATMI_EINVAL, "%s: %d query heads on %d key/value heads", what, H, Hkv);
    GATMI_REQUIRE(dtype == GATMI_DTYPE_F32 || dtype == GATMI_DTYPE_BF16, GATMI_EINVAL, "%s: dtype %d", what, dtype);
    const int unit = dtype == GATMI_DTYPE_F32 ? 4 : 8;
    GATMI_REQUIRE(D >= unit && D % unit == 0 && D <= 128, GATMI_EUNSUPPORTED, "%s: head width %d (a multiple of %d up to 128)", what, D, unit);
    GATMI_REQUIRE((int64_t)Nq * H < (1ll << 31) - 4096 && (int64_t)Nk < (1ll << 31) - 4096, GATMI_ERANGE, "%s: %d rows of %d heads do not fit 31 bits", what, Nq, H);
    return GATMI_OK;
}

static int dot_rows(const char *what, const char *name, DotRows *r, const void *p, const int64_t *stride, int32_t dtype) {
    GATMI_REQUIRE(p && stride, GATMI_EINVAL, "%s: %s is null", what, name);
    const int unit = dtype == GATMI_DTYPE_F32 ? 4 : 8;
    GATMI_REQUIRE(aligned16(p) && stride[0] % unit == 0 && stride[1] % unit == 0 && stride[2] % unit == 0, GATMI_EALIGN,
                  "%s: %s rows are not 16-byte aligned (strides %lld, %lld, %lld elements)", what, name, (long long)stride[0], (long long)stride[1], (long long)stride[2]);
    *r = DotRows{p, stride[0], stride[1], stride[2]};
    return GATMI_OK;
}

constexpr int64_t kDotBlocks = 1 << 22;      // blocks of one launch

// Rows per block: the four waves share 16 rows and walk different keys, or have 16 or 32 rows each.
static int dot_rows_per_block(int64_t rows, int nq) { return rows <= 16 ? 16 : (rows <= 64 ? 64 : 64 * nq); }

// Key ranges of a forward launch: as many blocks as are resident at once (two to a compute unit), ranges of 512 keys or more.
static int dot_splits(int64_t B, int64_t rows, int32_t Hkv, int32_t Nk) {
    const int per = dot_rows_per_block(rows, 2);
    const int64_t blocks = B * Hkv * ((rows + per - 1) / per);
    if (blocks >= 384 || Nk < 1024) return 1;
    return (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(kSplitsMax, Nk / 512), (512 + blocks / 2) / blocks));
}

// graphs that one launch takes
static int64_t dot_graphs(const DotArgs &a) {
    const int64_t per = (int64_t)a.tiles * a.splits * a.Hkv;
    return std::max<int64_t>(1, kDotBlocks / per);
}

template <typename K>
static int dot_launch(const char *what, K kernel, const DotArgs &a, size_t lds, hipStream_t st) {
    if (lds > 48 * 1024) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) return fail(GATMI_EHIP, "%s: %s", what, hipGetErrorString(e));
    }
    const int64_t inner = a.bias ? a.Hkv : (int64_t)a.tiles * a.splits, groups = (int64_t)a.B * a.Hkv * a.tiles * a.splits / inner;
    const int64_t blocks = 8 * (groups / 8 * inner + (groups % 8 * inner + 7) / 8);
    GATMI_REQUIRE(blocks <= 2 * kDotBlocks, GATMI_ERANGE, "%s: %lld blocks for one graph", what, (long long)blocks);
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(256), lds, st, a);
    return GATMI_OK;
}

}  // namespace gatmi

using namespace gatmi;

// Masks of fewer entries than this are never walked entry by entry.  Finding out (the count, launches that return at once) costs 8 to 20 us a forward and
// backward, 50 and 90 of 1024 masks.  Never - found out, in us, of masks that end in tiles (10 %): fp32 64 graphs of 128 nodes, 4 heads of 8: 33 - 46, 16 of 246, 4 of 64:
// 92 - 103, 50 of 246, 6 of 64: 239 - 259, one of 400, 8 of 8: 69 - 78, 1024 of 246, 8 of 8: 1401 - 1451; bf16 50 of 246: 105 - 122, 1024 of 246: 863 - 950.
// Of masks that are walked (1 %): fp32 34 - 46, 94 - 53, 245 - 128, 72 - 45, 1382 - 560; bf16 114 - 92, 919 - 808.  Graphs of so few nodes come as
// connectivity thresholded to 10 % and more, so they keep the tiles without asking; a batch of very sparse ones pays for it.
constexpr int64_t kEntriesMask = 512 * 512;
static bool dot_maybe_entries(int64_t Nq, int64_t Nk) { return Nq * Nk >= kEntriesMask; }
// "Few" is one entry of 16 for fp32, of 64 for bf16.  Forward and backward in us, 16 graphs of 1024 nodes, 4 heads, tiles - entries:
//   fp32, 8 wide: 0.2 % 168 - 39, 1.6 % 213 - 70, 6.4 % 211 - 154;  64 wide: 392 - 90, 438 - 189, 433 - 440;  128 wide: 1101 - 137, 1112 - 353, 1080 - 863
//   bf16, 64 wide: 0.2 % 175 - 87, 1.6 % 179 - 176, 3.2 % 165 - 254;  128 wide: 290 - 105, 306 - 236, 288 - 372
// Entries are counted over the whole mask.  A row's are walked one after the other, so long rows take longer than tiles do: 2708 nodes with 5 entries a
// row, 8 heads of 8, fp32: 281 - 57; as many with a power law (longest row 514): 326 - 286; with one full row and column: 319 - 993.
static int64_t dot_entries_share(int32_t dtype) { return dtype == GATMI_DTYPE_F32 ? 16 : 64; }

// floats that hold the words of `graphs` masks (rows, then columns), with the counts and flags of large ones
static size_t dot_mask_floats(int64_t graphs, int64_t Nq, int64_t Nk) {
    const size_t rw = (Nk + 63) / 64, cw = (Nq + 63) / 64;
    return (size_t)graphs * (4 * (Nq * rw + Nk * cw) + (dot_maybe_entries(Nq, Nk) ? rw * cw + 1 : 0));
}

// builds the words of the mask of one call (graphs: B, or 1 where all share it) and points `a` at them
static int dot_mask_words(const char *what, DotArgs *a, int64_t graphs, float *words, int32_t dtype, bool build, hipStream_t st) {
    GATMI_REQUIRE(words, GATMI_EINVAL, "%s: mask words are null", what);
    GATMI_REQUIRE_ALIGNED(words);
    const int64_t rw = (a->Nk + 63) / 64, cw = (a->Nq + 63) / 64, per = rw * cw;
    ulonglong2 *rows = reinterpret_cast<ulonglong2 *>(words), *cols = rows + graphs * a->Nq * rw;
    int32_t *counts = dot_maybe_entries(a->Nq, a->Nk) ? reinterpret_cast<int32_t *>(cols + graphs * a->Nk * cw) : nullptr, *flags = counts + (counts ? graphs * per : 0);
    a->row_words = rows;
    a->col_words = cols;
    a->row_words_batch = graphs > 1 ? a->Nq * rw : 0;
    a->col_words_batch = graphs > 1 ? a->Nk * cw : 0;
    a->sparse = flags;
    a->sparse_batch = graphs > 1;
    if (!build) return GATMI_OK;
    GATMI_REQUIRE(per <= kDotBlocks, GATMI_ERANGE, "%s: a mask of %d x %d", what, a->Nq, a->Nk);
    const int64_t step = std::max<int64_t>(1, kDotBlocks / per);
    for (int64_t b0 = 0; b0 < graphs; b0 += step) {
        const int64_t now = std::min(step, graphs - b0);
        int32_t *count = counts ? counts + b0 * per : nullptr;
        hipLaunchKernelGGL(dot_mask_kernel, dim3((unsigned)(now * per)), dim3(256), 0, st, a->bias + b0 * a->bias_batch, a->bias_batch, a->bias_row, a->Nq, a->Nk,
                           rows + b0 * a->Nq * rw, cols + b0 * a->Nk * cw, count);
        if (counts) hipLaunchKernelGGL(dot_mask_count_kernel, dim3((unsigned)now), dim3(256), 0, st, count, (int)per, (int64_t)a->Nq * a->Nk / dot_entries_share(dtype), flags + b0);
    }
    GATMI_LAUNCH_CHECK("dot_attn (mask)");
    return GATMI_OK;
}
template <int DP>
static dim3 dot_entries_grid(int64_t rows) { return dim3((unsigned)std::min<int64_t>(4096, (rows + Entries<DP>::ROWS - 1) / Entries<DP>::ROWS)); }

// whether the passes read the mask as words: more than one wave of rows walks it
static bool dot_wants_words(int64_t rows) { return rows > 16; }

extern "C" size_t gatmi_dot_attn_mask_floats(int64_t B, int32_t Nq, int32_t Nk, int64_t bias_batch) {
    if (B <= 0 || Nq <= 0 || Nk <= 0) return 0;
    return dot_mask_floats(bias_batch ? B : 1, Nq, Nk);
}

extern "C" size_t gatmi_dot_attn_fwd_ws_floats(int64_t B, int32_t Nq, int32_t Nk, int32_t H, int32_t Hkv, int32_t D) {
    if (B <= 0 || Nq <= 0 || Nk <= 0 || H <= 0 || Hkv <= 0 || H % Hkv || D <= 0) return 0;
    const int64_t rows = (int64_t)Nq * (H / Hkv);
    const int splits = dot_splits(B, rows, Hkv, Nk);
    return splits == 1 ? 0 : (size_t)B * Hkv * rows * splits * (D + 2);
}

// Whether fp32 rows are computed as three parts.  Splitting costs as much as so many rows by keys cost on the fp32 instructions; fp32 against parts,
// forward with backward / forward alone, 4 heads, masks of 10 %, in us:
//   32 wide: 256 graphs of 100: 116 / 29 - 117 / 40; of 150: 277 / 68 - 235 / 70; 64 of 512: 401 / 98 - 301 / 85
//   64 wide: 256 of 100: 228 / 58 - 215 / 70;  64 of 256: 222 / 56 - 176 / 54;  16 of 1024: 733 / 185 - 480 / 121
//   128 wide: 256 of 150: 844 / 192 - 934 / 305;  256 of 200: 1403 / 318 - 1365 / 419;  16 of 1024: 1509 / 344 - 1134 / 290
// Up to 16 wide the vector units, not the products, take the time, and parts add to their work (8 wide: 256 of 100: 59 - 83; 16 of 1024: 213 - 196).
static bool dot_splits_parts(int32_t dtype, int64_t rows, int32_t Nk, int32_t D, bool backward) {
    return dtype == GATMI_DTYPE_F32 && D > 16 && std::min<int64_t>(rows, Nk) > (backward ? (D > 64 ? 192 : 96) : (D > 64 ? 768 : 256));
}
static size_t dot_part_row_floats(int D) { return (D <= 32 ? 32 : (D <= 64 ? 64 : 128)) * 3 / 2; }

// where the parts of q, k and v of one call lie
template <int DP>
static void dot_part_rows(const DotArgs &a, int64_t B, float *planes, DotRows (&r)[3]) {
    constexpr int64_t COLS = Shape<Split3, DP>::COLS;
    uint16_t *p = reinterpret_cast<uint16_t *>(planes);
    const int64_t q = (int64_t)a.Nq * a.H * COLS, k = (int64_t)a.Nk * a.Hkv * COLS;
    r[0] = DotRows{p, q, a.H * COLS, COLS};
    r[1] = DotRows{p + B * q, k, a.Hkv * COLS, COLS};
    r[2] = DotRows{p + B * (q + k), k, a.Hkv * COLS, COLS};
}
template <int DP, bool DELTA>
static void dot_split_launch(const SplitArgs &a, int count, hipStream_t st) {
    const int64_t most = std::max(a.rows[0], std::max(a.rows[1], a.rows[2])), per = 256 / (DP / 8);
    hipLaunchKernelGGL((dot_split_kernel<DP, DELTA>), dim3((unsigned)std::min<int64_t>(1 << 20, (most + per - 1) / per), count), dim3(256), 0, st, a);
}

template <typename T, int DP>
static int dot_fwd_run(DotArgs a, int64_t B, float *planes, hipStream_t st) {
    using S = Shape<T, DP>;
    const int64_t rows = (int64_t)a.Nq * a.group;
    if (a.sparse) hipLaunchKernelGGL((dot_entries_fwd_kernel<Elem<T>, DP>), dot_entries_grid<DP>(B * a.Nq * a.H), dim3(256), 0, st, a, B * a.Nq * a.H);
    if constexpr (kSplit<T>) {
        DotRows r[3];
        dot_part_rows<DP>(a, B, planes, r);
        SplitArgs s = {};
        s.D = a.D;
        const DotRows *from[3] = {&a.q, &a.k, &a.v};
        for (int z = 0; z < 3; ++z) {
            s.x[z] = *from[z];
            s.out[z] = const_cast<void *>(r[z].p);
            s.N[z] = z ? a.Nk : a.Nq;
            s.heads[z] = z ? a.Hkv : a.H;
            s.rows[z] = B * s.N[z] * s.heads[z];
        }
        dot_split_launch<DP, false>(s, 3, st);
        a.q = r[0]; a.k = r[1]; a.v = r[2];
    }
    constexpr int NQ = S::NQ;
    constexpr bool COARSE = std::is_same_v<T, uint16_t>, FEW = !kSplit<T> && !COARSE;       // without a mask only; 64 rows or fewer come here
    const int per = rows <= 16 && FEW ? 16 : (rows <= 64 ? 64 : 64 * NQ);
    a.tiles = (int)((rows + per - 1) / per);
    const int64_t step = a.splits > 1 ? B : dot_graphs(a);              // split launches are small by construction
    const size_t lds = 4 * S::TILE, lds_keyw = std::max<size_t>(16 * S::KTW * S::ROW, 512 + 4 * S::DT * 1024);
    for (int64_t b0 = 0; b0 < B; b0 += step) {
        a.b0 = b0;
        a.B = (int)std::min(step, B - b0);
        int rc = GATMI_OK;
#define RUN(keyw, nq, split, bytes)                                                                                                      \
    (a.bias ? dot_launch("dot_attn_fwd", dot_fwd_kernel<T, DP, keyw, nq, split, COARSE ? kNoMask : (keyw ? kFloats : kBits)>, a, bytes, st) \
            : dot_launch("dot_attn_fwd", dot_fwd_kernel<T, DP, keyw, nq, split, kNoMask>, a, bytes, st))
        if (per == 16) {
            if constexpr (FEW) rc = a.splits > 1 ? RUN(true, 1, true, lds_keyw) : RUN(true, 1, false, lds_keyw);
        } else if (per == 64) {
            if constexpr (FEW) rc = a.splits > 1 ? RUN(false, 1, true, lds) : RUN(false, 1, false, lds);
        } else {
            if constexpr (NQ > 1) rc = a.splits > 1 ? RUN(false, NQ, true, lds) : RUN(false, NQ, false, lds);
        }
#undef RUN
        if (rc) return rc;
    }
    if (a.splits > 1) {
        a.b0 = 0;
        const int64_t total = B * a.Hkv * rows;
        const int64_t per_block = 256 / (a.D / 4);
        if (a.splits <= 16) hipLaunchKernelGGL((dot_join_few_kernel<Elem<T>>), dim3((unsigned)((total + per_block - 1) / per_block)), dim3(256), 0, st, a, total);
        else hipLaunchKernelGGL((dot_join_kernel<Elem<T>>), dim3((unsigned)std::min<int64_t>(1 << 16, total)), dim3(256), 0, st, a, total);
    }
    GATMI_LAUNCH_CHECK("dot_attn_fwd");
    return GATMI_OK;
}

// bf16: whether P and dz are two numbers each.  Rounded to one they add as much to the results' error as the rounding of the results does (1.41 times it
// together), whatever the number of nodes; over a mask's fewer entries it shows more (dq of 2 % masks: 1.53 times), so masks always have two.  Without a
// mask the second number costs up to half of the time at any size.  Forward and backward, one - two numbers, in us: 16 graphs of 1024, 4 heads of 64:
// 117 - 145, of 128: 194 - 270; 4 of 1024, 16 heads on 4 of 128: 374 - 347; 4 of 1536: 626 - 620; 8 of 1536, 4 heads of 128: 257 - 353; 8 of 2048: 340 - 501; 4 of
// 2048, 16 on 4 of 128: 881 - 979; 4 of 4096, 16 on 4 of 64: 1299 - 1749, of 128: 2539 - 3772.  So the border is a choice: up to 1024 nodes, the
// sizes of whole small graphs, the accuracy of a single rounding; beyond, where this is most of a step, the time.
static bool dot_wide16(int64_t rows, int64_t Nq, int64_t Nk, bool mask) { return mask || rows <= 64 || Nk <= 64 || std::max(Nq, Nk) <= 1024; }

#define GATMI_DOT_DISPATCH(RUN, parts)                                                             \
    if (dtype == GATMI_DTYPE_F32 && (parts)) {                                                     \
        if (D <= 32) return RUN(Split3, 32);                                                       \
        if (D <= 64) return RUN(Split3, 64);                                                       \
        return RUN(Split3, 128);                                                                   \
    }                                                                                              \
    if (dtype == GATMI_DTYPE_F32) {                                                                \
        if (D <= 8) return RUN(float, 8);                                                          \
        if (D <= 16) return RUN(float, 16);                                                        \
        if (D <= 32) return RUN(float, 32);                                                        \
        if (D <= 64) return RUN(float, 64);                                                        \
        return RUN(float, 128);                                                                    \
    }                                                                                              \
    if (dot_wide16((int64_t)Nq * (H / Hkv), Nq, Nk, bias != nullptr)) {                                             \
        if (D <= 16) return RUN(Wide16, 16);                                                       \
        if (D <= 32) return RUN(Wide16, 32);                                                       \
        if (D <= 64) return RUN(Wide16, 64);                                                       \
        return RUN(Wide16, 128);                                                                   \
    }                                                                                              \
    if (D <= 16) return RUN(uint16_t, 16);                                                         \
    if (D <= 32) return RUN(uint16_t, 32);                                                         \
    if (D <= 64) return RUN(uint16_t, 64);                                                         \
    return RUN(uint16_t, 128);

extern "C" size_t gatmi_dot_attn_planes_floats(int64_t B, int32_t Nq, int32_t Nk, int32_t H, int32_t Hkv, int32_t D, int32_t dtype, int32_t backward) {
    if (B <= 0 || Nq <= 0 || Nk <= 0 || H <= 0 || Hkv <= 0 || H % Hkv || D <= 0 || !dot_splits_parts(dtype, (int64_t)Nq * (H / Hkv), Nk, D, backward != 0)) return 0;
    return dot_part_row_floats(D) * (size_t)B * ((size_t)Nq * H + 2 * (size_t)Nk * Hkv);
}

extern "C" size_t gatmi_dot_attn_bwd_ws_floats(int64_t B, int32_t Nq, int32_t Nk, int32_t H, int32_t Hkv, int32_t D, int32_t dtype) {
    return gatmi_dot_attn_planes_floats(B, Nq, Nk, H, Hkv, D, dtype, 1) ? dot_part_row_floats(D) * (size_t)B * Nq * H : 0;
}

extern "C" int gatmi_dot_attn_fwd(int64_t B, int32_t Nq, int32_t Nk, int32_t H, int32_t Hkv, int32_t D, int32_t dtype, const void *q, const int64_t *q_stride,
                                  const void *k, const int64_t *k_stride, const void *v, const int64_t *v_stride, const float *bias, int64_t bias_batch,
                                  int64_t bias_row, const int32_t *key_sizes, const int32_t *query_sizes, float scale, void *out, void *out_low, float *lse, float *mask_words, float *planes, float *ws, void *stream) {
    if (int rc = dot_check("dot_attn_fwd", B, Nq, Nk, H, Hkv, D, dtype)) return rc;
    GATMI_REQUIRE(std::isfinite(scale), GATMI_EINVAL, "dot_attn_fwd: scale %g", (double)scale);
    if (B == 0 || Nq == 0) return GATMI_OK;
    DotArgs a = {};
    if (int rc = dot_rows("dot_attn_fwd", "q", &a.q, q, q_stride, dtype)) return rc;
    if (Nk > 0) {
        if (int rc = dot_rows("dot_attn_fwd", "k", &a.k, k, k_stride, dtype)) return rc;
        if (int rc = dot_rows("dot_attn_fwd", "v", &a.v, v, v_stride, dtype)) return rc;
    }
    GATMI_REQUIRE(out, GATMI_EINVAL, "dot_attn_fwd: out is null");
    GATMI_REQUIRE_ALIGNED(out);
    GATMI_REQUIRE(!bias || bias_row >= Nk || Nq == 1, GATMI_EINVAL, "dot_attn_fwd: bias row stride %lld below Nk = %d", (long long)bias_row, Nk);
    GATMI_REQUIRE(!out_low || dtype == GATMI_DTYPE_BF16, GATMI_EINVAL, "dot_attn_fwd: out_low is for bf16");
    GATMI_REQUIRE_ALIGNED(out_low);
    a.out = out; a.out_low = static_cast<uint16_t *>(out_low); a.lse = lse; a.bias = Nk > 0 ? bias : nullptr; a.bias_batch = bias_batch; a.bias_row = bias_row;
    a.key_sizes = key_sizes; a.query_sizes = query_sizes; a.scale = scale; a.scale2 = std::max(std::fabs(scale) * kLog2e, 1e-37f);      // above 0: -inf stays -inf
    a.Nq = Nq; a.Nk = Nk; a.H = H; a.Hkv = Hkv; a.group = H / Hkv; a.D = D;
    const int64_t rows = (int64_t)Nq * a.group;
    a.splits = dot_splits(B, rows, Hkv, Nk);
    if (a.splits > 1) {
        GATMI_REQUIRE(ws, GATMI_EINVAL, "dot_attn_fwd: workspace is null");
        GATMI_REQUIRE_ALIGNED(ws);
        a.part_o = ws;
        a.part_ml = ws + (size_t)B * Hkv * rows * a.splits * D;
    }
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    if (a.bias && (mask_words || dot_wants_words(rows)))
        if (int rc = dot_mask_words("dot_attn_fwd", &a, bias_batch ? B : 1, mask_words, dtype, true, st)) return rc;
    GATMI_REQUIRE_ALIGNED(planes);
#define RUN(T, dp) dot_fwd_run<T, dp>(a, B, planes, st)
    GATMI_DOT_DISPATCH(RUN, planes && dot_splits_parts(dtype, rows, Nk, D, lse != nullptr))
#undef RUN
}

template <typename T, int DP>
static int dot_bwd_run(DotArgs a, int64_t B, float *planes, float *ws, hipStream_t st) {
    using S = Shape<T, DP>;
    const int64_t rows = (int64_t)a.Nq * a.group;
    if (a.sparse) {
        hipLaunchKernelGGL((dot_entries_q_kernel<Elem<T>, DP>), dot_entries_grid<DP>(B * a.Nq * a.H), dim3(256), 0, st, a, B * a.Nq * a.H);
        hipLaunchKernelGGL((dot_entries_kv_kernel<Elem<T>, DP>), dot_entries_grid<DP>(B * a.Nk * a.Hkv), dim3(256), 0, st, a, B * a.Nk * a.Hkv);
    }
    if constexpr (kSplit<T>) {                                          // q, k, v as the forward left them; dout now, with delta
        DotRows r[3];
        dot_part_rows<DP>(a, B, planes, r);
        SplitArgs s = {};
        s.D = a.D;
        s.x[0] = a.d_o;
        s.o = a.o;
        s.delta = a.delta;
        s.out[0] = ws;
        s.N[0] = a.Nq;
        s.heads[0] = a.H;
        s.rows[0] = B * a.Nq * a.H;
        dot_split_launch<DP, true>(s, 1, st);
        a.q = r[0]; a.k = r[1]; a.v = r[2];
        a.d_o = DotRows{ws, r[0].batch, r[0].node, r[0].head};
    }
    a.splits = 1;
    constexpr int NQ = S::NQ, NK = S::nk(false), NKM = S::nk(true);
    constexpr bool COARSE = std::is_same_v<T, uint16_t>, FEW = !kSplit<T> && !COARSE;       // as in the forward
    constexpr int BITS = COARSE ? kNoMask : kBits;
    for (int pass = 0; pass < 2; ++pass) {
        const int64_t count = pass == 0 ? rows : a.Nk;
        if (count == 0) continue;
        const bool wide = count > 64;
        const int per = 64 * (wide ? (pass == 0 ? NQ : (a.bias ? NKM : NK)) : 1);
        a.tiles = (int)((count + per - 1) / per);
        const int64_t step = dot_graphs(a);
        for (int64_t b0 = 0; b0 < B; b0 += step) {
            a.b0 = b0;
            a.B = (int)std::min(step, B - b0);
            int rc = GATMI_OK;
#define RUN(kernel, n, mask) dot_launch("dot_attn_bwd", kernel<T, DP, n, mask>, a, 4 * S::TILE, st)
            if (pass == 0) {
                if (wide) rc = a.bias ? RUN(dot_bwd_q_kernel, NQ, BITS) : RUN(dot_bwd_q_kernel, NQ, kNoMask);
                else if constexpr (FEW) rc = a.bias ? RUN(dot_bwd_q_kernel, 1, BITS) : RUN(dot_bwd_q_kernel, 1, kNoMask);
            } else {
                if (wide) rc = a.bias ? RUN(dot_bwd_kv_kernel, (COARSE ? NK : NKM), BITS) : RUN(dot_bwd_kv_kernel, NK, kNoMask);
                else if constexpr (FEW) rc = a.bias ? RUN(dot_bwd_kv_kernel, 1, BITS) : RUN(dot_bwd_kv_kernel, 1, kNoMask);
            }
#undef RUN
            if (rc) return rc;
        }
    }
    GATMI_LAUNCH_CHECK("dot_attn_bwd");
    return GATMI_OK;
}

extern "C" int gatmi_dot_attn_bwd(int64_t B, int32_t Nq, int32_t Nk, int32_t H, int32_t Hkv, int32_t D, int32_t dtype, const void *q, const int64_t *q_stride,
                                  const void *k, const int64_t *k_stride, const void *v, const int64_t *v_stride, const void *out, const void *out_low, const void *dout,
                                  const int64_t *dout_stride, const float *lse, const float *bias, int64_t bias_batch, int64_t bias_row,
                                  const int32_t *key_sizes, const int32_t *query_sizes, float scale, float *mask_words, float *planes, void *dq, void *dk, void *dv,
                                  float *delta, float *ws, void *stream) {
    if (int rc = dot_check("dot_attn_bwd", B, Nq, Nk, H, Hkv, D, dtype)) return rc;
    GATMI_REQUIRE(std::isfinite(scale), GATMI_EINVAL, "dot_attn_bwd: scale %g", (double)scale);
    if (B == 0 || (Nq == 0 && Nk == 0)) return GATMI_OK;
    DotArgs a = {};
    const int64_t own[3] = {(int64_t)Nq * H * D, (int64_t)H * D, D};
    if (Nq > 0) {
        if (int rc = dot_rows("dot_attn_bwd", "q", &a.q, q, q_stride, dtype)) return rc;
        if (int rc = dot_rows("dot_attn_bwd", "out", &a.o, out, own, dtype)) return rc;
        if (int rc = dot_rows("dot_attn_bwd", "dout", &a.d_o, dout, dout_stride, dtype)) return rc;
        GATMI_REQUIRE(lse && delta && dq, GATMI_EINVAL, "dot_attn_bwd: null pointer");
        GATMI_REQUIRE_ALIGNED(dq);
    }
    if (Nk > 0) {
        if (int rc = dot_rows("dot_attn_bwd", "k", &a.k, k, k_stride, dtype)) return rc;
        if (int rc = dot_rows("dot_attn_bwd", "v", &a.v, v, v_stride, dtype)) return rc;
        GATMI_REQUIRE(dk && dv, GATMI_EINVAL, "dot_attn_bwd: null pointer");
        GATMI_REQUIRE_ALIGNED(dk);
        GATMI_REQUIRE_ALIGNED(dv);
    }
    GATMI_REQUIRE(!bias || bias_row >= Nk || Nq <= 1, GATMI_EINVAL, "dot_attn_bwd: bias row stride %lld below Nk = %d", (long long)bias_row, Nk);
    GATMI_REQUIRE(!out_low || dtype == GATMI_DTYPE_BF16, GATMI_EINVAL, "dot_attn_bwd: out_low is for bf16");
    GATMI_REQUIRE_ALIGNED(out_low);
    a.out_low = static_cast<uint16_t *>(const_cast<void *>(out_low));
    a.dq = dq; a.dk = dk; a.dv = dv; a.lse = const_cast<float *>(lse); a.delta = delta;
    a.bias = Nk > 0 && Nq > 0 ? bias : nullptr; a.bias_batch = bias_batch; a.bias_row = bias_row;
    a.key_sizes = key_sizes; a.query_sizes = query_sizes; a.scale = scale; a.scale2 = std::max(std::fabs(scale) * kLog2e, 1e-37f);      // above 0: -inf stays -inf
    a.Nq = Nq; a.Nk = Nk; a.H = H; a.Hkv = Hkv; a.group = H / Hkv; a.D = D;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    if (a.bias)
        if (int rc = dot_mask_words("dot_attn_bwd", &a, bias_batch ? B : 1, mask_words, dtype, false, st)) return rc;
    const bool parts = planes && dot_splits_parts(dtype, (int64_t)Nq * a.group, Nk, D, true);
    GATMI_REQUIRE(!parts || ws, GATMI_EINVAL, "dot_attn_bwd: workspace is null");
    GATMI_REQUIRE_ALIGNED(planes);
    GATMI_REQUIRE_ALIGNED(ws);
#define RUN(T, dp) dot_bwd_run<T, dp>(a, B, planes, ws, st)
    GATMI_DOT_DISPATCH(RUN, parts)
#undef RUN
}
