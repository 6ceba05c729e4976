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
// and the probabilities sit in the operand layout of the second product as they are: they never go through LDS.  bf16 rounds P and
// dz to bf16 for that product (half a step of 2^-8, as its other operand has and its result is stored with).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "common.h"
#include "device_common.h"

namespace gatmi {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef short i16x8 __attribute__((ext_vector_type(8)));
struct __attribute__((packed, aligned(4))) f32x4_u { float v[4]; };       // a 16-byte access at 4-byte alignment

constexpr float kAttended = -1e8f;
constexpr int kSplitsMax = 256;

// ---- operand fragments -------------------------------------------------------------------------------------------------
// DP: head width padded to what is staged.  A fragment is what a lane holds of 16 rows x KD elements: lane (r = l & 15,
// q = l >> 4) the PIECE bytes at q * PIECE of the fragment's part of row r.
template <typename T, int DP> struct Shape;
template <int DP> struct Shape<float, DP> {
    static constexpr int PIECE = DP == 8 ? 8 : 16, KD = PIECE, FRAGS = DP / KD;           // PIECE bytes = PIECE / 4 elements, 4 lane groups: KD = PIECE elements
    static constexpr int ROW = DP * 4, PAD = ROW + 16;                                    // bytes of a staged row, and its stride in LDS
    static constexpr int CHUNK = 16;                                                      // rows that one fragment of the second product covers
};
template <int DP> struct Shape<uint16_t, DP> {
    static constexpr int PIECE = 16, KD = 32, FRAGS = DP < 32 ? 1 : DP / 32;
    static constexpr int ROW = (DP < 32 ? 32 : DP) * 2, PAD = ROW + 16;
    static constexpr int CHUNK = 32;
};

struct FragF { float v[4]; };
struct FragH { uint4 v; };
template <typename T> struct FragOf;
template <> struct FragOf<float> { using type = FragF; };
template <> struct FragOf<uint16_t> { using type = FragH; };
template <typename T> using Frag = typename FragOf<T>::type;

template <typename T, int DP>
__device__ __forceinline__ Frag<T> frag_zero() {
    if constexpr (sizeof(T) == 4) return FragF{{0.f, 0.f, 0.f, 0.f}};
    else return FragH{make_uint4(0, 0, 0, 0)};
}
// from 16-byte aligned memory (8 for DP = 8)
template <typename T, int DP>
__device__ __forceinline__ Frag<T> frag_load(const char *p) {
    if constexpr (sizeof(T) == 4) {
        if constexpr (DP == 8) {
            const float2 u = *reinterpret_cast<const float2 *>(p);
            return FragF{{u.x, u.y, 0.f, 0.f}};
        } else {
            const float4 u = *reinterpret_cast<const float4 *>(p);
            return FragF{{u.x, u.y, u.z, u.w}};
        }
    } else {
        return FragH{*reinterpret_cast<const uint4 *>(p)};
    }
}

// acc += A B over the KD elements of one fragment
template <typename T, int DP>
__device__ __forceinline__ void mma(const Frag<T> &a, const Frag<T> &b, f32x4 &acc) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int t = 0; t < (DP == 8 ? 2 : 4); ++t) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[t], b.v[t], acc, 0, 0, 0);
    } else {
        acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a.v), __builtin_bit_cast(bf16x8, b.v), acc, 0, 0, 0);
    }
}

// The second product sums over CHUNK staged rows.  Its B operand is made of score tiles (C layout: row 4 q + r of a
// tile in register r), its A operand reads the staged rows column-wise in the same order of rows.
template <typename T>
__device__ __forceinline__ Frag<T> frag_scores(const f32x4 *tile) {
    if constexpr (sizeof(T) == 4) return FragF{{tile[0][0], tile[0][1], tile[0][2], tile[0][3]}};
    else return FragH{make_uint4(pack_bf16x2(tile[0][0], tile[0][1]), pack_bf16x2(tile[0][2], tile[0][3]), pack_bf16x2(tile[1][0], tile[1][1]), pack_bf16x2(tile[1][2], tile[1][3]))};
}
template <typename T, int DP>
__device__ __forceinline__ Frag<T> frag_turned(const char *tile, int row0, int d0) {
    const int lane = threadIdx.x & 63;
    if constexpr (sizeof(T) == 4) {
        const char *p = tile + (row0 + 4 * (lane >> 4)) * Shape<T, DP>::PAD + (d0 + (lane & 15)) * 4;
        FragF f;
#pragma unroll
        for (int r = 0; r < 4; ++r) f.v[r] = *reinterpret_cast<const float *>(p + r * Shape<T, DP>::PAD);
        return f;
    } else {
        // ds_read_b64_tr_b16: 16 lanes give the addresses of a 4 x 16 block (lane i: row i / 4, columns 4 (i % 4) ..), each gets a column of it
        const char *p = tile + (row0 + 4 * (lane >> 4) + ((lane & 15) >> 2)) * Shape<T, DP>::PAD + (d0 + (lane & 3) * 4) * 2;
        using lds4 = __attribute__((address_space(3))) i16x4;
        const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4 *)p);
        const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4 *)(p + 16 * Shape<T, DP>::PAD));
        return FragH{__builtin_bit_cast(uint4, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7))};
    }
}
// acc += A B over the rows of one such fragment (fp32: always four steps)
template <typename T>
__device__ __forceinline__ void mma_rows(const Frag<T> &a, const Frag<T> &b, f32x4 &acc) { mma<T, 16>(a, b, acc); }

// ---- arguments ---------------------------------------------------------------------------------------------------------
struct DotRows {              // [B, N, heads, D] rows: element strides, D contiguous
    const void *p;
    int64_t batch, node, head;
};

struct DotArgs {
    DotRows q, k, v, o, d_o;
    void *out, *dq, *dk, *dv;           // contiguous [B, N, heads, D]
    float *lse, *delta;                 // [B, H, Nq]: log2 of the row's sum of exponentials; <do, out>
    const float *bias;
    int64_t bias_batch, bias_row;
    const int32_t *key_sizes, *query_sizes;
    int64_t b0;                         // first graph of this launch
    int B, Nq, Nk, H, Hkv, group, D;
    int tiles, splits;                  // row (or key) tiles, key ranges
    int split_keys;                     // keys of a range
    float scale;
    float *part_o, *part_ml;            // split forward: [rows of the launch][splits][DP], [..][2]
};

__device__ __forceinline__ int graph_size(const int32_t *sizes, int64_t b, int n) { return sizes ? max(0, min(sizes[b], n)) : n; }

// one 16-byte (8-byte) piece of a row, zeros outside it
template <typename T, int DP>
__device__ __forceinline__ Frag<T> row_piece(const T *row, int elem, int D, bool ok) {
    return ok && elem < D ? frag_load<T, DP>(reinterpret_cast<const char *>(row + elem)) : frag_zero<T, DP>();
}

// ---- staging of KT rows of two tensors -----------------------------------------------------------------------------------
template <typename T, int DP, int KT, int THREADS>
struct Stage {
    using S = Shape<T, DP>;
    static constexpr int PIECES = S::ROW / S::PIECE, TOTAL = KT * PIECES, PER = (TOTAL + THREADS - 1) / THREADS, ELEMS = S::PIECE / (int)sizeof(T);
    Frag<T> a[PER], b[PER];
    // row r of the tile: rows.p + offset(r), valid while r < count
    template <typename Off>
    __device__ __forceinline__ void load(const DotRows &x, const DotRows &y, int count, int D, Off &&offset) {
#pragma unroll
        for (int u = 0; u < PER; ++u) {
            const int e = threadIdx.x + u * THREADS, r = e / PIECES, c = (e % PIECES) * ELEMS;
            const bool ok = (TOTAL % THREADS == 0 || e < TOTAL) && r < count && c < D;
            if (ok) {
                a[u] = frag_load<T, DP>(reinterpret_cast<const char *>(reinterpret_cast<const T *>(x.p) + offset(x, r) + c));
                b[u] = frag_load<T, DP>(reinterpret_cast<const char *>(reinterpret_cast<const T *>(y.p) + offset(y, r) + c));
            } else {
                a[u] = frag_zero<T, DP>();
                b[u] = frag_zero<T, DP>();
            }
        }
    }
    __device__ __forceinline__ void put(char *p, const Frag<T> &f) const {
        if constexpr (sizeof(T) == 4) {
            if constexpr (DP == 8) *reinterpret_cast<float2 *>(p) = make_float2(f.v[0], f.v[1]);
            else *reinterpret_cast<float4 *>(p) = make_float4(f.v[0], f.v[1], f.v[2], f.v[3]);
        } else {
            *reinterpret_cast<uint4 *>(p) = f.v;
        }
    }
    __device__ __forceinline__ void store(char *x, char *y) const {
#pragma unroll
        for (int u = 0; u < PER; ++u) {
            const int e = threadIdx.x + u * THREADS, r = e / PIECES, c = e % PIECES;
            if (TOTAL % THREADS == 0 || e < TOTAL) {
                put(x + r * S::PAD + c * S::PIECE, a[u]);
                put(y + r * S::PAD + c * S::PIECE, b[u]);
            }
        }
    }
};

// z of four consecutive keys j .. j + 3 of one query, -inf where the key is not attended
__device__ __forceinline__ void masked_logits(f32x4 &z, float scale, const float *bias_row, int j, int nk, int keys) {
    if (bias_row) {
        float bv[4];
        if (j + 3 < nk) {
            const f32x4_u u = *reinterpret_cast<const f32x4_u *>(bias_row + j);
#pragma unroll
            for (int r = 0; r < 4; ++r) bv[r] = u.v[r];
        } else {
#pragma unroll
            for (int r = 0; r < 4; ++r) bv[r] = j + r < nk ? bias_row[j + r] : -INFINITY;
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) z[r] = bv[r] > kAttended && j + r < keys ? fmaf(z[r], scale, bv[r]) : -INFINITY;
    } else {
#pragma unroll
        for (int r = 0; r < 4; ++r) z[r] = j + r < keys ? z[r] * scale : -INFINITY;
    }
}

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

// which (graph, key/value head, tile, split) a block of the 1-d grid works on
struct DotBlock { int64_t b; int hk, tile, split; };
__device__ __forceinline__ DotBlock dot_block(const DotArgs &a) {
    DotBlock r;
    uint32_t id = blockIdx.x;
    r.split = id % a.splits; id /= a.splits;
    r.tile = id % a.tiles; id /= a.tiles;
    r.hk = id % a.Hkv;
    r.b = a.b0 + id / a.Hkv;
    return r;
}

template <typename T, int DP> struct Tiles {
    static constexpr int KT = (sizeof(T) == 4 && DP == 128) ? 32 : 64;      // staged rows: both tensors' tiles stay below 64 KB
    static constexpr int DT = (DP + 15) / 16;                              // 16-wide tiles of a result row
    static constexpr int LDS = 2 * KT * Shape<T, DP>::PAD;
};

// ---- forward -------------------------------------------------------------------------------------------------------------
// WAVES x NQ x 16 rows per block.  SPLIT: the block covers one range of the keys and leaves its unnormalised row sums.
template <typename T, int DP, int WAVES, int NQ, bool SPLIT>
__global__ __launch_bounds__(64 * WAVES) void dot_fwd_kernel(DotArgs a) {
    using S = Shape<T, DP>;
    using TL = Tiles<T, DP>;
    constexpr int KT = TL::KT, DT = TL::DT, ROWS = WAVES * NQ * 16;
    __shared__ __attribute__((aligned(16))) char lds[TL::LDS];
    char *ks = lds, *vs = lds + KT * S::PAD;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 15, q4 = lane >> 4;
    const DotBlock blk = dot_block(a);
    const int64_t b = blk.b;
    const int keys = graph_size(a.key_sizes, b, a.Nk), queries = graph_size(a.query_sizes, b, a.Nq);
    const int j0 = SPLIT ? blk.split * a.split_keys : 0, j1 = SPLIT ? min(keys, j0 + a.split_keys) : keys;
    int row[NQ], qi[NQ], head[NQ];
    bool live[NQ];
    Frag<T> qf[NQ][S::FRAGS];
    const float *bias_row[NQ];
#pragma unroll
    for (int u = 0; u < NQ; ++u) {
        row[u] = blk.tile * ROWS + (wave * NQ + u) * 16 + n;
        qi[u] = row[u] / a.group;
        head[u] = blk.hk * a.group + row[u] % a.group;
        live[u] = qi[u] < queries;
        const T *qrow = reinterpret_cast<const T *>(a.q.p) + b * a.q.batch + (live[u] ? qi[u] : 0) * a.q.node + head[u] * a.q.head;
#pragma unroll
        for (int c = 0; c < S::FRAGS; ++c) qf[u][c] = row_piece<T, DP>(qrow, c * S::KD + q4 * (S::PIECE / (int)sizeof(T)), a.D, live[u]);
        bias_row[u] = a.bias ? a.bias + b * a.bias_batch + (int64_t)(live[u] ? qi[u] : 0) * a.bias_row : nullptr;
    }
    f32x4 o[NQ][DT];
    float m[NQ], l[NQ];
#pragma unroll
    for (int u = 0; u < NQ; ++u) {
        m[u] = -INFINITY;
        l[u] = 0.f;
#pragma unroll
        for (int t = 0; t < DT; ++t) o[u][t] = (f32x4){0.f, 0.f, 0.f, 0.f};
    }
    Stage<T, DP, KT, 64 * WAVES> st;
    const int64_t kb = b * a.k.batch + blk.hk * a.k.head, vb = b * a.v.batch + blk.hk * a.v.head;
    auto fetch = [&](int j) {
        st.load(a.k, a.v, j1 - j, a.D, [&](const DotRows &x, int r) { return (&x == &a.k ? kb : vb) + (int64_t)(j + r) * x.node; });
    };
    if (j0 < j1) fetch(j0);
    for (int j = j0; j < j1; j += KT) {
        __syncthreads();
        st.store(ks, vs);
        __syncthreads();
        if (j + KT < j1) fetch(j + KT);
        f32x4 z[NQ][KT / 16];
#pragma unroll
        for (int t = 0; t < KT / 16; ++t) {
#pragma unroll
            for (int u = 0; u < NQ; ++u) z[u][t] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < S::FRAGS; ++c) {
                const Frag<T> kf = frag_load<T, DP>(ks + (16 * t + n) * S::PAD + c * 4 * S::PIECE + q4 * S::PIECE);
#pragma unroll
                for (int u = 0; u < NQ; ++u) mma<T, DP>(kf, qf[u][c], z[u][t]);
            }
        }
#pragma unroll
        for (int u = 0; u < NQ; ++u) {
            float top = -INFINITY;
#pragma unroll
            for (int t = 0; t < KT / 16; ++t) {
                masked_logits(z[u][t], a.scale, bias_row[u], j + 16 * t + 4 * q4, a.Nk, j1);
                top = fmaxf(top, fmaxf(fmaxf(z[u][t][0], z[u][t][1]), fmaxf(z[u][t][2], z[u][t][3])));
            }
            top = over_groups_max(top) * kLog2e;                     // the maximum in units of log2: every term of the row uses the same rounded value
            const float now = fmaxf(m[u], top), base = now == -INFINITY ? 0.f : now;
            const float shrink = __builtin_amdgcn_exp2f(m[u] - base);
            m[u] = now;
            float sum = 0.f;
#pragma unroll
            for (int t = 0; t < KT / 16; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    z[u][t][r] = __builtin_amdgcn_exp2f(fmaf(z[u][t][r], kLog2e, -base));
                    sum += z[u][t][r];
                }
            l[u] = l[u] * shrink + sum;
#pragma unroll
            for (int t = 0; t < DT; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) o[u][t][r] *= shrink;
        }
#pragma unroll
        for (int c = 0; c < KT / S::CHUNK; ++c) {
            Frag<T> pf[NQ];
#pragma unroll
            for (int u = 0; u < NQ; ++u) pf[u] = frag_scores<T>(&z[u][c * (S::CHUNK / 16)]);
#pragma unroll
            for (int t = 0; t < DT; ++t) {
                const Frag<T> vf = frag_turned<T, DP>(vs, c * S::CHUNK, 16 * t);
#pragma unroll
                for (int u = 0; u < NQ; ++u) mma_rows<T>(vf, pf[u], o[u][t]);
            }
        }
    }
#pragma unroll
    for (int u = 0; u < NQ; ++u) {
        const float sum = over_groups_sum(l[u]);
        if (qi[u] >= a.Nq) continue;
        if constexpr (SPLIT) {
            const int64_t at = ((((b - a.b0) * a.Hkv + blk.hk) * (int64_t)a.Nq * a.group + row[u]) * a.splits + blk.split);
#pragma unroll
            for (int t = 0; t < DT; ++t)
                if (16 * t + 4 * q4 < a.D) store4<float>(a.part_o + at * a.D + 16 * t + 4 * q4, o[u][t]);
            if (q4 == 0) {
                a.part_ml[2 * at] = m[u];
                a.part_ml[2 * at + 1] = sum;
            }
        } else {
            const float inv = !live[u] || sum == 0.f ? 0.f : 1.0f / sum;
            T *orow = reinterpret_cast<T *>(a.out) + ((b * a.Nq + qi[u]) * a.H + head[u]) * (int64_t)a.D;
#pragma unroll
            for (int t = 0; t < DT; ++t)
                if (16 * t + 4 * q4 < a.D) {
                    f32x4 v = o[u][t];
#pragma unroll
                    for (int r = 0; r < 4; ++r) v[r] = inv == 0.f ? 0.f : v[r] * inv;
                    store4<T>(orow + 16 * t + 4 * q4, v);
                }
            if (a.lse && q4 == 0) a.lse[(b * a.H + head[u]) * a.Nq + qi[u]] = inv == 0.f ? INFINITY : m[u] + log2f(sum);
        }
    }
}

// joins the key ranges of a row: one thread per element of the result
template <typename T>
__global__ __launch_bounds__(256) void dot_join_kernel(DotArgs a, int64_t total) {
    for (int64_t e = blockIdx.x * 256ll + threadIdx.x; e < total; e += (int64_t)gridDim.x * 256) {
        const int d = (int)(e % a.D);
        const int64_t rr = e / a.D, rows = (int64_t)a.Nq * a.group;
        const int r = (int)(rr % rows), hk = (int)(rr / rows % a.Hkv), qi = r / a.group, head = hk * a.group + r % a.group;
        const int64_t b = a.b0 + rr / rows / a.Hkv;
        const float *ml = a.part_ml + 2 * rr * a.splits, *po = a.part_o + rr * a.splits * a.D + d;
        float top = -INFINITY;
        for (int s = 0; s < a.splits; ++s) top = fmaxf(top, ml[2 * s]);
        const float base = top == -INFINITY ? 0.f : top;
        float sum = 0.f, o = 0.f;
        for (int s = 0; s < a.splits; ++s) {
            const float w = __builtin_amdgcn_exp2f(ml[2 * s] - base);
            sum = fmaf(ml[2 * s + 1], w, sum);
            o = fmaf(po[(int64_t)s * a.D], w, o);
        }
        const bool live = qi < graph_size(a.query_sizes, b, a.Nq);
        const float inv = !live || sum == 0.f ? 0.f : 1.0f / sum;
        const float v = inv == 0.f ? 0.f : o * inv;
        T *out = reinterpret_cast<T *>(a.out) + ((b * a.Nq + qi) * a.H + head) * (int64_t)a.D + d;
        if constexpr (sizeof(T) == 4) *reinterpret_cast<float *>(out) = v;
        else *out = (T)pack_bf16x2(v, 0.f);
        if (a.lse && d == 0) a.lse[(b * a.H + head) * a.Nq + qi] = inv == 0.f ? INFINITY : top + log2f(sum);
    }
}

// ---- backward: dq and delta ------------------------------------------------------------------------------------------------
template <typename T, int DP, int WAVES, int NQ>
__global__ __launch_bounds__(64 * WAVES) void dot_bwd_q_kernel(DotArgs a) {
    using S = Shape<T, DP>;
    using TL = Tiles<T, DP>;
    constexpr int KT = TL::KT, DT = TL::DT, ROWS = WAVES * NQ * 16;
    __shared__ __attribute__((aligned(16))) char lds[TL::LDS];
    char *ks = lds, *vs = lds + KT * S::PAD;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 15, q4 = lane >> 4;
    const DotBlock blk = dot_block(a);
    const int64_t b = blk.b;
    const int keys = graph_size(a.key_sizes, b, a.Nk), queries = graph_size(a.query_sizes, b, a.Nq);
    int qi[NQ], head[NQ];
    float lse[NQ], delta[NQ];
    Frag<T> qf[NQ][S::FRAGS], df[NQ][S::FRAGS];
    const float *bias_row[NQ];
#pragma unroll
    for (int u = 0; u < NQ; ++u) {
        const int row = blk.tile * ROWS + (wave * NQ + u) * 16 + n;
        qi[u] = row / a.group;
        head[u] = blk.hk * a.group + row % a.group;
        const bool live = qi[u] < queries;
        const int64_t i = live ? qi[u] : 0;
        const T *qrow = reinterpret_cast<const T *>(a.q.p) + b * a.q.batch + i * a.q.node + head[u] * a.q.head;
        const T *drow = reinterpret_cast<const T *>(a.d_o.p) + b * a.d_o.batch + i * a.d_o.node + head[u] * a.d_o.head;
        const T *orow = reinterpret_cast<const T *>(a.o.p) + b * a.o.batch + i * a.o.node + head[u] * a.o.head;
        float dot = 0.f;
#pragma unroll
        for (int c = 0; c < S::FRAGS; ++c) {
            const int e = c * S::KD + q4 * (S::PIECE / (int)sizeof(T));
            qf[u][c] = row_piece<T, DP>(qrow, e, a.D, live);
            df[u][c] = row_piece<T, DP>(drow, e, a.D, live);
            const Frag<T> of = row_piece<T, DP>(orow, e, a.D, live);
            if constexpr (sizeof(T) == 4) {
#pragma unroll
                for (int t = 0; t < 4; ++t) dot = fmaf(df[u][c].v[t], of.v[t], dot);
            } else {
                const uint32_t *x = reinterpret_cast<const uint32_t *>(&df[u][c].v), *y = reinterpret_cast<const uint32_t *>(&of.v);
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    dot = fmaf(__uint_as_float(x[t] << 16), __uint_as_float(y[t] << 16), dot);
                    dot = fmaf(__uint_as_float(x[t] & 0xffff0000u), __uint_as_float(y[t] & 0xffff0000u), dot);
                }
            }
        }
        delta[u] = over_groups_sum(dot);
        lse[u] = live ? a.lse[(b * a.H + head[u]) * a.Nq + qi[u]] : INFINITY;
        if (q4 == 0 && qi[u] < a.Nq) a.delta[(b * a.H + head[u]) * a.Nq + qi[u]] = delta[u];
        bias_row[u] = a.bias ? a.bias + b * a.bias_batch + i * a.bias_row : nullptr;
    }
    f32x4 acc[NQ][DT];
#pragma unroll
    for (int u = 0; u < NQ; ++u)
#pragma unroll
        for (int t = 0; t < DT; ++t) acc[u][t] = (f32x4){0.f, 0.f, 0.f, 0.f};
    Stage<T, DP, KT, 64 * WAVES> st;
    const int64_t kb = b * a.k.batch + blk.hk * a.k.head, vb = b * a.v.batch + blk.hk * a.v.head;
    auto fetch = [&](int j) {
        st.load(a.k, a.v, keys - j, a.D, [&](const DotRows &x, int r) { return (&x == &a.k ? kb : vb) + (int64_t)(j + r) * x.node; });
    };
    if (keys > 0) fetch(0);
    for (int j = 0; j < keys; j += KT) {
        __syncthreads();
        st.store(ks, vs);
        __syncthreads();
        if (j + KT < keys) fetch(j + KT);
#pragma unroll
        for (int c = 0; c < KT / S::CHUNK; ++c) {
            f32x4 z[NQ][S::CHUNK / 16];
#pragma unroll
            for (int t = 0; t < S::CHUNK / 16; ++t) {
                const int r0 = c * S::CHUNK + 16 * t;
                f32x4 dp[NQ];
#pragma unroll
                for (int u = 0; u < NQ; ++u) z[u][t] = dp[u] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int f = 0; f < S::FRAGS; ++f) {
                    const int at = (r0 + n) * S::PAD + f * 4 * S::PIECE + q4 * S::PIECE;
                    const Frag<T> kf = frag_load<T, DP>(ks + at), vf = frag_load<T, DP>(vs + at);
#pragma unroll
                    for (int u = 0; u < NQ; ++u) {
                        mma<T, DP>(kf, qf[u][f], z[u][t]);
                        mma<T, DP>(vf, df[u][f], dp[u]);
                    }
                }
#pragma unroll
                for (int u = 0; u < NQ; ++u) {
                    masked_logits(z[u][t], a.scale, bias_row[u], j + r0 + 4 * q4, a.Nk, keys);
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float p = __builtin_amdgcn_exp2f(fmaf(z[u][t][r], kLog2e, -lse[u]));
                        z[u][t][r] = p * (dp[u][r] - delta[u]);
                    }
                }
            }
            Frag<T> zf[NQ];
#pragma unroll
            for (int u = 0; u < NQ; ++u) zf[u] = frag_scores<T>(z[u]);
#pragma unroll
            for (int t = 0; t < DT; ++t) {
                const Frag<T> kf = frag_turned<T, DP>(ks, c * S::CHUNK, 16 * t);
#pragma unroll
                for (int u = 0; u < NQ; ++u) mma_rows<T>(kf, zf[u], acc[u][t]);
            }
        }
    }
#pragma unroll
    for (int u = 0; u < NQ; ++u) {
        if (qi[u] >= a.Nq) continue;
        T *row = reinterpret_cast<T *>(a.dq) + ((b * a.Nq + qi[u]) * a.H + head[u]) * (int64_t)a.D;
#pragma unroll
        for (int t = 0; t < DT; ++t)
            if (16 * t + 4 * q4 < a.D) {
                f32x4 v = acc[u][t];
#pragma unroll
                for (int r = 0; r < 4; ++r) v[r] *= a.scale;
                store4<T>(row + 16 * t + 4 * q4, v);
            }
    }
}

// ---- backward: dk and dv -----------------------------------------------------------------------------------------------------
// A wave owns NK x 16 keys (one per lane of a row of 16) and walks all rows of the sharing heads.
template <typename T, int DP, int WAVES, int NK>
__global__ __launch_bounds__(64 * WAVES) void dot_bwd_kv_kernel(DotArgs a) {
    using S = Shape<T, DP>;
    using TL = Tiles<T, DP>;
    constexpr int QT = TL::KT, DT = TL::DT, KEYS = WAVES * NK * 16;
    __shared__ __attribute__((aligned(16))) char lds[TL::LDS];
    __shared__ __attribute__((aligned(16))) float lses[QT], deltas[QT];
    char *qs = lds, *ds = lds + QT * S::PAD;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 15, q4 = lane >> 4;
    const DotBlock blk = dot_block(a);
    const int64_t b = blk.b;
    const int keys = graph_size(a.key_sizes, b, a.Nk), queries = graph_size(a.query_sizes, b, a.Nq);
    const int rows = queries * a.group;
    int key[NK];
    Frag<T> kf[NK][S::FRAGS], vf[NK][S::FRAGS];
    f32x4 dk[NK][DT], dv[NK][DT];
#pragma unroll
    for (int u = 0; u < NK; ++u) {
        key[u] = blk.tile * KEYS + (wave * NK + u) * 16 + n;
        const bool live = key[u] < keys;
        const int64_t j = live ? key[u] : 0;
        const T *krow = reinterpret_cast<const T *>(a.k.p) + b * a.k.batch + j * a.k.node + blk.hk * a.k.head;
        const T *vrow = reinterpret_cast<const T *>(a.v.p) + b * a.v.batch + j * a.v.node + blk.hk * a.v.head;
#pragma unroll
        for (int c = 0; c < S::FRAGS; ++c) {
            const int e = c * S::KD + q4 * (S::PIECE / (int)sizeof(T));
            kf[u][c] = row_piece<T, DP>(krow, e, a.D, live);
            vf[u][c] = row_piece<T, DP>(vrow, e, a.D, live);
        }
#pragma unroll
        for (int t = 0; t < DT; ++t) dk[u][t] = dv[u][t] = (f32x4){0.f, 0.f, 0.f, 0.f};
    }
    Stage<T, DP, QT, 64 * WAVES> st;
    float next_lse = 0.f, next_delta = 0.f;
    auto fetch = [&](int r0) {
        st.load(a.q, a.d_o, rows - r0, a.D, [&](const DotRows &x, int r) {
            const int row = r0 + r, i = row / a.group;
            return b * x.batch + (int64_t)i * x.node + (blk.hk * a.group + row - i * a.group) * x.head;
        });
        if (threadIdx.x < QT) {
            const int row = r0 + threadIdx.x, i = row / a.group;
            const bool ok = row < rows;
            const int64_t at = (b * a.H + blk.hk * a.group + row - i * a.group) * a.Nq + i;
            next_lse = ok ? a.lse[at] : INFINITY;
            next_delta = ok ? a.delta[at] : 0.f;
        }
    };
    if (rows > 0) fetch(0);
    for (int r0 = 0; r0 < rows; r0 += QT) {
        __syncthreads();
        st.store(qs, ds);
        if (threadIdx.x < QT) {
            lses[threadIdx.x] = next_lse;
            deltas[threadIdx.x] = next_delta;
        }
        __syncthreads();
        if (r0 + QT < rows) fetch(r0 + QT);
#pragma unroll
        for (int c = 0; c < QT / S::CHUNK; ++c) {
            f32x4 p[NK][S::CHUNK / 16], z[NK][S::CHUNK / 16];
#pragma unroll
            for (int t = 0; t < S::CHUNK / 16; ++t) {
                const int s0 = c * S::CHUNK + 16 * t;
                f32x4 dp[NK];
#pragma unroll
                for (int u = 0; u < NK; ++u) z[u][t] = dp[u] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int f = 0; f < S::FRAGS; ++f) {
                    const int at = (s0 + n) * S::PAD + f * 4 * S::PIECE + q4 * S::PIECE;
                    const Frag<T> qf = frag_load<T, DP>(qs + at), df = frag_load<T, DP>(ds + at);
#pragma unroll
                    for (int u = 0; u < NK; ++u) {
                        mma<T, DP>(qf, kf[u][f], z[u][t]);
                        mma<T, DP>(df, vf[u][f], dp[u]);
                    }
                }
                const f32x4 lse = *reinterpret_cast<const f32x4 *>(&lses[s0 + 4 * q4]), delta = *reinterpret_cast<const f32x4 *>(&deltas[s0 + 4 * q4]);
#pragma unroll
                for (int u = 0; u < NK; ++u)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int row = r0 + s0 + 4 * q4 + r;
                        bool seen = key[u] < keys && row < rows;
                        float zz = z[u][t][r] * a.scale;
                        if (a.bias && seen) {
                            const float bv = a.bias[b * a.bias_batch + (int64_t)(row / a.group) * a.bias_row + key[u]];
                            seen = bv > kAttended;
                            zz = fmaf(z[u][t][r], a.scale, bv);
                        }
                        const float pv = seen ? __builtin_amdgcn_exp2f(fmaf(zz, kLog2e, -lse[r])) : 0.f;
                        p[u][t][r] = pv;
                        z[u][t][r] = pv * (dp[u][r] - delta[r]);
                    }
            }
            Frag<T> pf[NK], zf[NK];
#pragma unroll
            for (int u = 0; u < NK; ++u) {
                pf[u] = frag_scores<T>(p[u]);
                zf[u] = frag_scores<T>(z[u]);
            }
#pragma unroll
            for (int t = 0; t < DT; ++t) {
                const Frag<T> df = frag_turned<T, DP>(ds, c * S::CHUNK, 16 * t), qf = frag_turned<T, DP>(qs, c * S::CHUNK, 16 * t);
#pragma unroll
                for (int u = 0; u < NK; ++u) {
                    mma_rows<T>(df, pf[u], dv[u][t]);
                    mma_rows<T>(qf, zf[u], dk[u][t]);
                }
            }
        }
    }
#pragma unroll
    for (int u = 0; u < NK; ++u) {
        if (key[u] >= a.Nk) continue;
        const int64_t at = ((b * a.Nk + key[u]) * a.Hkv + blk.hk) * (int64_t)a.D;
#pragma unroll
        for (int t = 0; t < DT; ++t)
            if (16 * t + 4 * q4 < a.D) {
                f32x4 v = dk[u][t];
#pragma unroll
                for (int r = 0; r < 4; ++r) v[r] *= a.scale;
                store4<T>(reinterpret_cast<T *>(a.dk) + at + 16 * t + 4 * q4, v);
                store4<T>(reinterpret_cast<T *>(a.dv) + at + 16 * t + 4 * q4, dv[u][t]);
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

// Rows per block: four waves of 32 rows, of 16 where that leaves most of a block idle, one wave of 16 for the rows of single queries.
static int dot_rows_per_block(int64_t rows) { return rows <= 16 ? 16 : (rows <= 64 ? 64 : 128); }

// Key ranges of a forward launch: enough blocks for every compute unit twice, ranges of 256 keys or more.
static int dot_splits(int64_t B, int64_t rows, int32_t Hkv, int32_t Nk) {
    const int per = dot_rows_per_block(rows);
    const int64_t blocks = B * Hkv * ((rows + per - 1) / per);
    if (blocks >= 512 || Nk < 512) return 1;
    return (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(kSplitsMax, Nk / 256), (1024 + blocks - 1) / std::max<int64_t>(1, blocks)));
}

}  // namespace gatmi

using namespace gatmi;

extern "C" size_t gatmi_dot_attn_fwd_ws_floats(int64_t B, int32_t Nq, int32_t Nk, int32_t H, int32_t Hkv, int32_t D) {
    if (B <= 0 || Nq <= 0 || Nk <= 0 || H <= 0 || Hkv <= 0 || H % Hkv || D <= 0) return 0;
    const int64_t rows = (int64_t)Nq * (H / Hkv);
    const int splits = dot_splits(B, rows, Hkv, Nk);
    return splits == 1 ? 0 : (size_t)B * Hkv * rows * splits * (D + 2);
}

template <typename T, int DP>
static int dot_fwd_run(DotArgs a, int64_t B, hipStream_t st) {
    const int64_t rows = (int64_t)a.Nq * a.group;
    const int per = dot_rows_per_block(rows);
    a.tiles = (int)((rows + per - 1) / per);
    const int64_t per_graph = (int64_t)a.tiles * a.Hkv * a.splits;
    GATMI_REQUIRE(per_graph <= kDotBlocks, GATMI_ERANGE, "dot_attn_fwd: %lld blocks for one graph", (long long)per_graph);
    const int64_t step = a.splits > 1 ? B : kDotBlocks / per_graph;              // split launches are small by construction
    for (int64_t b0 = 0; b0 < B; b0 += step) {
        const int64_t now = std::min(step, B - b0);
        a.b0 = b0;
        const dim3 grid((unsigned)(per_graph * now));
#define RUN(w, nq)                                                                                                                 \
    do {                                                                                                                           \
        if (a.splits > 1) hipLaunchKernelGGL((dot_fwd_kernel<T, DP, w, nq, true>), grid, dim3(64 * w), 0, st, a);                  \
        else hipLaunchKernelGGL((dot_fwd_kernel<T, DP, w, nq, false>), grid, dim3(64 * w), 0, st, a);                              \
    } while (0)
        if (per == 16) RUN(1, 1);
        else if (per == 64) RUN(4, 1);
        else RUN(4, 2);
#undef RUN
    }
    if (a.splits > 1) {
        a.b0 = 0;
        const int64_t total = B * a.Hkv * rows * a.D;
        hipLaunchKernelGGL((dot_join_kernel<T>), dim3((unsigned)std::min<int64_t>(4096, (total + 255) / 256)), dim3(256), 0, st, a, total);
    }
    GATMI_LAUNCH_CHECK("dot_attn_fwd");
    return GATMI_OK;
}

#define GATMI_DOT_DISPATCH(RUN)                                                                    \
    if (dtype == GATMI_DTYPE_F32) {                                                                \
        if (D <= 8) return RUN(float, 8);                                                          \
        if (D <= 16) return RUN(float, 16);                                                        \
        if (D <= 32) return RUN(float, 32);                                                        \
        if (D <= 64) return RUN(float, 64);                                                        \
        return RUN(float, 128);                                                                    \
    }                                                                                              \
    if (D <= 16) return RUN(uint16_t, 16);                                                         \
    if (D <= 32) return RUN(uint16_t, 32);                                                         \
    if (D <= 64) return RUN(uint16_t, 64);                                                         \
    return RUN(uint16_t, 128);

extern "C" int gatmi_dot_attn_fwd(int64_t B, int32_t Nq, int32_t Nk, int32_t H, int32_t Hkv, int32_t D, int32_t dtype, const void *q, const int64_t *q_stride,
                                  const void *k, const int64_t *k_stride, const void *v, const int64_t *v_stride, const float *bias, int64_t bias_batch,
                                  int64_t bias_row, const int32_t *key_sizes, const int32_t *query_sizes, float scale, void *out, float *lse, float *ws, void *stream) {
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
    a.out = out; a.lse = lse; a.bias = Nk > 0 ? bias : nullptr; a.bias_batch = bias_batch; a.bias_row = bias_row;
    a.key_sizes = key_sizes; a.query_sizes = query_sizes; a.scale = scale;
    a.Nq = Nq; a.Nk = Nk; a.H = H; a.Hkv = Hkv; a.group = H / Hkv; a.D = D;
    const int64_t rows = (int64_t)Nq * a.group;
    a.splits = dot_splits(B, rows, Hkv, Nk);
    a.split_keys = a.splits > 1 ? ((Nk + a.splits - 1) / a.splits + 63) / 64 * 64 : Nk;
    if (a.splits > 1) {
        GATMI_REQUIRE(ws, GATMI_EINVAL, "dot_attn_fwd: workspace is null");
        GATMI_REQUIRE_ALIGNED(ws);
        a.part_o = ws;
        a.part_ml = ws + (size_t)B * Hkv * rows * a.splits * D;
    }
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
#define RUN(T, dp) dot_fwd_run<T, dp>(a, B, st)
    GATMI_DOT_DISPATCH(RUN)
#undef RUN
}

template <typename T, int DP>
static int dot_bwd_run(DotArgs a, int64_t B, hipStream_t st) {
    const int64_t rows = (int64_t)a.Nq * a.group;
    constexpr int NQ = (sizeof(T) == 4 && DP == 128) ? 1 : 2, NK = DP == 128 ? 1 : 2;      // registers: two row tiles per wave where the accumulators leave room
    for (int pass = 0; pass < 2; ++pass) {
        const bool wide = pass == 0 ? rows > 64 : a.Nk > 64;
        const int per = pass == 0 ? (wide ? 64 * NQ : 64) : (wide ? 64 * NK : 64);
        const int64_t count = pass == 0 ? rows : a.Nk;
        if (count == 0) continue;
        a.tiles = (int)((count + per - 1) / per);
        a.splits = 1;
        const int64_t per_graph = (int64_t)a.tiles * a.Hkv;
        GATMI_REQUIRE(per_graph <= kDotBlocks, GATMI_ERANGE, "dot_attn_bwd: %lld blocks for one graph", (long long)per_graph);
        const int64_t step = kDotBlocks / per_graph;
        for (int64_t b0 = 0; b0 < B; b0 += step) {
            a.b0 = b0;
            const dim3 grid((unsigned)(per_graph * std::min(step, B - b0)));
            if (pass == 0) {
                if (wide) hipLaunchKernelGGL((dot_bwd_q_kernel<T, DP, 4, NQ>), grid, dim3(256), 0, st, a);
                else hipLaunchKernelGGL((dot_bwd_q_kernel<T, DP, 4, 1>), grid, dim3(256), 0, st, a);
            } else {
                if (wide) hipLaunchKernelGGL((dot_bwd_kv_kernel<T, DP, 4, NK>), grid, dim3(256), 0, st, a);
                else hipLaunchKernelGGL((dot_bwd_kv_kernel<T, DP, 4, 1>), grid, dim3(256), 0, st, a);
            }
        }
    }
    GATMI_LAUNCH_CHECK("dot_attn_bwd");
    return GATMI_OK;
}

extern "C" int gatmi_dot_attn_bwd(int64_t B, int32_t Nq, int32_t Nk, int32_t H, int32_t Hkv, int32_t D, int32_t dtype, const void *q, const int64_t *q_stride,
                                  const void *k, const int64_t *k_stride, const void *v, const int64_t *v_stride, const void *out, const void *dout,
                                  const int64_t *dout_stride, const float *lse, const float *bias, int64_t bias_batch, int64_t bias_row,
                                  const int32_t *key_sizes, const int32_t *query_sizes, float scale, void *dq, void *dk, void *dv, float *delta, void *stream) {
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
    a.dq = dq; a.dk = dk; a.dv = dv; a.lse = const_cast<float *>(lse); a.delta = delta;
    a.bias = Nk > 0 && Nq > 0 ? bias : nullptr; a.bias_batch = bias_batch; a.bias_row = bias_row;
    a.key_sizes = key_sizes; a.query_sizes = query_sizes; a.scale = scale;
    a.Nq = Nq; a.Nk = Nk; a.H = H; a.Hkv = Hkv; a.group = H / Hkv; a.D = D;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
#define RUN(T, dp) dot_bwd_run<T, dp>(a, B, st)
    GATMI_DOT_DISPATCH(RUN)
#undef RUN
}
