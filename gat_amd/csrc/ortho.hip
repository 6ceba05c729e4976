// Orthogonalised updates: `steps` Newton-Schulz steps X <- a X + b (X X^T) X + c (X X^T)^2 X of every matrix of a batch,
// from X = x / (|x|_F + eps).  Each step applies the odd polynomial a s + b s^3 + c s^5 to the singular values.
//
// The polynomial's slope at 0 is a, so what a step rounds off in the directions of small singular values is multiplied by
// a in every step that follows (3.44^5 = 485 for the usual coefficients): with 16-bit operands five steps leave errors
// of 2 to 10 %.  Two ways keep fp32's accuracy, by the length n of the shorter side:
//
// n <= 64 and more than 128 long (`narrow`): with G = X^T X (n x n; the longer side is summed over), all factors are polynomials in G and
//   commute: the result is X Q(G) with an n x n matrix Q.  Three launches: G, Q, X Q, whatever the longer side.  Squaring the
//   singular values doubles the digits that small ones need, so G, Q and the last product are formed in fp64 on
//   v_mfma_f64_16x16x4_f64 (128 flop / clock / CU): for n <= 64 they are small.  |x|_F is the root of G's trace.
//
// Otherwise the steps themselves, three products each, on the 16-bit matrix instructions at fp32 accuracy: an
//   operand v is kept as hi + lo, two fp16 numbers of 11 bits each, and hi hi + hi lo + lo hi is summed in fp32 (relative error 2^-22;
//   the missing lo lo is below it).  fp16 has few exponent bits, but the iteration bounds its operands: entries of X, X X^T and of the
//   polynomial are below kMaxEntry (checked on the host for the given coefficients), so that one fixed scale
//   2^13 keeps hi in range and lo of every entry that matters above the subnormals: an entry is kept to 2^-22 of itself or 2^-38 of
//   |X|_F, whichever is larger.  Where |x|_F is not far above eps, X is tiny: it is
//   then kept times 2^e with e falling from step to step as X can grow (NsShift).  3 products at 16 times the rate of fp32's.
//   `small` (n <= 64, at most 128 long): all steps in one block's LDS, one launch.  `wide` (n > 64): a launch per product; X X^T and its square
//   are symmetric: only tiles on and above the diagonal are formed, each is stored twice.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "common.h"
#include "device_common.h"

namespace gatmi {

typedef double f64x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));

constexpr int kNarrow = 64;
constexpr int kGramParts = 256;              // partial sums of G per matrix, at most
constexpr int kMaxSteps = 32;
constexpr int64_t kBatchAtOnce = 32768;      // matrices of one set of launches (grid.y, grid.z)
constexpr int64_t kMaxSide = 1 << 20;        // of a wide matrix
constexpr float kPlaneScale = 8192.f;        // 2^13
constexpr double kMaxEntry = 7.5;            // kPlaneScale * kMaxEntry < 65504

struct NsMatrix {                            // the batch as given: element (i, j) of matrix b at x + b * batch + i * row + j
    const void *x;
    void *out;
    int64_t x_batch, x_row, out_batch, out_row;
    int64_t m, n;
};

template <typename T>
__device__ __forceinline__ float ns_load(const T *p) {
    if constexpr (sizeof(T) == 4) return *reinterpret_cast<const float *>(p);
    else return __uint_as_float((uint32_t)*reinterpret_cast<const uint16_t *>(p) << 16);
}
template <typename T>
__device__ __forceinline__ void ns_store(T *p, float v) {
    if constexpr (sizeof(T) == 4) *reinterpret_cast<float *>(p) = v;
    else *reinterpret_cast<uint16_t *>(p) = (uint16_t)pack_bf16x2(v, 0.f);
}

// ---- narrow ------------------------------------------------------------------------------------------------------------
// S = index along the short side (0..n), L = along the long side.  TALL: the long side is the row of x.
template <typename T, bool TALL>
__device__ __forceinline__ int64_t ns_at(int64_t row, int64_t s, int64_t l) {
    return TALL ? l * row + s : s * row + l;
}

struct NarrowArgs {
    NsMatrix a;
    int n;                     // short side
    int64_t len;               // long side
    int parts;
    int64_t per_part;          // a multiple of 16
    double *gram;              // [batch][parts][np * np], upper tiles
    double *q;                 // [batch][np * np]
    int steps;
    double ca, cb, cc, eps;
};

// One wave per part of the long side: all upper tiles of G in registers, each loaded value is both operands.
template <typename T, bool TALL, int TILES>
__global__ __launch_bounds__(64) void ns_gram_kernel(NarrowArgs a) {
    constexpr int NP = 16 * TILES;
    const int lane = threadIdx.x, i = lane & 15, kq = lane >> 4;
    const T *x = reinterpret_cast<const T *>(a.a.x) + (int64_t)blockIdx.y * a.a.x_batch;
    const int64_t l0 = blockIdx.x * a.per_part, l1 = min(a.len, l0 + a.per_part);
    f64x4 acc[TILES][TILES];
#pragma unroll
    for (int p = 0; p < TILES; ++p)
#pragma unroll
        for (int q = p; q < TILES; ++q) acc[p][q] = (f64x4){0, 0, 0, 0};
    for (int64_t l = l0; l < l1; l += 16) {
        float v[TILES][4];
#pragma unroll
        for (int p = 0; p < TILES; ++p)
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const int64_t at = l + 4 * kq + t;                // slot kq of product t: any order of the sum, the same for both operands
                const int s = 16 * p + i;
                v[p][t] = s < a.n && at < l1 ? ns_load<T>(x + ns_at<T, TALL>(a.a.x_row, s, at)) : 0.f;
            }
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int p = 0; p < TILES; ++p)
#pragma unroll
                for (int q = p; q < TILES; ++q)
                    acc[p][q] = __builtin_amdgcn_mfma_f64_16x16x4f64((double)v[p][t], (double)v[q][t], acc[p][q], 0, 0, 0);
    }
    double *g = a.gram + ((size_t)blockIdx.y * a.parts + blockIdx.x) * (NP * NP);
#pragma unroll
    for (int p = 0; p < TILES; ++p)
#pragma unroll
        for (int q = p; q < TILES; ++q)
#pragma unroll
            for (int r = 0; r < 4; ++r) g[(16 * p + kq + 4 * r) * NP + 16 * q + i] = acc[p][q][r];      // C: row kq + 4 r, column i
}

// C = A B for symmetric commuting A and B in LDS: the waves share the upper tiles, results stay in registers
// until every wave has read its operands.
template <int TILES>
struct NsProduct {
    static constexpr int NP = 16 * TILES, LD = NP + 2, COUNT = TILES * (TILES + 1) / 2, WAVES = TILES <= 2 ? 4 : 8, THREADS = 64 * WAVES;
    static constexpr int PER = (COUNT + WAVES - 1) / WAVES;
    f64x4 acc[PER];
    __device__ static void tile(int t, int &p, int &q) {
        p = 0;
        while (t >= TILES - p) { t -= TILES - p; ++p; }
        q = p + t;
    }
    __device__ __forceinline__ void multiply(const double *A, const double *B) {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, kq = lane >> 4;
#pragma unroll
        for (int u = 0; u < PER; ++u) {
            acc[u] = (f64x4){0, 0, 0, 0};
            const int t = wave + u * WAVES;
            if (t < COUNT) {
                int p, q;
                tile(t, p, q);
                const double *ar = A + (16 * p + i) * LD + kq, *br = B + (16 * q + i) * LD + kq;        // B symmetric: its column is its row
#pragma unroll
                for (int k = 0; k < NP; k += 4) acc[u] = __builtin_amdgcn_mfma_f64_16x16x4f64(ar[k], br[k], acc[u], 0, 0, 0);
                // the wait states before the first other reader, which comes behind a branch, taken here (see settle in dot_attn.hip)
                asm volatile("s_nop 15\n\ts_nop 3" : "+v"(acc[u]));
            }
        }
    }
    // C_ij = alpha acc_ij + beta D_ij + diag, written to both halves
    __device__ __forceinline__ void store(double *C, double alpha, double beta, const double *D, double diag) const {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, kq = lane >> 4;
#pragma unroll
        for (int u = 0; u < PER; ++u) {
            const int t = wave + u * WAVES;
            if (t < COUNT) {
                int p, q;
                tile(t, p, q);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int row = 16 * p + kq + 4 * r, col = 16 * q + i;
                    if (row <= col) {                             // of a tile on the diagonal only one half is stored, to both places
                        double v = alpha * acc[u][r];
                        if (D) v += beta * D[row * LD + col];
                        if (row == col) v += diag;
                        C[row * LD + col] = v;
                        C[col * LD + row] = v;
                    }
                }
            }
        }
    }
};

// Q of one matrix per block: P_k = a I + b A_k + c A_k^2, Q = P_0 P_1 ..., A_{k+1} = A_k P_k^2, from A_0 = G / (|x|_F + eps)^2.
// The scale of x goes into Q.
template <int TILES>
__global__ __launch_bounds__(NsProduct<TILES>::THREADS) void ns_poly_kernel(NarrowArgs a) {
    using Product = NsProduct<TILES>;
    constexpr int NP = Product::NP, LD = Product::LD, THREADS = Product::THREADS;
    extern __shared__ double lds[];
    double *A = lds, *P = A + NP * LD, *Q = P + NP * LD;
    const double *g = a.gram + (size_t)blockIdx.x * a.parts * (NP * NP);
    for (int e = threadIdx.x; e < NP * NP; e += THREADS) {
        const int row = e / NP, col = e % NP;
        const int up = row / 16 <= col / 16 ? e : col * NP + row;          // tiles below the diagonal are not formed
        double s = 0;
#pragma unroll 16
        for (int p = 0; p < a.parts; ++p) s += g[(size_t)p * (NP * NP) + up];
        A[row * LD + col] = s;
    }
    __syncthreads();
    double trace = 0;
#pragma unroll 16
    for (int d = 0; d < NP; ++d) trace += A[d * LD + d];              // zeros behind n
    const double inv = 1.0 / (sqrt(trace) + a.eps);
    __syncthreads();
    for (int e = threadIdx.x; e < NP * NP; e += THREADS) A[e / NP * LD + e % NP] *= inv * inv;
    if (a.steps == 0)
        for (int e = threadIdx.x; e < NP * NP; e += THREADS) Q[e / NP * LD + e % NP] = e / NP == e % NP ? 1.0 : 0.0;
    __syncthreads();
    Product pr;
    for (int step = 0; step < a.steps; ++step) {
        pr.multiply(A, A);
        pr.store(P, a.cc, a.cb, A, a.ca);
        __syncthreads();
        if (step == 0) {
            for (int e = threadIdx.x; e < NP * LD; e += THREADS) Q[e] = P[e];
        } else {
            pr.multiply(Q, P);
            __syncthreads();
            pr.store(Q, 1.0, 0.0, nullptr, 0.0);
        }
        if (step + 1 < a.steps) {
            for (int half = 0; half < 2; ++half) {
                pr.multiply(A, P);
                __syncthreads();
                pr.store(A, 1.0, 0.0, nullptr, 0.0);
                __syncthreads();
            }
        }
        __syncthreads();
    }
    double *q = a.q + (size_t)blockIdx.x * (NP * NP);
    for (int e = threadIdx.x; e < NP * NP; e += THREADS) q[e] = Q[e / NP * LD + e % NP] * inv;
}

// out = X Q, 16 places of the long side per wave
template <typename T, bool TALL, int TILES>
__global__ __launch_bounds__(256) void ns_apply_kernel(NarrowArgs a) {
    constexpr int NP = 16 * TILES, LD = NP + 2;
    extern __shared__ double lds[];
    const double *q = a.q + (size_t)blockIdx.y * (NP * NP);
    for (int e = threadIdx.x; e < NP * NP; e += 256) lds[e / NP * LD + e % NP] = q[e];
    __syncthreads();
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, kq = lane >> 4;
    const T *x = reinterpret_cast<const T *>(a.a.x) + (int64_t)blockIdx.y * a.a.x_batch;
    T *out = reinterpret_cast<T *>(a.a.out) + (int64_t)blockIdx.y * a.a.out_batch;
    for (int64_t l0 = (blockIdx.x * 4 + wave) * (int64_t)16; l0 < a.len; l0 += (int64_t)gridDim.x * 64) {
        float v[TILES][4];
#pragma unroll
        for (int c = 0; c < TILES; ++c)
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const int s = 16 * c + 4 * kq + t;
                v[c][t] = s < a.n && l0 + i < a.len ? ns_load<T>(x + ns_at<T, TALL>(a.a.x_row, s, l0 + i)) : 0.f;
            }
#pragma unroll
        for (int p = 0; p < TILES; ++p) {
            f64x4 acc = {0, 0, 0, 0};
#pragma unroll
            for (int c = 0; c < TILES; ++c)
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    const double qv = lds[(16 * p + i) * LD + 16 * c + 4 * kq + t];
                    // the contiguous direction of `out` lies across the lanes of a row of C
                    acc = TALL ? __builtin_amdgcn_mfma_f64_16x16x4f64((double)v[c][t], qv, acc, 0, 0, 0)
                               : __builtin_amdgcn_mfma_f64_16x16x4f64(qv, (double)v[c][t], acc, 0, 0, 0);
                }
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int64_t l = l0 + (TALL ? kq + 4 * r : i);
                const int s = 16 * p + (TALL ? i : kq + 4 * r);
                if (l < a.len && s < a.n) ns_store<T>(out + ns_at<T, TALL>(a.a.out_row, s, l), (float)acc[r]);
            }
        }
    }
}

// ---- wide --------------------------------------------------------------------------------------------------------------
constexpr int kWT = 128;          // sides are padded to this: rows and columns of the larger tile
constexpr int kWK = 32;           // depth of a step
constexpr int kNormBlocks = 256;  // partial sums of squares per matrix

// A matrix [rows][K] of values (hi + lo) / kPlaneScale: every 32 entries of a row are 32 hi and then their 32 lo, so that a step of depth 32
// reads whole 128-byte lines.
struct Planes {
    _Float16 *p;
    __device__ static __forceinline__ int64_t at(int64_t row, int64_t k, int64_t K) { return row * 2 * K + (k >> 5) * 64 + (k & 31); }
    __device__ __forceinline__ void put(int64_t at, _Float16 hi, _Float16 lo) const { p[at] = hi; p[at + 32] = lo; }
};

struct WideArgs {
    NsMatrix a;
    int64_t n, len;               // short and long side
    int64_t np, lp;               // padded to whole tiles (zeros)
    Planes x, xt, g, p;           // X [np][lp], X^T [lp][np], X X^T and the polynomial [np][np]; per matrix
    Planes xt_new;                // a step's X^T: other blocks still read the old one
    int64_t x_plane, g_plane;     // fp16 numbers of one matrix
    double *norm;                 // [batch][kNormBlocks]
    int32_t *shift;               // [batch]: e of the first step
    float ca, cb, cc;
    double eps;
    int step, growth;             // a step multiplies X by at most 2^growth
    float *parts;                 // sums of pieces of tiles, or null: see ns_piece_kernel
    int batch, workers;           // of the launch with pieces
};

// X is stored times 2^e, e = max(0, e_0 - step growth): |X| 2^e_0 is in [1/2, 1) before the first step where eps makes X small, and
// e_0 = 0 otherwise.
struct NsShift {
    float now, next;
};
__device__ __forceinline__ NsShift ns_shift(const WideArgs &a, int64_t b) {
    const int e0 = a.shift[b];
    return NsShift{ldexpf(1.f, max(0, e0 - a.step * a.growth)), ldexpf(1.f, max(0, e0 - (a.step + 1) * a.growth))};
}

__device__ __forceinline__ void split16(float v, _Float16 &hi, _Float16 &lo) {
    const float s = v * kPlaneScale;
    hi = (_Float16)s;
    lo = (_Float16)(s - (float)hi);
}

// Partial sums of squares: pieces of kNormPiece entries of a row, dealt to the blocks in turn.  VEC: rows start 4 elements aligned.
constexpr int kNormPiece = 4096;
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void ns_norm_kernel(WideArgs a) {
    __shared__ double part[4];
    const T *x = reinterpret_cast<const T *>(a.a.x) + (int64_t)blockIdx.y * a.a.x_batch;
    const int64_t per_row = (a.a.n + kNormPiece - 1) / kNormPiece;
    double s = 0;
    for (int64_t item = blockIdx.x; item < a.a.m * per_row; item += gridDim.x) {
        const int64_t i = item / per_row, j0 = (item - i * per_row) * kNormPiece, j1 = min(a.a.n, j0 + kNormPiece);
        const T *row = x + i * a.a.x_row;
        if constexpr (VEC) {
            const int64_t j4 = j0 + (j1 - j0) / 4 * 4;
#pragma unroll 4
            for (int64_t j = j0 + 4 * (int)threadIdx.x; j < j4; j += 4 * 256) {
                float v[4];
                if constexpr (sizeof(T) == 4) {
                    const float4 u = *reinterpret_cast<const float4 *>(row + j);
                    v[0] = u.x; v[1] = u.y; v[2] = u.z; v[3] = u.w;
                } else {
                    const uint2 u = *reinterpret_cast<const uint2 *>(row + j);
                    v[0] = __uint_as_float(u.x << 16); v[1] = __uint_as_float(u.x & 0xffff0000u);
                    v[2] = __uint_as_float(u.y << 16); v[3] = __uint_as_float(u.y & 0xffff0000u);
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) s += (double)v[k] * (double)v[k];
            }
            for (int64_t j = j4 + threadIdx.x; j < j1; j += 256) {
                const double v = ns_load<T>(row + j);
                s += v * v;
            }
        } else {
#pragma unroll 4
            for (int64_t j = j0 + threadIdx.x; j < j1; j += 256) {
                const double v = ns_load<T>(row + j);
                s += v * v;
            }
        }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) a.norm[blockIdx.y * kNormBlocks + blockIdx.x] = (part[0] + part[1]) + (part[2] + part[3]);
}

// sum over the 256 threads of a block, the same in all of them
__device__ __forceinline__ double block_sum_f64(double s, double *part, int waves) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
    __syncthreads();
    double total = 0;
    for (int w = 0; w < waves; ++w) total += part[w];
    return total;
}

// e of the first step from |X|_F = unit
__device__ __forceinline__ int ns_first_shift(double unit) { return unit > 0.0 && unit < 0.5 ? min(120, -ilogb(unit) - 1) : 0; }

// X and X^T as planes, zero in the padding: 32 x 32 tiles through LDS
template <typename T, bool TALL>
__global__ __launch_bounds__(256) void ns_split_kernel(WideArgs a) {
    __shared__ float tile[32][33];
    __shared__ double part[4];
    const double s = block_sum_f64(a.norm[blockIdx.z * kNormBlocks + threadIdx.x], part, 4);
    double inv = 1.0 / (sqrt(s) + a.eps);
    const double unit = sqrt(s) * inv;                                     // |X|_F
    const int e0 = ns_first_shift(unit);
    if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) a.shift[blockIdx.z] = e0;
    inv = ldexp(inv, e0);
    const T *x = reinterpret_cast<const T *>(a.a.x) + (int64_t)blockIdx.z * a.a.x_batch;
    const int64_t i0 = blockIdx.y * 32ll, j0 = blockIdx.x * 32ll;          // rows and columns of x
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const int64_t rows = TALL ? a.lp : a.np, cols = TALL ? a.np : a.lp;
    Planes straight = TALL ? a.xt : a.x, turned = TALL ? a.x : a.xt;
    straight.p += blockIdx.z * a.x_plane;
    turned.p += blockIdx.z * a.x_plane;
#pragma unroll
    for (int r = 0; r < 32; r += 8) {
        const int64_t i = i0 + ty + r, j = j0 + tx;
        const float v = i < a.a.m && j < a.a.n ? (float)((double)ns_load<T>(x + i * a.a.x_row + j) * inv) : 0.f;
        tile[ty + r][tx] = v;
        _Float16 hi, lo;
        split16(v, hi, lo);
        straight.put(Planes::at(i, j, cols), hi, lo);
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < 32; r += 8) {
        const int64_t j = j0 + ty + r, i = i0 + tx;
        _Float16 hi, lo;
        split16(tile[tx][ty + r], hi, lo);
        turned.put(Planes::at(j, i, rows), hi, lo);
    }
}

// MODE: what becomes of a product.
constexpr int kNsGram = 0, kNsPoly = 1, kNsStep = 2, kNsLast = 3;
// Stages in LDS.  The symmetric products have about one 128 x 128 block to a compute unit: three.  Tiles of 64 are so small that five of two
// blocks fit (five steps in us, with two or three - with five: 512 x 2048: 299 - 293, 1024 x 4096: 546 - 516, 2 x 1024 x 1024: 475 - 454, 256 x 256: 126 - 129).
template <int MODE> constexpr int ns_stages(int tile) { return tile == 64 ? 5 : (MODE == kNsGram || MODE == kNsPoly ? 3 : 2); }
template <int MODE> struct NsMode { static constexpr bool SYM = MODE == kNsGram || MODE == kNsPoly; };

template <int MODE>
__device__ __forceinline__ const _Float16 *ns_left(const WideArgs &a, int64_t b) {
    return MODE == kNsGram ? a.x.p + b * a.x_plane : (MODE == kNsPoly ? a.g.p : a.p.p) + b * a.g_plane;
}
template <int MODE>
__device__ __forceinline__ const _Float16 *ns_right(const WideArgs &a, int64_t b) {
    return MODE == kNsPoly ? a.g.p + b * a.g_plane : (MODE == kNsGram ? a.x.p : a.xt.p) + b * a.x_plane;
}

// acc += U V^T over the depths k0 .. k1 of planes U [WT rows][K], V [WT rows][K] (from k0 on; k1 - k0 a multiple of kWK), a quarter of the
// WT x WT tile per wave.  STAGES of U and V in LDS, rows of 128 bytes, all but one on their way.
template <int WT, int STAGES>
__device__ __forceinline__ void ns_product(const _Float16 *U, const _Float16 *V, int64_t K, int64_t k0, int64_t k1, char *lds, f32x4 (&acc)[WT / 32][WT / 32]) {
    constexpr int WV = WT / 2, F = WV / 16;                                       // a wave's part of the tile, in fragments
    _Float16 (*buf)[2][WT * 2 * kWK] = reinterpret_cast<_Float16 (*)[2][WT * 2 * kWK]>(lds);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    // Rows go straight to LDS, eight a load of 64 lanes x 16 bytes; piece c of row r lies at place c ^ (r / 2 % 8), so that the lanes of a
    // fragment read, which want one piece of 16 rows, find them in different banks.
    const _Float16 *mine = (wave < 2 ? U : V) + (lane >> 3) * 2 * K + ((lane & 7) ^ ((lane >> 4) & 3)) * 8;
    constexpr int LOADS = WT / 16;                                                // of a wave: half of the rows of one operand
    auto stage = [&](int s, int64_t k) {
#pragma unroll
        for (int c = 0; c < LOADS; ++c) {
            const int r0 = ((wave & 1) * LOADS + c) * 8;
            // (r / 2) % 8 of row r0 + lane / 8 is lane / 16 with 4 added for odd r0 / 8
            const _Float16 *src = mine + (int64_t)r0 * 2 * K + 2 * k;
            const int flip = (r0 >> 3) & 1 ? 32 : 0;                              // piece index ^ 4: 32 numbers up or down
            src += flip ? (((lane & 7) ^ ((lane >> 4) & 3)) & 4 ? -32 : 32) : 0;
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)src,
                                             (__attribute__((address_space(3))) void *)(&buf[s][wave >> 1][r0 * 64]), 16, 0, 0);
        }
    };
    // the loads of the other waves have to be in LDS too: each waits for its own (all but those of the stages after the next) before the barrier
    auto arrived = [&](bool all) {
        if (all) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        else asm volatile("s_waitcnt vmcnt(%0)" ::"n"((STAGES - 2) * LOADS) : "memory");
        __syncthreads();
    };
    const int wi = (wave >> 1) * WV, wj = (wave & 1) * WV;
    const int turn = ((lane & 15) >> 1) & 7, row0 = (lane & 15) * 64;
    const int at_hi = row0 + ((lane >> 4) ^ turn) * 8, at_lo = row0 + (((lane >> 4) + 4) ^ turn) * 8;
    constexpr int64_t AHEAD = (STAGES - 1) * kWK;
#pragma unroll
    for (int g = 0; g < STAGES - 1; ++g)
        if (k0 + g * kWK < k1) stage(g, k0 + g * kWK);
    arrived(k0 + AHEAD > k1);
    int s = 0;
    for (int64_t k = k0; k < k1; k += kWK, s = s + 1 == STAGES ? 0 : s + 1) {
        const bool more = k + AHEAD < k1;
        if (more) stage(s == 0 ? STAGES - 1 : s - 1, k + AHEAD);
        f16x8 uh[F], ul[F], vh[F], vl[F];
#pragma unroll
        for (int i = 0; i < F; ++i) {
            const _Float16 *u = &buf[s][0][(wi + 16 * i) * 64], *v = &buf[s][1][(wj + 16 * i) * 64];
            uh[i] = *reinterpret_cast<const f16x8 *>(u + at_hi);
            ul[i] = *reinterpret_cast<const f16x8 *>(u + at_lo);
            vh[i] = *reinterpret_cast<const f16x8 *>(v + at_hi);
            vl[i] = *reinterpret_cast<const f16x8 *>(v + at_lo);
        }
#pragma unroll
        for (int i = 0; i < F; ++i)
#pragma unroll
            for (int j = 0; j < F; ++j)
                acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ul[i], vh[j], acc[i][j], 0, 0, 0);
#pragma unroll
        for (int i = 0; i < F; ++i)
#pragma unroll
            for (int j = 0; j < F; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(uh[i], vl[j], acc[i][j], 0, 0, 0);
#pragma unroll
        for (int i = 0; i < F; ++i)
#pragma unroll
            for (int j = 0; j < F; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(uh[i], vh[j], acc[i][j], 0, 0, 0);
        arrived(!more);
    }
}

// Stores the four results of a lane, rows row .. row + 3 of column col of the product of matrix b.  turn: also where the tile lies mirrored.
template <int MODE, typename T, bool TALL>
__device__ __forceinline__ void ns_finish(const WideArgs &a, int64_t b, const NsShift &sh, int64_t row, int64_t col, f32x4 sum, bool turn) {
    constexpr bool SYM = NsMode<MODE>::SYM;
    constexpr float kInv = 1.0f / (kPlaneScale * kPlaneScale);
    const float unscale = MODE == kNsGram ? kInv / sh.now / sh.now : (MODE == kNsStep ? kInv * (sh.next / sh.now) : (MODE == kNsLast ? kInv / sh.now : kInv));
    float v[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] = sum[r] * unscale;
    if constexpr (MODE == kNsLast) {
        T *out = reinterpret_cast<T *>(a.a.out) + b * a.a.out_batch;
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (row + r < a.n && col < a.len) ns_store<T>(out + ns_at<T, TALL>(a.a.out_row, row + r, col), v[r]);
    } else {
        const Planes C = MODE == kNsGram ? a.g : (MODE == kNsPoly ? a.p : a.x);
        const Planes Ct = MODE == kNsStep ? a.xt_new : C;
        const int64_t off = SYM ? b * a.g_plane : b * a.x_plane, ld = SYM ? a.np : a.lp;
        const int64_t turned = off + Planes::at(col, row, a.np);                   // four consecutive numbers of row `col`
        if constexpr (MODE == kNsPoly) {                                           // a I + b G + c G^2, G symmetric
            const f16x4 gh = *reinterpret_cast<const f16x4 *>(a.g.p + turned), gl = *reinterpret_cast<const f16x4 *>(a.g.p + turned + 32);
#pragma unroll
            for (int r = 0; r < 4; ++r)
                v[r] = a.cc * v[r] + a.cb * (((float)gh[r] + (float)gl[r]) * (1.0f / kPlaneScale)) + (row + r == col ? a.ca : 0.f);
        }
        f16x4 hi, lo;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            _Float16 h, l;
            split16(v[r], h, l);
            hi[r] = h;
            lo[r] = l;
            C.put(off + Planes::at(row + r, col, ld), h, l);
        }
        if (turn) {
            *reinterpret_cast<f16x4 *>(Ct.p + turned) = hi;
            *reinterpret_cast<f16x4 *>(Ct.p + turned + 32) = lo;
        }
    }
}

struct NsTile { int64_t b; int ti, tj; };
__device__ __forceinline__ NsTile ns_tile(int ty, int64_t tile) {         // tiles of a matrix: tj >= ti, row by row
    const int per = ty * (ty + 1) / 2;
    NsTile t;
    t.b = tile / per;
    int r = (int)(tile - t.b * per);
    for (t.ti = 0; r >= ty - t.ti; ++t.ti) r -= ty - t.ti;
    t.tj = t.ti + r;
    return t;
}

// One product, a tile per block.  2048 x 4096: P X in 114 us, 904 TFLOP/s of fp16 products (a large one of the library: 1111).
template <int MODE, int WT, typename T, bool TALL>
__global__ __launch_bounds__(256) void ns_gemm_kernel(WideArgs a) {
    constexpr int WV = WT / 2, F = WV / 16;
    constexpr int STAGES = ns_stages<MODE>(WT);
    extern __shared__ __attribute__((aligned(16))) char ns_lds[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t b = blockIdx.z;
    // Blocks go to the eight dies in turn; each die gets an eighth of the tiles in one piece, ordered by squares of 4 x 4 tiles: the blocks
    // that run together on a die then share rows of U and V in its L2.
    constexpr bool SYM = NsMode<MODE>::SYM;
    const int ty = (int)(a.np / WT), tx = SYM ? ty : (int)(a.lp / WT), sx = (tx + 3) / 4, squares = SYM ? sx * (sx + 1) / 2 : (ty + 3) / 4 * sx, per = squares * 2;
    const int slot = (blockIdx.x & 7) * per + (int)(blockIdx.x >> 3), sq = slot >> 4;
    const NsTile at = SYM ? ns_tile(sx, sq) : NsTile{0, sq / sx, sq % sx};             // of a symmetric result only the upper tiles
    const int ti = at.ti * 4 + ((slot >> 2) & 3), tj = at.tj * 4 + (slot & 3);
    if (ti >= ty || tj >= tx || (SYM && tj < ti)) return;
    const int64_t K = MODE == kNsGram ? a.lp : a.np;
    f32x4 acc[F][F];
#pragma unroll
    for (int i = 0; i < F; ++i)
#pragma unroll
        for (int j = 0; j < F; ++j) acc[i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};
    ns_product<WT, STAGES>(ns_left<MODE>(a, b) + ti * (int64_t)WT * 2 * K, ns_right<MODE>(a, b) + tj * (int64_t)WT * 2 * K, K, 0, K, ns_lds, acc);
    const NsShift sh = ns_shift(a, b);
    const int wi = (wave >> 1) * WV, wj = (wave & 1) * WV, n0 = lane & 15, m0 = (lane >> 4) * 4;       // C: row m0 + r, column n0
#pragma unroll
    for (int i = 0; i < F; ++i)
#pragma unroll
        for (int j = 0; j < F; ++j)
            ns_finish<MODE, T, TALL>(a, b, sh, ti * (int64_t)WT + wi + 16 * i + m0, tj * (int64_t)WT + wj + 16 * j + n0, acc[i][j], !SYM || ti != tj);
}

// ---- symmetric products in pieces -------------------------------------------------------------------------------------------
// A symmetric product has few tiles: 136 of 128 x 128 for 2048 rows, on 256 compute units.  Its steps (tile by tile, depth by depth) are therefore
// cut into as many equal ranges as there are units.  A range crosses at most one border between tiles (there are no more tiles than
// ranges); what it has of each of its two tiles is left as a piece, and ns_join_kernel adds the pieces of a tile in order.  2048 x 4096: 82 + 14 us where a block
// per tile took 119; the square: 45 + 20 and 72.
struct NsRange { int64_t from, to; };               // steps
__host__ __device__ __forceinline__ NsRange ns_range(int64_t total, int workers, int w) { return NsRange{total * w / workers, total * (w + 1) / workers}; }
constexpr int kPieceFloats = 128 * 128;

template <int MODE>
__global__ __launch_bounds__(256) void ns_piece_kernel(WideArgs a) {
    extern __shared__ __attribute__((aligned(16))) char ns_lds[];
    const int per_die = (a.workers + 7) / 8, w = (blockIdx.x & 7) * per_die + (blockIdx.x >> 3);       // neighbours on one die share rows in its L2
    if ((int)(blockIdx.x >> 3) >= per_die || w >= a.workers) return;
    const int ty = (int)(a.np / 128), per = ty * (ty + 1) / 2;
    const int64_t K = MODE == kNsGram ? a.lp : a.np, steps = K / kWK;
    const NsRange range = ns_range(steps * per * a.batch, a.workers, w);
    int64_t at = range.from;
    for (int piece = 0; at < range.to; ++piece) {
        const int64_t tile = at / steps, end = min(range.to, (tile + 1) * steps);
        const NsTile t = ns_tile(ty, tile);
        f32x4 acc[4][4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};
        ns_product<128, 3>(ns_left<MODE>(a, t.b) + t.ti * 128ll * 2 * K, ns_right<MODE>(a, t.b) + t.tj * 128ll * 2 * K, K, (at - tile * steps) * kWK, (end - tile * steps) * kWK, ns_lds, acc);
        float4 *out = reinterpret_cast<float4 *>(a.parts + (2ll * w + piece) * kPieceFloats) + threadIdx.x;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) out[(i * 4 + j) * 256] = make_float4(acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]);
        at = end;
    }
}

// four blocks a tile
template <int MODE>
__global__ __launch_bounds__(256) void ns_join_kernel(WideArgs a) {
    const int ty = (int)(a.np / 128), per = ty * (ty + 1) / 2;
    const int64_t steps = (MODE == kNsGram ? a.lp : a.np) / kWK, total = steps * per * a.batch, tile = blockIdx.x >> 2, from = tile * steps, to = from + steps;
    const int i = blockIdx.x & 3;
    int w = (int)(from * a.workers / total);                             // the range that `from` lies in, or a neighbour of it
    while (w > 0 && ns_range(total, a.workers, w).from > from) --w;
    while (ns_range(total, a.workers, w).to <= from) ++w;
    f32x4 acc[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[j] = (f32x4){0.f, 0.f, 0.f, 0.f};
    for (; w < a.workers; ++w) {
        const NsRange range = ns_range(total, a.workers, w);
        if (range.from >= to) break;
        const float4 *in = reinterpret_cast<const float4 *>(a.parts + (2ll * w + (range.from < from ? 1 : 0)) * kPieceFloats) + threadIdx.x;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float4 v = in[(i * 4 + j) * 256];
            acc[j] += (f32x4){v.x, v.y, v.z, v.w};
        }
    }
    const NsTile t = ns_tile(ty, tile);
    const NsShift sh = ns_shift(a, t.b);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t row = t.ti * 128ll + (wave >> 1) * 64 + 16 * i + (lane >> 4) * 4, col = t.tj * 128ll + (wave & 1) * 64 + (lane & 15);
#pragma unroll
    for (int j = 0; j < 4; ++j) ns_finish<MODE, float, false>(a, t.b, sh, row, col + 16 * j, acc[j], t.ti != t.tj);
}

// ---- small -------------------------------------------------------------------------------------------------------------
// 60 matrices of 64 x 64 in one launch of 16 us, five dependent steps of three small products between barriers: latency.
constexpr int kSmallThreads = 1024;          // 16 waves: one 16 x 16 tile of G and of the polynomial each
constexpr int kSmallLong = 128;

struct SmallArgs {
    NsMatrix a;
    int n, len;                              // short and long side
    int steps, growth;
    float ca, cb, cc;
    double eps;
};

// Planes in LDS: row r of [rows][64 * G] values, 64 at a time as 32 hi, 32 lo, 32 hi, 32 lo; 16 bytes between rows spread the rows of a fragment
// read over the banks.
template <int G>
struct LdsPlanes {
    static constexpr int STRIDE = 128 * G + 8;
    _Float16 *p;
    __device__ __forceinline__ void put(int row, int k, float v) const {
        _Float16 hi, lo;
        split16(v, hi, lo);
        _Float16 *q = p + row * STRIDE + (k >> 5) * 64 + (k & 31);
        q[0] = hi;
        q[32] = lo;
    }
    // hi and lo of the fragment of 16 rows at depth 32 c
    __device__ __forceinline__ void frag(int row0, int c, f16x8 &hi, f16x8 &lo) const {
        const int lane = threadIdx.x & 63;
        const _Float16 *q = p + (row0 + (lane & 15)) * STRIDE + c * 64 + (lane >> 4) * 8;
        hi = *reinterpret_cast<const f16x8 *>(q);
        lo = *reinterpret_cast<const f16x8 *>(q + 32);
    }
};
// acc += U V^T over depth 32 c .. of the rows at u0 and v0
template <int GU, int GV>
__device__ __forceinline__ void small_mma(const LdsPlanes<GU> &U, int u0, const LdsPlanes<GV> &V, int v0, int c, f32x4 &acc) {
    f16x8 uh, ul, vh, vl;
    U.frag(u0, c, uh, ul);
    V.frag(v0, c, vh, vl);
    acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(ul, vh, acc, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(uh, vl, acc, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(uh, vh, acc, 0, 0, 0);
}

// One matrix per block.  LT: the long side in pieces of 64.  A step: G = X X^T, then P = a I + b G + c G^2, then X <- P X; each
// wave keeps its tile of G in registers for the sum of the second product.
template <typename T, bool TALL, int LT>
__global__ __launch_bounds__(kSmallThreads) void ns_small_kernel(SmallArgs a) {
    extern __shared__ __attribute__((aligned(16))) char ns_lds[];
    LdsPlanes<LT> X{reinterpret_cast<_Float16 *>(ns_lds)};
    LdsPlanes<1> Xt{X.p + 64 * LdsPlanes<LT>::STRIDE}, G{Xt.p + 64 * LT * LdsPlanes<1>::STRIDE}, P{G.p + 64 * LdsPlanes<1>::STRIDE};
    __shared__ double part[kSmallThreads / 64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n0 = lane & 15, m0 = (lane >> 4) * 4;
    const T *x = reinterpret_cast<const T *>(a.a.x) + (int64_t)blockIdx.x * a.a.x_batch;
    T *out = reinterpret_cast<T *>(a.a.out) + (int64_t)blockIdx.x * a.a.out_batch;
    constexpr int PER = 64 * 64 * LT / kSmallThreads;
    const int rows = TALL ? a.len : a.n, cols = TALL ? a.n : a.len;
    // thread t holds elements t, t + 1024, ... of the padded matrix, whose rows have W entries
    constexpr int W = TALL ? 64 : 64 * LT;
    float v[PER];
    double s = 0;
#pragma unroll
    for (int u = 0; u < PER; ++u) {
        const int e = threadIdx.x + u * kSmallThreads, i = e / W, j = e % W;
        v[u] = i < rows && j < cols ? ns_load<T>(x + i * a.a.x_row + j) : 0.f;
        s += (double)v[u] * (double)v[u];
    }
    s = block_sum_f64(s, part, kSmallThreads / 64);
    double inv = 1.0 / (sqrt(s) + a.eps);
    const int e0 = ns_first_shift(sqrt(s) * inv);
    inv = ldexp(inv, e0);
#pragma unroll
    for (int u = 0; u < PER; ++u) {
        const int e = threadIdx.x + u * kSmallThreads, i = e / W, j = e % W, sh = TALL ? j : i, lg = TALL ? i : j;
        const float y = (float)((double)v[u] * inv);
        X.put(sh, lg, y);
        Xt.put(lg, sh, y);
    }
    __syncthreads();
    constexpr float kInv = 1.0f / (kPlaneScale * kPlaneScale);
    const int ti = (wave >> 2) * 16, tj = (wave & 3) * 16;
    for (int step = 0; step < a.steps; ++step) {
        const float now = ldexpf(1.f, max(0, e0 - step * a.growth)), next = ldexpf(1.f, max(0, e0 - (step + 1) * a.growth));
        f32x4 g = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < 2 * LT; ++c) small_mma(X, ti, X, tj, c, g);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            g[r] = g[r] * (kInv / now / now);
            G.put(tj + n0, ti + m0 + r, g[r]);                       // G is symmetric: four consecutive entries of row tj + n0
        }
        __syncthreads();
        f32x4 p = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < 2; ++c) small_mma(G, ti, G, tj, c, p);
#pragma unroll
        for (int r = 0; r < 4; ++r) P.put(tj + n0, ti + m0 + r, a.cc * (p[r] * kInv) + a.cb * g[r] + (ti + m0 + r == tj + n0 ? a.ca : 0.f));
        __syncthreads();
        f32x4 y[LT];
#pragma unroll
        for (int u = 0; u < LT; ++u) {
            y[u] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < 2; ++c) small_mma(P, ti, Xt, tj + 64 * u, c, y[u]);
        }
        const bool last = step + 1 == a.steps;
        const float scale = last ? kInv / now : kInv * (next / now);
#pragma unroll
        for (int u = 0; u < LT; ++u)
#pragma unroll
            for (int r = 0; r < 4; ++r) y[u][r] *= scale;
        if (last) {
#pragma unroll
            for (int u = 0; u < LT; ++u)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int i = ti + m0 + r, j = tj + 64 * u + n0;
                    if (i < a.n && j < a.len) ns_store<T>(out + ns_at<T, TALL>(a.a.out_row, i, j), y[u][r]);
                }
        } else {
            __syncthreads();                                         // X^T has been read by all
#pragma unroll
            for (int u = 0; u < LT; ++u)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    X.put(ti + m0 + r, tj + 64 * u + n0, y[u][r]);
                    Xt.put(tj + 64 * u + n0, ti + m0 + r, y[u][r]);
                }
            __syncthreads();
        }
    }
}

// ---- entry points ------------------------------------------------------------------------------------------------------
}  // namespace gatmi

using namespace gatmi;

static int64_t round_up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

static int gram_parts(int64_t batch, int64_t len) {
    const int64_t per_matrix = std::max<int64_t>(1, 512 / std::max<int64_t>(1, batch));
    return (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(kGramParts, per_matrix), (len + 63) / 64));
}

// Largest entry that X, X X^T or the polynomial can reach: |X|_2 <= s with s_0 = 1 and s_{k+1} = max over t in [0, s_k] of
// |a t + b t^3 + c t^5|.  Extremes lie at the ends or where a derivative vanishes: g = t^2 = -b / 2c for the polynomial
// a + b g + c g^2, the roots of a + 3 b g + 5 c g^2 for t times it.
static double ns_bound(int steps, double a, double b, double c) {
    double s = 1.0, worst = 1.0;
    const double disc = 9 * b * b - 20 * a * c, root = std::sqrt(std::max(0.0, disc));
    const double at[4] = {-b / (2 * c), (-3 * b + root) / (10 * c), (-3 * b - root) / (10 * c), -a / (3 * b)};      // the last for c = 0
    for (int k = 0; k < steps; ++k) {
        const double top = s * s;
        auto poly = [&](double g) { return std::fabs(a + b * g + c * g * g); };
        double next = s * poly(top);
        worst = std::max(worst, std::max(poly(0.0), poly(top)));
        for (double g : at)
            if (g > 0.0 && g < top) {                             // false for the quotients by zero
                next = std::max(next, std::sqrt(g) * poly(g));
                worst = std::max(worst, poly(g));
            }
        s = next;
        worst = std::max(worst, std::max(s, s * s));
        if (!(worst < 1e6)) return 1e6;
    }
    return worst;
}

// a step multiplies X by at most 2^this
static int ns_growth(int steps, double a, double b, double c) { return std::max(1, (int)std::ceil(std::log2(ns_bound(steps, a, b, c)))); }

static bool ns_is_small(int64_t s, int64_t l) { return s <= kNarrow && l <= kSmallLong; }

static size_t narrow_ws(int64_t batch, int64_t n, int64_t len) {
    const size_t np = (size_t)round_up(n, 16);
    return 2 * (size_t)batch * (gram_parts(batch, len) + 1) * np * np;
}
static size_t wide_head(int64_t batch) { return 2 * (size_t)batch * kNormBlocks + ((size_t)batch + 3) / 4 * 4; }      // norms and shifts
// Ranges of a symmetric product of depth K, 0: a block per tile.  Writing, reading and joining the pieces takes what 64 steps take (all five steps
// in us, without - with pieces: 1024 x 1024: 348 - 408, 1536 x 1536: 666 - 687, 2048 x 2048: 1063 - 989, 2816 x 2816: 2923 - 2298; long sides: 128 x 512: 120 -
// 155, 512 x 2048: 348 - 320, 2048 x 4096: 1482 - 1319, 90 x 100000: 8879 - 1567).
constexpr int64_t kPieceDepth = 2048;
static int ns_workers(int64_t batch, int64_t np, int64_t K) {
    const int64_t ty = np / 128, tiles = ty * (ty + 1) / 2 * batch;
    if (tiles > 256 || K < kPieceDepth) return 0;
    return (int)std::min<int64_t>(256, tiles * (K / kWK) / 4);                // four steps or more each: no fewer ranges than tiles, none empty
}
static size_t wide_planes(int64_t batch, size_t np, size_t lp) { return wide_head(batch) + (size_t)batch * (3 * np * lp + 2 * np * np); }      // X, X^T twice, G, P: two fp16 a float
static size_t wide_ws(int64_t batch, int64_t n, int64_t len) {
    const int64_t np = round_up(n, kWT), lp = round_up(len, kWT);
    // a last, smaller set of matrices may have pieces where the others have none: it needs less than their planes take
    return wide_planes(batch, (size_t)np, (size_t)lp) + 2 * (size_t)kPieceFloats * std::max(ns_workers(batch, np, lp), ns_workers(batch, np, np));
}

extern "C" size_t gatmi_newton_schulz_ws_floats(int64_t batch, int64_t m, int64_t n) {
    if (batch <= 0 || m <= 0 || n <= 0) return 0;
    const int64_t s = std::min(m, n), l = std::max(m, n);
    if (ns_is_small(s, l)) return 0;
    const int64_t at_once = std::min<int64_t>(batch, kBatchAtOnce);
    return s <= kNarrow ? narrow_ws(at_once, s, l) : wide_ws(at_once, s, l);
}

template <typename T, bool TALL>
static int run_narrow(const NsMatrix &mat, int64_t batch, int steps, double ca, double cb, double cc, double eps, float *ws, hipStream_t st) {
    NarrowArgs a;
    a.a = mat;
    a.n = (int)std::min(mat.m, mat.n);
    a.len = std::max(mat.m, mat.n);
    a.parts = gram_parts(batch, a.len);
    a.per_part = round_up((a.len + a.parts - 1) / a.parts, 16);
    a.steps = steps; a.ca = ca; a.cb = cb; a.cc = cc; a.eps = eps;
    const int tiles = (a.n + 15) / 16, np = 16 * tiles;
    a.gram = reinterpret_cast<double *>(ws);
    a.q = a.gram + (size_t)batch * a.parts * np * np;
    hipError_t e = hipSuccess;
    const unsigned apply = (unsigned)std::min<int64_t>(1024, (a.len + 63) / 64);
#define RUN(t)                                                                                                                              \
    if (tiles == t) {                                                                                                                       \
        const size_t one = (size_t)(16 * t) * (16 * t + 2) * sizeof(double);                                                                \
        hipLaunchKernelGGL((ns_gram_kernel<T, TALL, t>), dim3(a.parts, (unsigned)batch), dim3(64), 0, st, a);                               \
        if (3 * one > 48 * 1024) e = hipFuncSetAttribute(reinterpret_cast<const void *>(&ns_poly_kernel<t>), hipFuncAttributeMaxDynamicSharedMemorySize, (int)(3 * one)); \
        if (e != hipSuccess) return fail(GATMI_EHIP, "newton_schulz: %s", hipGetErrorString(e));                                            \
        hipLaunchKernelGGL((ns_poly_kernel<t>), dim3((unsigned)batch), dim3(NsProduct<t>::THREADS), 3 * one, st, a);                               \
        hipLaunchKernelGGL((ns_apply_kernel<T, TALL, t>), dim3(apply, (unsigned)batch), dim3(256), one, st, a);                             \
    }
    RUN(1) RUN(2) RUN(3) RUN(4)
#undef RUN
    GATMI_LAUNCH_CHECK("newton_schulz");
    return GATMI_OK;
}

// One product.  Tiles of 128, of 64 where those are fewer than kTileBlocks.
constexpr int64_t kTileBlocks = 128;
template <int MODE, typename T, bool TALL>
static int ns_gemm(const WideArgs &a, int64_t batch, hipStream_t st) {
    constexpr bool SYM = NsMode<MODE>::SYM;
    if constexpr (SYM) {
        WideArgs p = a;
        p.batch = (int)batch;
        p.workers = ns_workers(batch, a.np, MODE == kNsGram ? a.lp : a.np);
        if (p.workers) {
            const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(&ns_piece_kernel<MODE>), hipFuncAttributeMaxDynamicSharedMemorySize, 3 * 128 * 256);
            if (e != hipSuccess) return fail(GATMI_EHIP, "newton_schulz: %s", hipGetErrorString(e));
            const int64_t t = a.np / 128;
            hipLaunchKernelGGL((ns_piece_kernel<MODE>), dim3((unsigned)((p.workers + 7) / 8 * 8)), dim3(256), 3 * 128 * 256, st, p);
            hipLaunchKernelGGL((ns_join_kernel<MODE>), dim3((unsigned)(4 * t * (t + 1) / 2 * batch)), dim3(256), 0, st, p);
            return GATMI_OK;
        }
    }
    const int64_t ty = a.np / 128, tx = SYM ? ty : a.lp / 128;
    auto blocks = [&](int64_t w) {
        const int64_t y = (a.np / w + 3) / 4, x = SYM ? y : (a.lp / w + 3) / 4;
        return dim3((unsigned)((SYM ? y * (y + 1) / 2 : y * x) * 16), 1, (unsigned)batch);
    };
    const bool wide = (SYM ? ty * (ty + 1) / 2 : ty * tx) * batch >= kTileBlocks;
    const size_t lds = (size_t)ns_stages<MODE>(wide ? 128 : 64) * (wide ? 128 : 64) * 256;
    auto kernel = wide ? ns_gemm_kernel<MODE, 128, T, TALL> : ns_gemm_kernel<MODE, 64, T, TALL>;
    if (lds > 48 * 1024) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) return fail(GATMI_EHIP, "newton_schulz: %s", hipGetErrorString(e));
    }
    hipLaunchKernelGGL(kernel, blocks(wide ? 128 : 64), dim3(256), lds, st, a);
    return GATMI_OK;
}

template <typename T, bool TALL>
static int run_small(const NsMatrix &mat, int64_t batch, int steps, double ca, double cb, double cc, double eps, hipStream_t st) {
    SmallArgs a;
    a.a = mat;
    a.n = (int)std::min(mat.m, mat.n);
    a.len = (int)std::max(mat.m, mat.n);
    a.steps = steps;
    a.growth = ns_growth(steps, ca, cb, cc);
    a.ca = (float)ca; a.cb = (float)cb; a.cc = (float)cc; a.eps = eps;
    const int lt = a.len <= 64 ? 1 : 2;
    const size_t lds = sizeof(_Float16) * (64 * (128 * lt + 8) + (64 * lt + 128) * (size_t)LdsPlanes<1>::STRIDE);
    auto kernel = lt == 1 ? ns_small_kernel<T, TALL, 1> : ns_small_kernel<T, TALL, 2>;
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (e != hipSuccess) return fail(GATMI_EHIP, "newton_schulz: %s", hipGetErrorString(e));
    hipLaunchKernelGGL(kernel, dim3((unsigned)batch), dim3(kSmallThreads), lds, st, a);
    GATMI_LAUNCH_CHECK("newton_schulz");
    return GATMI_OK;
}

template <typename T, bool TALL>
static int run_wide(const NsMatrix &mat, int64_t batch, int steps, double ca, double cb, double cc, double eps, float *ws, hipStream_t st) {
    WideArgs a;
    a.a = mat;
    a.n = std::min(mat.m, mat.n);
    a.len = std::max(mat.m, mat.n);
    a.np = round_up(a.n, kWT);
    a.lp = round_up(a.len, kWT);
    a.x_plane = 2 * a.np * a.lp;
    a.g_plane = 2 * a.np * a.np;
    a.ca = (float)ca; a.cb = (float)cb; a.cc = (float)cc; a.eps = eps;
    a.growth = ns_growth(steps, ca, cb, cc);
    a.norm = reinterpret_cast<double *>(ws);
    a.shift = reinterpret_cast<int32_t *>(ws + 2 * (size_t)batch * kNormBlocks);
    _Float16 *p = reinterpret_cast<_Float16 *>(ws + wide_head(batch));
    const size_t xs = (size_t)batch * a.x_plane, gs = (size_t)batch * a.g_plane;
    a.x.p = p;
    a.xt.p = p + xs;
    a.xt_new.p = p + 2 * xs;
    a.g.p = p + 3 * xs;
    a.p.p = p + 3 * xs + gs;
    a.parts = ws + wide_planes(batch, (size_t)a.np, (size_t)a.lp);
    const bool vec = mat.x_row % 4 == 0 && mat.x_batch % 4 == 0 && reinterpret_cast<uintptr_t>(mat.x) % (4 * sizeof(T)) == 0;
    if (vec) hipLaunchKernelGGL((ns_norm_kernel<T, true>), dim3(kNormBlocks, (unsigned)batch), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((ns_norm_kernel<T, false>), dim3(kNormBlocks, (unsigned)batch), dim3(256), 0, st, a);
    const int64_t rows = TALL ? a.lp : a.np, cols = TALL ? a.np : a.lp;
    hipLaunchKernelGGL((ns_split_kernel<T, TALL>), dim3((unsigned)(cols / 32), (unsigned)(rows / 32), (unsigned)batch), dim3(256), 0, st, a);
    for (int k = 0; k < steps; ++k) {
        a.step = k;
        if (int rc = ns_gemm<kNsGram, T, TALL>(a, batch, st)) return rc;
        if (int rc = ns_gemm<kNsPoly, T, TALL>(a, batch, st)) return rc;
        if (int rc = k + 1 < steps ? ns_gemm<kNsStep, T, TALL>(a, batch, st) : ns_gemm<kNsLast, T, TALL>(a, batch, st)) return rc;
        std::swap(a.xt, a.xt_new);
    }
    GATMI_LAUNCH_CHECK("newton_schulz");
    return GATMI_OK;
}

extern "C" int gatmi_newton_schulz(int64_t batch, int64_t m, int64_t n, const void *x, int64_t x_batch, int64_t x_row, int32_t dtype, int32_t steps,
                                   double a, double b, double c, double eps, void *out, int64_t out_batch, int64_t out_row, float *ws, void *stream) {
    GATMI_REQUIRE(batch >= 0 && m >= 0 && n >= 0, GATMI_EINVAL, "newton_schulz: batch = %lld, m = %lld, n = %lld", (long long)batch, (long long)m, (long long)n);
    GATMI_REQUIRE(dtype == GATMI_DTYPE_F32 || dtype == GATMI_DTYPE_BF16, GATMI_EINVAL, "newton_schulz: dtype %d", dtype);
    GATMI_REQUIRE(steps >= 1 && steps <= kMaxSteps, GATMI_EINVAL, "newton_schulz: %d steps (1 to %d)", steps, kMaxSteps);
    GATMI_REQUIRE(eps > 0.0 && eps < 1.0, GATMI_EINVAL, "newton_schulz: eps = %g (above 0, below 1)", eps);
    GATMI_REQUIRE(std::isfinite(a) && std::isfinite(b) && std::isfinite(c), GATMI_EINVAL, "newton_schulz: coefficients %g, %g, %g", a, b, c);
    const double worst = ns_bound(steps, a, b, c);
    GATMI_REQUIRE(worst <= kMaxEntry, GATMI_EUNSUPPORTED,
                  "newton_schulz: with a = %g, b = %g, c = %g the iteration can reach %g in %d steps (at most %g): the coefficients do not keep the singular values bounded",
                  a, b, c, worst, steps, kMaxEntry);
    if (batch == 0 || m == 0 || n == 0) return GATMI_OK;
    const bool small = ns_is_small(std::min(m, n), std::max(m, n));
    GATMI_REQUIRE(x && out && (ws || small), GATMI_EINVAL, "newton_schulz: null pointer");
    GATMI_REQUIRE_ALIGNED(ws);
    GATMI_REQUIRE(x_row >= n || m == 1, GATMI_EINVAL, "newton_schulz: row stride %lld below n = %lld", (long long)x_row, (long long)n);
    GATMI_REQUIRE(out_row >= n || m == 1, GATMI_EINVAL, "newton_schulz: row stride %lld of the result below n = %lld", (long long)out_row, (long long)n);
    const bool tall = m > n, narrow = std::min(m, n) <= kNarrow;
    GATMI_REQUIRE(narrow || std::max(m, n) <= kMaxSide, GATMI_ERANGE, "newton_schulz: a side of %lld (at most %lld)", (long long)std::max(m, n), (long long)kMaxSide);
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    const int64_t size = dtype == GATMI_DTYPE_F32 ? 4 : 2;
    for (int64_t b0 = 0; b0 < batch; b0 += kBatchAtOnce) {
        NsMatrix mat{static_cast<const char *>(x) + b0 * x_batch * size, static_cast<char *>(out) + b0 * out_batch * size, x_batch, x_row, out_batch, out_row, m, n};
        const int64_t now = std::min(kBatchAtOnce, batch - b0);
        int rc;
#define RUN(T)                                                                                                                                  rc = small    ? (tall ? run_small<T, true>(mat, now, steps, a, b, c, eps, st) : run_small<T, false>(mat, now, steps, a, b, c, eps, st))            \
         : narrow ? (tall ? run_narrow<T, true>(mat, now, steps, a, b, c, eps, ws, st) : run_narrow<T, false>(mat, now, steps, a, b, c, eps, ws, st))                   : (tall ? run_wide<T, true>(mat, now, steps, a, b, c, eps, ws, st) : run_wide<T, false>(mat, now, steps, a, b, c, eps, ws, st))
        if (dtype == GATMI_DTYPE_F32) RUN(float);
        else RUN(uint16_t);
#undef RUN
        if (rc) return rc;
    }
    return GATMI_OK;
}
