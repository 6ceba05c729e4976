// Learned rows by id: out[t] = scale * table[id_t], and the gradient of the table by sorted ids,
//   dtable[r] = scale * sum over the tokens t with id_t = r of dout[t],
// every row's sum taken in the order of its tokens, in fp32, and rounded once: no float atomics, the same bits every run.
// An id outside [0, rows) stands for padding: a row of zeros, and nothing in the gradient.
//
// Gradient, three steps:
//   1. the ids are sorted with their positions, stably, by a radix sort of 8 bits a pass (as many passes as the row
//      count has bits).  Up to kOneBlock tokens one block does all passes in LDS; beyond, a pass is a histogram, a scan
//      and a scatter over tiles of kTile tokens.  Ranks inside a wave come from ballots (which lanes hold my digit), so
//      equal ids keep their order.
//   2. the sorted tokens are cut into chunks of equal length whatever rows they fall on (a hub's row may own a fifth of all
//      tokens); a lane group walks a chunk and sums runs of equal ids.  A run inside one chunk is finished there, a run that
//      crosses a border leaves partial rows.
//   3. the partial rows of each run that crosses borders are added, in order; rows that no token hit (a bit per row says so) are
//      filled with zeros by the other blocks of the same launch, so that no row of the gradient is written twice.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "common.h"
#include "device_common.h"

namespace gatmi {

constexpr int kSortThreads = 256;
constexpr int kSortRounds = 16;                                   // 64-token rounds of a wave
constexpr int kTile = kSortThreads * kSortRounds;                 // tokens of a block
constexpr int kOneBlock = 4096;                                   // tokens up to which one block sorts in LDS
constexpr int kOneThreads = 1024;
constexpr uint32_t kShortRun = 64;                                // chunks of a run that one lane group adds up
// Tokens a lane group sums.  16 puts four times as many groups to work, 64 leaves a quarter of the partial rows: both kernels together take 11 (16)
// and 26 us (64) for 2708 tokens, 21.8 and 21.5 us for 252 thousand, 1074 and 828 us for four million.
static inline uint32_t embed_chunk(int64_t tokens) { return tokens <= 65536 ? 16 : 64; }

// ---- rows as units: E consecutive elements of T, one load or store ------------------------------------------------
template <typename T, int E> struct UnitBytes { static constexpr int value = (int)sizeof(T) * E; };
template <typename T, int E>
__device__ __forceinline__ void load_unit(const T *p, float (&v)[E]) {
    if constexpr (sizeof(T) == 4) {
        if constexpr (E == 4) {
            const float4 u = *reinterpret_cast<const float4 *>(p);
            v[0] = u.x; v[1] = u.y; v[2] = u.z; v[3] = u.w;
        } else {
            v[0] = *reinterpret_cast<const float *>(p);
        }
    } else {
        if constexpr (E == 8) {
            const uint4 u = *reinterpret_cast<const uint4 *>(p);
            const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[2 * i] = __uint_as_float(w[i] << 16);
                v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
            }
        } else if constexpr (E == 2) {
            const uint32_t w = *reinterpret_cast<const uint32_t *>(p);
            v[0] = __uint_as_float(w << 16);
            v[1] = __uint_as_float(w & 0xffff0000u);
        } else {
            v[0] = __uint_as_float((uint32_t)*reinterpret_cast<const uint16_t *>(p) << 16);
        }
    }
}
template <typename T, int E>
__device__ __forceinline__ void store_unit(T *p, const float (&v)[E]) {
    if constexpr (sizeof(T) == 4) {
        if constexpr (E == 4) *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
        else *reinterpret_cast<float *>(p) = v[0];
    } else {
        if constexpr (E == 8)
            *reinterpret_cast<uint4 *>(p) = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
        else if constexpr (E == 2) *reinterpret_cast<uint32_t *>(p) = pack_bf16x2(v[0], v[1]);
        else *reinterpret_cast<uint16_t *>(p) = (uint16_t)pack_bf16x2(v[0], 0.f);
    }
}

template <int E>
__device__ __forceinline__ void load_unit_f32(const float *p, float (&v)[E]) {
    if constexpr (E % 4 == 0) {
#pragma unroll
        for (int i = 0; i < E; i += 4) {
            const float4 u = *reinterpret_cast<const float4 *>(p + i);
            v[i] = u.x; v[i + 1] = u.y; v[i + 2] = u.z; v[i + 3] = u.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i) v[i] = p[i];
    }
}

template <bool ID64>
__device__ __forceinline__ uint32_t load_key(const void *ids, int64_t t, uint32_t rows) {
    if constexpr (ID64) {
        const int64_t v = reinterpret_cast<const int64_t *>(ids)[t];
        return v >= 0 && v < (int64_t)rows ? (uint32_t)v : rows;      // anything outside: one key behind the last row
    } else {
        const int32_t v = reinterpret_cast<const int32_t *>(ids)[t];
        return v >= 0 && (uint32_t)v < rows ? (uint32_t)v : rows;
    }
}

// ---- lookup ---------------------------------------------------------------------------------------------------------
struct EmbedFwdArgs {
    const void *ids, *table;
    void *out;
    int64_t tokens, ld;
    uint32_t rows, units;           // units of a row
    int tokens_per_block;
    int64_t tiles;                  // runs of tokens_per_block tokens
    float scale;
};

// Bound by memory: 4 million tokens of 100 fp32 in 592 us (1.6 GB written, 32 MB of ids and up to 1 GB of rows read: 4.4 TB/s; a copy: 4.7).
// A block takes tokens_per_block tokens at a time: that part of the output is contiguous, thread i writes units i, i + 256, ...
template <typename T, int E, bool ID64>
__global__ __launch_bounds__(256) void embed_fwd_kernel(EmbedFwdArgs a) {
    const T *table = reinterpret_cast<const T *>(a.table);
    for (int64_t tile = blockIdx.x; tile < a.tiles; tile += gridDim.x) {
        const int64_t t0 = tile * a.tokens_per_block;
        const uint32_t count = (uint32_t)min((int64_t)a.tokens_per_block, a.tokens - t0) * a.units;
        T *out = reinterpret_cast<T *>(a.out) + t0 * (int64_t)a.units * E;
        for (uint32_t e0 = threadIdx.x; e0 < count; e0 += 4 * 256) {
            float v[4][E];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const uint32_t e = e0 + u * 256;
                if (e < count) {
                    const uint32_t t = e / a.units, c = e - t * a.units;
                    const uint32_t key = load_key<ID64>(a.ids, t0 + t, a.rows);
#pragma unroll
                    for (int i = 0; i < E; ++i) v[u][i] = 0.f;
                    if (key < a.rows) load_unit<T, E>(table + (int64_t)key * a.ld + (int64_t)c * E, v[u]);
                }
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const uint32_t e = e0 + u * 256;
                if (e < count) {
#pragma unroll
                    for (int i = 0; i < E; ++i) v[u][i] *= a.scale;
                    store_unit<T, E>(out + (int64_t)e * E, v[u]);
                }
            }
        }
    }
}

// ---- stable radix sort of (key, position) ------------------------------------------------------------------------------
// lanes of the wave whose digit is mine, among the lanes of `valid`
__device__ __forceinline__ uint64_t same_digit(uint32_t digit, uint64_t valid) {
    uint64_t m = valid;
#pragma unroll
    for (int b = 0; b < 8; ++b) {
        const uint64_t w = __ballot((digit >> b) & 1);
        m &= (digit >> b) & 1 ? w : ~w;
    }
    return m;
}

// This wave's `rounds` rounds of 64 tokens: rank of each token among the wave's tokens of its digit; count[] ends as the
// wave's histogram.  Called by whole waves.
template <int ROUNDS>
__device__ __forceinline__ void wave_ranks(const uint32_t (&digit)[ROUNDS], const bool (&valid)[ROUNDS], uint32_t *count, uint32_t (&rank)[ROUNDS]) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        const uint64_t m = same_digit(digit[r], __ballot(valid[r]));
        const int leader = m ? __ffsll((unsigned long long)m) - 1 : lane;
        uint32_t before = 0;
        if (valid[r] && lane == leader) before = atomicAdd(&count[digit[r]], (uint32_t)__popcll(m));      // one lane per digit
        before = __shfl(before, leader, 64);
        rank[r] = before + (uint32_t)__popcll(m & ((1ull << lane) - 1));
    }
}

// exclusive scan of 256 counters by the first 256 threads of a block (all threads call it)
__device__ __forceinline__ uint32_t scan256(uint32_t v, uint32_t *wave_total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t inc = (uint32_t)wave_scan_add((int)v);
    if (threadIdx.x < 256 && lane == 63) wave_total[wave] = inc;
    __syncthreads();
    uint32_t base = 0;
    for (int w = 0; w < wave && w < 4; ++w) base += wave_total[w];
    return base + inc - v;
}

struct SortArgs {
    const void *ids;                     // first pass
    const uint32_t *key_in, *pos_in;     // later passes
    uint32_t *key_out, *pos_out;
    uint32_t *hist;                      // [256][blocks]
    uint32_t *total;                     // [256]
    uint32_t n, rows, blocks;
    int shift;
    uint32_t *bits;                      // cleared by the first histogram
    uint32_t bit_words;
};

template <bool FIRST, bool ID64>
__device__ __forceinline__ uint32_t pass_key(const SortArgs &a, uint32_t t) {
    if constexpr (FIRST) return load_key<ID64>(a.ids, t, a.rows);
    else return a.key_in[t];
}

template <bool FIRST, bool ID64>
__global__ __launch_bounds__(kSortThreads) void sort_hist_kernel(SortArgs a) {
    __shared__ uint32_t h[256];
    h[threadIdx.x] = 0;
    __syncthreads();
    if constexpr (FIRST)
        for (uint32_t w = blockIdx.x * kSortThreads + threadIdx.x; w < a.bit_words; w += a.blocks * kSortThreads) a.bits[w] = 0;
    const uint32_t t0 = blockIdx.x * (uint32_t)kTile;
#pragma unroll
    for (int r = 0; r < kSortRounds; ++r) {
        const uint32_t t = t0 + r * kSortThreads + threadIdx.x;
        const bool ok = t < a.n;
        const uint32_t d = ok ? (pass_key<FIRST, ID64>(a, t) >> a.shift) & 255 : 0;
        const uint64_t m = same_digit(d, __ballot(ok));
        if (ok && (int)(threadIdx.x & 63) == __ffsll((unsigned long long)m) - 1) atomicAdd(&h[d], (uint32_t)__popcll(m));
    }
    __syncthreads();
    a.hist[(size_t)threadIdx.x * a.blocks + blockIdx.x] = h[threadIdx.x];
}

// block d: exclusive scan of digit d's counts over the tiles, and their total
__global__ __launch_bounds__(256) void sort_scan_kernel(SortArgs a) {
    __shared__ uint32_t wave_total[4];
    uint32_t *row = a.hist + (size_t)blockIdx.x * a.blocks;
    uint32_t carry = 0;
    for (uint32_t b0 = 0; b0 < a.blocks; b0 += 256) {
        const uint32_t b = b0 + threadIdx.x;
        const uint32_t v = b < a.blocks ? row[b] : 0;
        const uint32_t before = scan256(v, wave_total);
        if (b < a.blocks) row[b] = carry + before;
        carry += wave_total[0] + wave_total[1] + wave_total[2] + wave_total[3];
        __syncthreads();
    }
    if (threadIdx.x == 0) a.total[blockIdx.x] = carry;
}

template <bool FIRST, bool ID64>
__global__ __launch_bounds__(kSortThreads) void sort_scatter_kernel(SortArgs a) {
    constexpr int WAVES = kSortThreads / 64;
    __shared__ uint32_t count[WAVES][256];
    __shared__ uint32_t wave_total[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int w = 0; w < WAVES; ++w) count[w][threadIdx.x] = 0;
    __syncthreads();
    const uint32_t digit_base = scan256(a.total[threadIdx.x], wave_total);
    const uint32_t t0 = blockIdx.x * (uint32_t)kTile + wave * 64 * kSortRounds;       // a wave's tokens are consecutive
    uint32_t key[kSortRounds], digit[kSortRounds], rank[kSortRounds];
    bool valid[kSortRounds];
#pragma unroll
    for (int r = 0; r < kSortRounds; ++r) {
        const uint32_t t = t0 + r * 64 + lane;
        valid[r] = t < a.n;
        key[r] = valid[r] ? pass_key<FIRST, ID64>(a, t) : 0;
        digit[r] = (key[r] >> a.shift) & 255;
    }
    wave_ranks<kSortRounds>(digit, valid, count[wave], rank);
    __syncthreads();
    {
        uint32_t run = digit_base + a.hist[(size_t)threadIdx.x * a.blocks + blockIdx.x];
        for (int w = 0; w < WAVES; ++w) {
            const uint32_t c = count[w][threadIdx.x];
            count[w][threadIdx.x] = run;
            run += c;
        }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kSortRounds; ++r)
        if (valid[r]) {
            const uint32_t at = count[wave][digit[r]] + rank[r];
            const uint32_t t = t0 + r * 64 + lane;
            a.key_out[at] = key[r];
            a.pos_out[at] = FIRST ? t : a.pos_in[t];
        }
}

// up to kOneBlock tokens: all passes in one block
template <bool ID64>
__global__ __launch_bounds__(kOneThreads) void sort_one_block_kernel(SortArgs a, int passes) {
    constexpr int WAVES = kOneThreads / 64, ROUNDS = kOneBlock / kOneThreads;
    __shared__ uint32_t count[WAVES][256];
    __shared__ uint32_t keys[kOneBlock], poss[kOneBlock];
    __shared__ uint32_t wave_total[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (uint32_t w = threadIdx.x; w < a.bit_words; w += kOneThreads) a.bits[w] = 0;
    for (uint32_t t = threadIdx.x; t < a.n; t += kOneThreads) {
        keys[t] = load_key<ID64>(a.ids, t, a.rows);
        poss[t] = t;
    }
    for (int p = 0; p < passes; ++p) {
        for (int i = threadIdx.x; i < WAVES * 256; i += kOneThreads) (&count[0][0])[i] = 0;
        __syncthreads();
        uint32_t key[ROUNDS], pos[ROUNDS], digit[ROUNDS], rank[ROUNDS];
        bool valid[ROUNDS];
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r) {
            const uint32_t t = wave * 64 * ROUNDS + r * 64 + lane;
            valid[r] = t < a.n;
            key[r] = valid[r] ? keys[t] : 0;
            pos[r] = valid[r] ? poss[t] : 0;
            digit[r] = (key[r] >> (8 * p)) & 255;
        }
        wave_ranks<ROUNDS>(digit, valid, count[wave], rank);
        __syncthreads();
        uint32_t sum = 0;
        if (threadIdx.x < 256)
            for (int w = 0; w < WAVES; ++w) sum += count[w][threadIdx.x];
        uint32_t run = scan256(sum, wave_total);
        if (threadIdx.x < 256)
            for (int w = 0; w < WAVES; ++w) {
                const uint32_t c = count[w][threadIdx.x];
                count[w][threadIdx.x] = run;
                run += c;
            }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r)
            if (valid[r]) {
                const uint32_t at = count[wave][digit[r]] + rank[r];
                keys[at] = key[r];
                poss[at] = pos[r];
            }
        __syncthreads();
    }
    for (uint32_t t = threadIdx.x; t < a.n; t += kOneThreads) {
        a.key_out[t] = keys[t];
        a.pos_out[t] = poss[t];
    }
}

// ---- sums over the sorted tokens --------------------------------------------------------------------------------------
struct SegArgs {
    const uint32_t *key, *pos;
    const void *dout;
    void *dtable;
    float *partial;                      // [chunks][2][width padded to whole units]
    uint32_t *bits;
    int64_t ld;                          // elements between rows of dout
    uint32_t n, rows, units, chunks, chunk;       // chunks of `chunk` tokens
    float scale;
};

template <typename T, int E>
__device__ __forceinline__ void store_scaled(const SegArgs &a, uint32_t row, uint32_t unit, const float (&acc)[E]) {
    float v[E];
#pragma unroll
    for (int i = 0; i < E; ++i) v[i] = acc[i] * a.scale;
    store_unit<T, E>(reinterpret_cast<T *>(a.dtable) + (int64_t)row * a.units * E + (int64_t)unit * E, v);
}

// L lanes per chunk (a power of two), L units of a row at a time (grid.y covers wider rows).  4 million rows of 400 bytes in sorted, that is scattered,
// order: 619 us, 2.6 TB/s read beside the finished rows that it writes; sorting takes 245 us before, joining and filling 207 us after.
template <typename T, int E, int L>
__global__ __launch_bounds__(256) void embed_seg_kernel(SegArgs a) {
    constexpr int GROUPS = 256 / L, BATCH = 8;
    const int sub = threadIdx.x % L;
    const uint32_t chunk = blockIdx.x * GROUPS + threadIdx.x / L;
    const uint32_t unit = blockIdx.y * L + sub;
    if (chunk >= a.chunks) return;
    const bool active = unit < a.units;
    const uint32_t c0 = chunk * a.chunk, c1 = min(a.n, c0 + a.chunk);
    const T *dout = reinterpret_cast<const T *>(a.dout) + (int64_t)(active ? unit : 0) * E;
    const uint32_t before = c0 > 0 ? a.key[c0 - 1] : 0xffffffffu, after = c1 < a.n ? a.key[c1] : 0xffffffffu;
    float acc[E];
#pragma unroll
    for (int i = 0; i < E; ++i) acc[i] = 0.f;
    uint32_t cur = a.key[c0];
    bool first = true;
    auto flush = [&](bool last) {
        if (cur >= a.rows) return;                                           // padding
        const bool from_before = first && cur == before, goes_on = last && cur == after;
        if (!from_before && sub == 0 && blockIdx.y == 0) atomicOr(&a.bits[cur >> 5], 1u << (cur & 31));
        if (!active) return;
        if (!from_before && !goes_on) {
            store_scaled<T, E>(a, cur, unit, acc);
        } else {
            float *p = a.partial + ((size_t)(2 * chunk + (from_before ? 0 : 1)) * a.units + unit) * E;
            if constexpr (E % 4 == 0) {
#pragma unroll
                for (int i = 0; i < E; i += 4) *reinterpret_cast<float4 *>(p + i) = make_float4(acc[i], acc[i + 1], acc[i + 2], acc[i + 3]);
            } else {
#pragma unroll
                for (int i = 0; i < E; ++i) p[i] = acc[i];
            }
        }
    };
    for (uint32_t i0 = c0; i0 < c1; i0 += BATCH) {
        uint32_t k[BATCH];
        float v[BATCH][E];
#pragma unroll
        for (int u = 0; u < BATCH; ++u) {
            const uint32_t i = min(i0 + u, c1 - 1);
            k[u] = a.key[i];
            const uint32_t p = a.pos[i];
            load_unit<T, E>(dout + (int64_t)p * a.ld, v[u]);                  // padding's row is read and not used
        }
#pragma unroll
        for (int u = 0; u < BATCH; ++u) {
            if (i0 + u >= c1) break;
            if (k[u] != cur) {
                flush(false);
                cur = k[u];
                first = false;
#pragma unroll
                for (int i = 0; i < E; ++i) acc[i] = v[u][i];
            } else {
#pragma unroll
                for (int i = 0; i < E; ++i) acc[i] += v[u][i];
            }
        }
    }
    flush(true);
}

// The first fill_blocks blocks fill the rows without a bit with zeros.  In the others a lane group looks at a chunk: where a run starts in
// it and goes on behind it, the group adds its partial rows, or, of a run over more than kShortRun chunks, the block does: its groups
// take consecutive shares, their sums are added in order.  That one block is what a run of most tokens waits for: the gradient of 4 million tokens on one row of
// 100 fp32 takes 1987 us, spread over 2.4 million rows 1042.
template <typename T, int E, int L>
__global__ __launch_bounds__(256) void embed_join_kernel(SegArgs a, uint32_t join_blocks, uint32_t fill_blocks) {
    constexpr int GROUPS = 256 / L;
    __shared__ float sums[GROUPS][L * E];
    __shared__ uint32_t long_runs, long_list[GROUPS];
    if (blockIdx.x < fill_blocks) {
        if (blockIdx.y != 0) return;
        const uint32_t words = (a.rows + 31) / 32;
        float zero[E];
#pragma unroll
        for (int i = 0; i < E; ++i) zero[i] = 0.f;
        // a wave takes a word of bits: its lanes walk the units of those 32 rows and store where the row has no bit
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        for (uint32_t w = blockIdx.x * 4 + wave; w < words; w += fill_blocks * 4) {
            const uint32_t hit = a.bits[w];
            if (hit == 0xffffffffu) continue;
            const uint32_t count = min(32u, a.rows - w * 32) * a.units;
            T *p = reinterpret_cast<T *>(a.dtable) + (int64_t)w * 32 * a.units * E;
            // e / units without a division per unit: the row moves on by 64 / units and a carry
            uint32_t row = (uint32_t)lane / a.units, in = lane - row * a.units;
            const uint32_t whole = 64 / a.units, rest = 64 - whole * a.units;
            for (uint32_t e = lane; e < count; e += 64) {
                if (!(hit >> row & 1)) store_unit<T, E>(p + (int64_t)e * E, zero);
                row += whole;
                in += rest;
                if (in >= a.units) {
                    in -= a.units;
                    ++row;
                }
            }
        }
        return;
    }
    const int sub = threadIdx.x % L, group = threadIdx.x / L;
    const uint32_t unit = blockIdx.y * L + sub;
    float acc[E];
    // partial rows [p0, p1) of the run that starts in `chunk`: its first lies in the second place of that chunk, the others in the first
    // place of theirs
    auto add = [&](uint32_t chunk, uint32_t p0, uint32_t p1) {
#pragma unroll
        for (int i = 0; i < E; ++i) acc[i] = 0.f;
        if (unit >= a.units) return;
        const float *rows = a.partial + ((size_t)(2 * chunk) * a.units + unit) * E;
        const size_t stride = (size_t)2 * a.units * E;
        for (uint32_t p = p0; p < p1; p += 8) {
            float v[8][E];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const uint32_t at = min(p + u, p1 - 1);
                load_unit_f32<E>(rows + at * stride + (at == 0 ? stride / 2 : 0), v[u]);
            }
#pragma unroll
            for (int u = 0; u < 8; ++u)
                if (p + u < p1)
#pragma unroll
                    for (int i = 0; i < E; ++i) acc[i] += v[u][i];
        }
    };
    for (uint32_t base = (blockIdx.x - fill_blocks) * GROUPS; base < a.chunks; base += join_blocks * GROUPS) {
        if (threadIdx.x == 0) long_runs = 0;
        __syncthreads();
        const uint32_t chunk = base + group;
        if (chunk + 1 < a.chunks) {                                              // nothing goes on behind the last chunk
            const uint32_t c0 = chunk * a.chunk, c1 = c0 + a.chunk, run = a.key[c1 - 1];
            // a run that started further ahead belongs to that chunk's group
            if (run < a.rows && a.key[c1] == run && !(a.key[c0] == run && c0 > 0 && a.key[c0 - 1] == run)) {
                uint32_t parts = 2;
                for (uint32_t more = L; more == L && parts <= kShortRun; parts += more) {        // L chunks at a time: how many begin with the run
                    const uint32_t at = chunk + parts + sub;
                    const uint64_t same = __ballot(at < a.chunks && a.key[min(at, a.chunks - 1) * a.chunk] == run) >> (threadIdx.x & 63 & ~(L - 1));
                    const uint64_t differ = ~same & (L == 64 ? ~0ull : (1ull << (L & 63)) - 1);
                    more = differ ? (uint32_t)__ffsll((unsigned long long)differ) - 1 : L;
                }
                if (parts <= kShortRun) {
                    add(chunk, 0, parts);
                    if (unit < a.units) store_scaled<T, E>(a, run, unit, acc);
                } else if (sub == 0) {
                    long_list[atomicAdd(&long_runs, 1u)] = chunk;
                }
            }
        }
        __syncthreads();
        for (uint32_t k = 0; k < long_runs; ++k) {                               // the whole block adds each of the long ones
            const uint32_t first = long_list[k], run = a.key[first * a.chunk + a.chunk - 1];
            // the last chunk whose first key is the run: keys are sorted, so chunks with that property are consecutive
            uint32_t lo = first + 1, hi = a.chunks - 1;
            while (lo < hi) {
                const uint32_t mid = lo + (hi - lo + 1) / 2;
                if (a.key[mid * a.chunk] == run) lo = mid;
                else hi = mid - 1;
            }
            const uint32_t parts = lo - first + 1, share = (parts + GROUPS - 1) / GROUPS;
            add(first, min(parts, group * share), min(parts, (group + 1) * share));
#pragma unroll
            for (int i = 0; i < E; ++i) sums[group][sub * E + i] = acc[i];
            __syncthreads();
            if (group == 0 && unit < a.units) {
                for (int g = 1; g < GROUPS; ++g)
#pragma unroll
                    for (int i = 0; i < E; ++i) acc[i] += sums[g][sub * E + i];
                store_scaled<T, E>(a, run, unit, acc);
            }
            __syncthreads();
        }
        __syncthreads();
    }
}

// no token at all: the whole gradient is zero
template <typename T>
__global__ __launch_bounds__(256) void embed_zero_kernel(T *p, int64_t n) {
    for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) p[i] = T(0);
}

static int check_embed(const char *what, int64_t tokens, int64_t rows, int32_t width, int32_t dtype) {
    GATMI_REQUIRE(tokens >= 0 && rows >= 0 && width >= 1, GATMI_EINVAL, "%s: tokens = %lld, rows = %lld, width = %d", what, (long long)tokens, (long long)rows, width);
    GATMI_REQUIRE(tokens < (1ll << 31) - kTile && rows < (1ll << 31) - 1, GATMI_ERANGE, "%s: %lld tokens / %lld rows do not fit 31 bits", what, (long long)tokens, (long long)rows);
    GATMI_REQUIRE(width <= 65536, GATMI_EUNSUPPORTED, "%s: width %d > 65536", what, width);
    GATMI_REQUIRE(dtype == GATMI_DTYPE_F32 || dtype == GATMI_DTYPE_BF16, GATMI_EINVAL, "%s: dtype %d", what, dtype);
    return GATMI_OK;
}

// elements a lane moves at once: 16 bytes where rows and pointers allow it, then 4, then one element
static int unit_elems(int32_t width, int32_t dtype, int64_t ld, const void *p, const void *q) {
    const int size = dtype == GATMI_DTYPE_F32 ? 4 : 2;
    const uintptr_t low = reinterpret_cast<uintptr_t>(p) | reinterpret_cast<uintptr_t>(q) | (uintptr_t)((int64_t)width * size) | (uintptr_t)(ld * size);
    if ((low & 15) == 0) return 16 / size;
    if ((low & 3) == 0) return 4 / size;
    return 1;
}

static int sort_passes(int64_t rows) {
    int bits = 1;
    while (bits < 32 && (rows >> bits) != 0) ++bits;      // keys 0..rows
    return (bits + 7) / 8;
}

}  // namespace gatmi

using namespace gatmi;

extern "C" int gatmi_embed_fwd(const void *ids, int32_t id_bits, int64_t tokens, const void *table, int64_t ld_table, int64_t rows, int32_t width,
                               int32_t dtype, float scale, void *out, void *stream) {
    if (int rc = check_embed("embed_fwd", tokens, rows, width, dtype)) return rc;
    GATMI_REQUIRE(id_bits == 32 || id_bits == 64, GATMI_EINVAL, "embed_fwd: ids of %d bits", id_bits);
    if (tokens == 0) return GATMI_OK;
    GATMI_REQUIRE(ids && out && (table || rows == 0), GATMI_EINVAL, "embed_fwd: null pointer");
    GATMI_REQUIRE(ld_table >= width || rows <= 1, GATMI_EINVAL, "embed_fwd: row stride %lld below width %d", (long long)ld_table, width);
    const int E = unit_elems(width, dtype, ld_table, table, out);
    EmbedFwdArgs a;
    a.ids = ids; a.table = table; a.out = out; a.tokens = tokens; a.ld = ld_table;
    a.rows = (uint32_t)rows; a.units = (uint32_t)(width / E); a.scale = scale;
    // about four units a thread and block, at least one token
    a.tokens_per_block = (int)std::max<int64_t>(1, 1024 / a.units);
    a.tiles = (tokens + a.tokens_per_block - 1) / a.tokens_per_block;
    const int64_t blocks = std::min<int64_t>(a.tiles, 1 << 20);
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
#define RUN(T, e)                                                                                                                          \
    do {                                                                                                                                   \
        if (id_bits == 64) hipLaunchKernelGGL((embed_fwd_kernel<T, e, true>), dim3((unsigned)blocks), dim3(256), 0, st, a);                \
        else hipLaunchKernelGGL((embed_fwd_kernel<T, e, false>), dim3((unsigned)blocks), dim3(256), 0, st, a);                             \
    } while (0)
    if (dtype == GATMI_DTYPE_F32) {
        if (E == 4) RUN(float, 4); else RUN(float, 1);
    } else {
        if (E == 8) RUN(uint16_t, 8); else if (E == 2) RUN(uint16_t, 2); else RUN(uint16_t, 1);
    }
#undef RUN
    GATMI_LAUNCH_CHECK("embed_fwd");
    return GATMI_OK;
}

// workspace: sorted keys and positions twice, histograms, row bits, partial rows
static void embed_bwd_layout(int64_t tokens, int64_t rows, int32_t width, size_t *hist, size_t *bits, size_t *partial, size_t *total) {
    const size_t n4 = ((size_t)tokens + 3) / 4 * 4;
    const size_t blocks = ((size_t)tokens + kTile - 1) / kTile;
    *hist = 4 * n4;
    *bits = *hist + 256 * blocks + 256;
    *partial = (*bits + ((size_t)rows + 31) / 32 + 3) / 4 * 4;
    *total = *partial + 2 * (((size_t)tokens + embed_chunk(tokens) - 1) / embed_chunk(tokens)) * (size_t)width;
}

extern "C" size_t gatmi_embed_bwd_ws_floats(int64_t tokens, int64_t rows, int32_t width) {
    if (tokens <= 0 || rows <= 0 || width < 1) return 0;
    size_t h, b, p, t;
    embed_bwd_layout(tokens, rows, width, &h, &b, &p, &t);
    return t;
}

extern "C" int gatmi_embed_bwd(const void *ids, int32_t id_bits, int64_t tokens, const void *dout, int64_t ld_dout, int64_t rows, int32_t width,
                               int32_t dtype, float scale, void *dtable, float *ws, void *stream) {
    if (int rc = check_embed("embed_bwd", tokens, rows, width, dtype)) return rc;
    GATMI_REQUIRE(id_bits == 32 || id_bits == 64, GATMI_EINVAL, "embed_bwd: ids of %d bits", id_bits);
    if (rows == 0) return GATMI_OK;
    GATMI_REQUIRE(dtable, GATMI_EINVAL, "embed_bwd: null pointer");
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    if (tokens == 0) {
        const int64_t n = rows * width;
        const unsigned blocks = (unsigned)std::min<int64_t>(4096, (n + 255) / 256);
        if (dtype == GATMI_DTYPE_F32) hipLaunchKernelGGL((embed_zero_kernel<float>), dim3(blocks), dim3(256), 0, st, reinterpret_cast<float *>(dtable), n);
        else hipLaunchKernelGGL((embed_zero_kernel<uint16_t>), dim3(blocks), dim3(256), 0, st, reinterpret_cast<uint16_t *>(dtable), n);
        GATMI_LAUNCH_CHECK("embed_bwd");
        return GATMI_OK;
    }
    GATMI_REQUIRE(ids && dout && ws, GATMI_EINVAL, "embed_bwd: null pointer");
    GATMI_REQUIRE_ALIGNED(ws);
    GATMI_REQUIRE(ld_dout >= width || tokens == 1, GATMI_EINVAL, "embed_bwd: row stride %lld below width %d", (long long)ld_dout, width);
    size_t hist, bits, partial, total;
    embed_bwd_layout(tokens, rows, width, &hist, &bits, &partial, &total);
    uint32_t *w = reinterpret_cast<uint32_t *>(ws);
    const size_t n4 = ((size_t)tokens + 3) / 4 * 4;
    uint32_t *keys[2] = {w, w + 2 * n4}, *poss[2] = {w + n4, w + 3 * n4};
    const int passes = sort_passes(rows);
    SortArgs s;
    s.ids = ids; s.n = (uint32_t)tokens; s.rows = (uint32_t)rows; s.blocks = (uint32_t)((tokens + kTile - 1) / kTile);
    s.hist = w + hist; s.total = s.hist + 256 * (size_t)s.blocks; s.bits = w + bits; s.bit_words = (uint32_t)((rows + 31) / 32);
    int at = 0;
    if (tokens <= kOneBlock) {
        s.key_out = keys[0]; s.pos_out = poss[0];
        if (id_bits == 64) hipLaunchKernelGGL((sort_one_block_kernel<true>), dim3(1), dim3(kOneThreads), 0, st, s, passes);
        else hipLaunchKernelGGL((sort_one_block_kernel<false>), dim3(1), dim3(kOneThreads), 0, st, s, passes);
    } else {
        for (int p = 0; p < passes; ++p) {
            s.shift = 8 * p;
            s.key_in = keys[at]; s.pos_in = poss[at];
            const int to = p == 0 ? 0 : 1 - at;
            s.key_out = keys[to]; s.pos_out = poss[to];
#define PASS(kernel)                                                                                                                          \
    do {                                                                                                                                      \
        if (p > 0) hipLaunchKernelGGL((kernel<false, true>), dim3(s.blocks), dim3(kSortThreads), 0, st, s);                                   \
        else if (id_bits == 64) hipLaunchKernelGGL((kernel<true, true>), dim3(s.blocks), dim3(kSortThreads), 0, st, s);                       \
        else hipLaunchKernelGGL((kernel<true, false>), dim3(s.blocks), dim3(kSortThreads), 0, st, s);                                         \
    } while (0)
            PASS(sort_hist_kernel);
            hipLaunchKernelGGL(sort_scan_kernel, dim3(256), dim3(256), 0, st, s);
            PASS(sort_scatter_kernel);
#undef PASS
            at = to;
        }
    }
    GATMI_LAUNCH_CHECK("embed_bwd (sort)");
    const int E = unit_elems(width, dtype, ld_dout, dout, dtable);
    SegArgs a;
    a.key = keys[at]; a.pos = poss[at]; a.dout = dout; a.dtable = dtable; a.partial = ws + partial; a.bits = s.bits;
    a.ld = ld_dout; a.n = s.n; a.rows = s.rows; a.units = (uint32_t)(width / E); a.chunk = embed_chunk(tokens); a.chunks = (s.n + a.chunk - 1) / a.chunk; a.scale = scale;
    int L = 4;
    while (L < 64 && (uint32_t)L < a.units) L *= 2;
    const unsigned slices = (a.units + L - 1) / L;
    const uint32_t joins = std::min<uint32_t>((a.chunks + 256 / L - 1) / (256 / L), 1 << 14);
    const uint32_t fill = (uint32_t)std::min<int64_t>(1024, (s.bit_words + 3) / 4);
#define SEG(T, e, l)                                                                                                                          \
    do {                                                                                                                                      \
        hipLaunchKernelGGL((embed_seg_kernel<T, e, l>), dim3((a.chunks + 256 / l - 1) / (256 / l), slices), dim3(256), 0, st, a);             \
        hipLaunchKernelGGL((embed_join_kernel<T, e, l>), dim3(joins + fill, slices), dim3(256), 0, st, a, joins, fill);                 \
    } while (0)
#define SEG_L(T, e)                                                                                                                           \
    do {                                                                                                                                      \
        if (L == 4) SEG(T, e, 4); else if (L == 8) SEG(T, e, 8); else if (L == 16) SEG(T, e, 16); else if (L == 32) SEG(T, e, 32); else SEG(T, e, 64); \
    } while (0)
    if (dtype == GATMI_DTYPE_F32) {
        if (E == 4) SEG_L(float, 4); else SEG_L(float, 1);
    } else {
        if (E == 8) SEG_L(uint16_t, 8); else if (E == 2) SEG_L(uint16_t, 2); else SEG_L(uint16_t, 1);
    }
#undef SEG_L
#undef SEG
    GATMI_LAUNCH_CHECK("embed_bwd");
    return GATMI_OK;
}
