// Attention over pages on the warps' matrix instruction: the kernel of a few rows a request (decoding, drafts).
//
// What bounds it is the cache's bytes: a step of one row a request and R = heads / kv_heads heads that share their keys does 4 R
// operations on every value it reads.  So tiles are 16 rows high (mma.sync m16n8k16: tcgen05's 128 would be padding), a tile's rows
// are a request's (row, head of one group) pairs, and each of a block's WARPS warps streams keys and values of its own: 32 keys at a
// time into its ring of STAGES stages by 16-byte asynchronous copies, without a barrier among the warps.  Where a request brings
// more rows than a tile holds, RW warps work on the same keys, each on 16 rows of its own, and share the ring.
//
// Codes become halves in registers (exact) and meet queries as halves, which carry a power of two a row so that every one of them
// is exact that is not 2^-28 of the row's largest; a key's power of two multiplies its finished score.  A value's power joins its
// key's score instead, before the exponential: with s the scores and n the values' exponents (both to base 2)
//     w = 2^(s + n - max (s + n)),   o = sum w code / sum 2^(s - max s) * 2^(max (s + n) - max s),
// so that weights are halves between 0 and 2^14 whatever the values' sizes, with both maxima and the sum in 32 bits.  Queries in
// 32 bits, and their weights, are two halves each.  Over bfloat16 pages queries, keys, values and weights are bfloat16.
//
// A row's head axis is walked in an order that lets a lane read its keys in 16-byte pieces: piece 4h + c of a row's bytes belongs to
// lane c of four, and queries are laid out the same way.  A tile's keys are walked in such an order too: column 2c + x of the
// instruction's j-th eight is key 8c + 2j + x, so that a lane's eight scores a row are of eight keys that follow one another (their
// exponents are one read).  Pieces of rows lie exchanged in shared memory (`place`) so that neither the reads of keys (rows 2j and
// 2j + 1 at a time) nor the transposing ones of values (rows 2j, 2j + 1, 8 + 2j, ...) meet in a bank.
#pragma once
#include "e4m3.cuh"
#include <cuda_fp16.h>
#include <math.h>

namespace mma_pages {

constexpr int TILE = 32;             // keys of a stage
constexpr int WARPS = 4;
constexpr int MOST_KEYS = 1 << 30;   // of a request: places are counted in 32 bits
constexpr float RAISED = 14.0f;      // weights are 2^14 times themselves: the largest in the half's upper range, small ones above its steps

struct Rows {                        // whose rows these are and where their keys lie
    const int* row_start;
    const int* row_count;
    const int* history;
    const int* tables;               // [requests, table_stride]
    int table_stride, total_rows, pages, page_size, window;
    const unsigned* tree;            // [rows, tree_words] or null
    int tree_words;
    unsigned run_pages;              // 2^31 / (page_size / 16), rounded up: t / page_size = (t / 16) * run_pages >> 31 for t < 2^30
    int max_rows;                    // the most rows of a request of this call; one with more is another's
};

template <bool EIGHT, int D>
struct Shape {
    static constexpr int ROW = EIGHT ? D : 2 * D;              // bytes of a key
    static constexpr int PIECES = ROW / 16;
    static constexpr int PLANE = TILE * ROW;
    static constexpr int STAGE = 2 * PLANE + (EIGHT ? 2 * TILE : 0);
    static constexpr int STAGES = 3;
};

__device__ __forceinline__ uint32_t shared_address(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

// Where piece `piece` of row `row` lies.  Rows of 64 bytes share a line of 128 by twos.
template <int ROW>
__device__ __forceinline__ uint32_t place(int row, int piece) {
    if constexpr (ROW == 64) return (uint32_t)(row * 64 + ((piece ^ (row >> 3)) << 4));
    else return (uint32_t)(row * ROW + ((piece ^ (((row & 1) << 2) | (row >> 3))) << 4));
}

__device__ __forceinline__ void copy16(uint32_t to, const void* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copy16_or_zeros(uint32_t to, const void* from, bool real) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(real ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_end() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ uint4 read16(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ void read_transposed(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
template <bool EIGHT>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (EIGHT)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float exp2_fast(float x) {        // -inf gives 0
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float2 from_halves(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }
__device__ __forceinline__ float4 read4(const float* p) { return *reinterpret_cast<const float4*>(p); }
__device__ __forceinline__ float4 read4(const __nv_bfloat16* p) {
    const uint2 t = *reinterpret_cast<const uint2*>(p);
    const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&t.x)), b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&t.y));
    return make_float4(a.x, a.y, b.x, b.y);
}
__device__ __forceinline__ void write4(float* p, float4 v) { *reinterpret_cast<float4*>(p) = v; }
__device__ __forceinline__ void write4(__nv_bfloat16* p, float4 v) { *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w)); }

// The state of a row over some keys: o (sum of weights and codes, of 2^14 relative to `top`), `top` = max (s + n), `peak` = max s, `sum`.
constexpr int PART = 4;              // floats beside a row's D: top, peak, sum, one unused (16-byte rows)
// A state's weight in a state with the maximum `most`: none for one without keys; NaN stays.
__device__ __forceinline__ float share(float mine, float most) { return mine == -INFINITY ? 0.0f : exp2_fast(mine - most); }

template <typename QT, bool EIGHT, int D, int RW>
__global__ void __launch_bounds__(WARPS * 32)
few_rows_kernel(const QT* __restrict__ q, const uint8_t* __restrict__ cache, const uint8_t* __restrict__ exponents, QT* __restrict__ out,
                float* __restrict__ partial, Rows a, int heads, int kv_heads, int splits, float scale_log2) {
    using S = Shape<EIGHT, D>;
    constexpr int STAGES = S::STAGES, RUNS = WARPS / RW;         // groups of warps that each walk keys of their own
    constexpr int PARTS = EIGHT && sizeof(QT) == 4 ? 2 : 1;
    constexpr int STEPS = D / 16, TILES = D / 8;
    pdl_trigger();
    pdl_wait();
    extern __shared__ __align__(128) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const int run = warp / RW, rw = warp % RW;
    const int split = blockIdx.x % splits, row_tile = blockIdx.x / splits, kv = blockIdx.y, r = blockIdx.z;
    const int ratio = heads / kv_heads;
    const int count = a.row_count[r], history = min(max(a.history[r], 0), MOST_KEYS), start = a.row_start[r];
    const int first = row_tile * (16 * RW);                      // the tile's first (row, head) pair
    if (count > a.max_rows || start < 0 || start > a.total_rows) return;
    const int pairs = min(count, a.total_rows - start) * ratio;
    if (first >= pairs) return;
    const int first_row = first / ratio, last_row = (min(first + 16 * RW, pairs) - 1) / ratio;

    // The keys that some row of the tile sees, as tiles of 32, and this block's share of them.
    const int reach = (int)min((long long)a.table_stride * a.page_size, (long long)MOST_KEYS);
    const int end = (int)min((long long)reach, a.tree ? (long long)history + min(count, 32 * a.tree_words) : (long long)history + last_row + 1);
    const int low = a.window > 0 ? max(0, history + first_row - a.window + 1) : 0;
    const int tile0 = low / TILE, tiles = max((end + TILE - 1) / TILE - tile0, 0);
    const int from = tile0 + (int)((long long)tiles * split / splits), to = tile0 + (int)((long long)tiles * (split + 1) / splits);
    const int mine = max(0, (to - from - run + RUNS - 1) / RUNS);             // tiles of this group: from + run, + RUNS, ...

    const int* table = a.tables + (size_t)r * a.table_stride;
    uint8_t* ring = smem + run * (STAGES * S::STAGE);
    const uint32_t ring_at = shared_address(ring);
    // A tile's keys lie in two runs of 16, each within a page.  Lookups are made one tile ahead of the copies.
    const int runs_a_page = a.page_size >> 4;
    auto page_of = [&](int sixteenth) { return (int)(((uint64_t)(unsigned)sixteenth * a.run_pages) >> 31); };
    int page_a = -1, page_b = -1;
    auto look_up = [&](int i) {
        const int n = 2 * (from + run + i * RUNS);
        page_a = i < mine ? table[page_of(n)] : -1;
        page_b = i < mine && (n + 1) * 16 < end ? table[page_of(n + 1)] : -1;
    };
    constexpr int EACH = TILE * S::PIECES / (32 * RW);           // pieces of a plane for a lane
    auto fetch = [&](int i) {
        const int n = 2 * (from + run + i * RUNS), t = n * 16;
        const uint32_t stage = ring_at + (i % STAGES) * S::STAGE;
        const bool in_a = page_a >= 0 && page_a < a.pages, in_b = page_b >= 0 && page_b < a.pages;
        const size_t row_a = ((size_t)(in_a ? page_a : 0) * 2 * kv_heads + kv) * a.page_size + (n - page_of(n) * runs_a_page) * 16;
        const size_t row_b = ((size_t)(in_b ? page_b : 0) * 2 * kv_heads + kv) * a.page_size + (n + 1 - page_of(n + 1) * runs_a_page) * 16;
        const size_t plane = (size_t)kv_heads * a.page_size;
        if (in_a && in_b && t >= low && t + TILE <= end) {
            // A run's rows follow one another, and 512 bytes of them are one warp's copy.
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                const uint8_t* lower = cache + (row_a + p * plane) * S::ROW + lane * 16;
                const uint8_t* upper = cache + (row_b + p * plane) * S::ROW + lane * 16 - 16 * S::ROW;
#pragma unroll
                for (int j = 0; j < EACH; ++j) {
                    const int piece = (j * RW + rw) * 32;
                    copy16(stage + p * S::PLANE + place<S::ROW>((piece + lane) / S::PIECES, (piece + lane) % S::PIECES),
                           (piece >= 16 * S::PIECES ? upper : lower) + piece * 16);
                }
            }
        } else {
#pragma unroll
            for (int p = 0; p < 2; ++p)
#pragma unroll
                for (int j = 0; j < EACH; ++j) {
                    const int piece = (j * RW + rw) * 32 + lane, row = piece / S::PIECES, col = piece % S::PIECES;
                    const bool upper = row >= 16, real = (upper ? in_b : in_a) && t + row < end && t + row >= low;
                    const size_t at = (upper ? row_b + (row - 16) : row_a + row) + p * plane;
                    copy16_or_zeros(stage + p * S::PLANE + place<S::ROW>(row, col), cache + (real ? at * S::ROW + col * 16 : 0), real);
                }
        }
        if (EIGHT && rw == 0 && lane < 4) {                      // exponents: keys' 32, values' 32
            const bool upper = lane & 1, real = upper ? in_b : in_a;
            const size_t at = (upper ? row_b : row_a) + (lane >> 1) * plane;
            copy16_or_zeros(stage + 2 * S::PLANE + (lane >> 1) * TILE + (lane & 1) * 16, exponents + (real ? at : 0), real);
        }
    };
    look_up(0);
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) {
        if (i < mine) fetch(i);
        copies_end();
        look_up(i + 1);
    }

    // This warp's 16 rows: this lane's are g and g + 8.
    const int pair0 = first + rw * 16;
    uint32_t qa[PARTS][STEPS][4];
    float factor[2];                                            // what a score over codes is multiplied by
    int position[2];                                            // history + row; -1: no row
    const unsigned* bits[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const int pair = pair0 + g + 8 * u;
        const bool real = pair < pairs;
        const int row = real ? pair / ratio : 0;
        position[u] = real ? history + row : -1;
        bits[u] = a.tree ? a.tree + (size_t)(start + row) * a.tree_words : nullptr;
        const QT* src = q + ((size_t)(start + row) * heads + kv * ratio + (real ? pair % ratio : 0)) * D;
        float4 x[STEPS];
        unsigned most = 0;
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            const int d = EIGHT ? 64 * (s / 4) + 16 * c + 4 * (s % 4) : 8 * (4 * (s / 2) + c) + 4 * (s % 2);
            x[s] = real ? read4(src + d) : make_float4(0.f, 0.f, 0.f, 0.f);
            most = max(max(most, max(__float_as_uint(x[s].x) & 0x7FFFFFFFu, __float_as_uint(x[s].y) & 0x7FFFFFFFu)),
                       max(__float_as_uint(x[s].z) & 0x7FFFFFFFu, __float_as_uint(x[s].w) & 0x7FFFFFFFu));
        }
        if constexpr (EIGHT) {
            most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
            most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
            const int e = max((int)(most >> 23) - 127, -100);    // the row's largest lies in 2^e .. 2^(e + 1): to 2^14 .. 2^15
            const float f = __int_as_float((127 + 14 - e) << 23);
            factor[u] = __int_as_float((127 - 14 + e) << 23) * scale_log2;
#pragma unroll
            for (int s = 0; s < STEPS; ++s) {
                const float4 y = make_float4(x[s].x * f, x[s].y * f, x[s].z * f, x[s].w * f);
                const uint32_t lo = pack_half(y.x, y.y), hi = pack_half(y.z, y.w);
                qa[0][s][u] = lo;
                qa[0][s][2 + u] = hi;
                if constexpr (PARTS == 2) {
                    const float2 l = from_halves(lo), h = from_halves(hi);
                    qa[1][s][u] = pack_half(y.x - l.x, y.y - l.y);
                    qa[1][s][2 + u] = pack_half(y.z - h.x, y.w - h.y);
                }
            }
        } else {
            factor[u] = scale_log2;
#pragma unroll
            for (int s = 0; s < STEPS; ++s) {
                qa[0][s][u] = pack_bf16(x[s].x, x[s].y);
                qa[0][s][2 + u] = pack_bf16(x[s].z, x[s].w);
            }
        }
    }
    const int warp_row0 = pair0 / ratio, warp_row1 = max(warp_row0, (min(pair0 + 16, pairs) - 1) / ratio);

    float o[TILES][4];
#pragma unroll
    for (int j = 0; j < TILES; ++j)
#pragma unroll
        for (int x = 0; x < 4; ++x) o[j][x] = 0.0f;
    float top[2] = {-INFINITY, -INFINITY}, peak[2] = {-INFINITY, -INFINITY}, sum[2] = {0.0f, 0.0f};     // `sum`: this lane's keys'

    for (int i = 0; i < mine; ++i) {
        copies_wait<STAGES - 2>();
        if constexpr (RW == 1) __syncwarp();
        else asm volatile("bar.sync %0, %1;" ::"r"(1 + run), "n"(RW * 32) : "memory");
        if (i + STAGES - 1 < mine) fetch(i + STAGES - 1);
        copies_end();
        look_up(i + STAGES);
        const uint32_t stage = ring_at + (i % STAGES) * S::STAGE;
        const int t0 = (from + run + i * RUNS) * TILE;
        if (pair0 >= pairs) continue;

        // Scores.
        float s[4][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
#pragma unroll
            for (int x = 0; x < 4; ++x) s[j][x] = 0.0f;
#pragma unroll
            for (int h = 0; h < S::PIECES / 4; ++h) {
                const uint4 k = read16(stage + place<S::ROW>(8 * (g >> 1) + 2 * j + (g & 1), 4 * h + c));
                if constexpr (EIGHT) {
                    const uint32_t w[4] = {k.x, k.y, k.z, k.w};
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const uint32_t b0 = e4m3::halves((unsigned short)(w[x] & 0xffffu)), b1 = e4m3::halves((unsigned short)(w[x] >> 16));
#pragma unroll
                        for (int p = 0; p < PARTS; ++p) mma<EIGHT>(s[j], qa[p][4 * h + x], b0, b1);
                    }
                } else {
                    mma<EIGHT>(s[j], qa[0][2 * h], k.x, k.y);
                    mma<EIGHT>(s[j], qa[0][2 * h + 1], k.z, k.w);
                }
            }
        }
        float vn[8];                                             // the values' exponents; [2j + x]: key 8c + 2j + x
        if constexpr (EIGHT) {
            uint32_t kb[2], vb[2];
            asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(kb[0]), "=r"(kb[1]) : "r"(stage + 2 * S::PLANE + 8 * c) : "memory");
            asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(vb[0]), "=r"(vb[1]) : "r"(stage + 2 * S::PLANE + TILE + 8 * c) : "memory");
#pragma unroll
            for (int n = 0; n < 8; ++n) {
                // Keys' powers: 255 becomes an infinity, which makes NaN of its codes' zeros.
                const float k = __uint_as_float(__byte_perm(kb[n >> 2], 0, 0x0444 | (n & 3) << 12) >> 1);
                s[n >> 1][n & 1] *= k;
                s[n >> 1][2 + (n & 1)] *= k;
                vn[n] = __uint_as_float(__byte_perm(vb[n >> 2], 0x4B000000u, 0x7440 | (n & 3))) - (8388608.0f + 127.0f);
            }
            if (__any_sync(0xffffffffu, __vcmpeq4(vb[0], 0xffffffffu) | __vcmpeq4(vb[1], 0xffffffffu)))
#pragma unroll
                for (int n = 0; n < 8; ++n)
                    if ((vb[n >> 2] >> (8 * (n & 3)) & 255u) == e4m3::NOT_NUMBERS) vn[n] = NAN;
        }
        // Who sees what.  Tiles that all of the warp's rows see whole are not looked at one by one.
        const int sure = a.tree ? history : min(history + warp_row0 + 1, end);
        const bool whole = t0 + TILE <= sure && t0 + TILE <= end && t0 >= low && (a.window <= 0 || t0 > history + warp_row1 - a.window);
        unsigned seen[2] = {0xffffu, 0xffffu};                   // bit 2j + x: key 8c + 2j + x
        if (!whole) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                seen[u] = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const int t = t0 + 8 * c + 2 * j + x;
                        bool ok = position[u] >= 0 && t < end && t >= low;
                        if (a.tree) ok = ok && (t < history || (bits[u][(t - history) >> 5] >> ((t - history) & 31) & 1u));
                        else ok = ok && t <= position[u] && (a.window <= 0 || t > position[u] - a.window);
                        if (ok) seen[u] |= 1u << (2 * j + x);
                        else s[j][2 * u + x] = -INFINITY;
                    }
            }
        }
        float w[4][4];                                           // scores with the values' powers, then weights
        bool grown = false;
        float fade[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            float p = -INFINITY, m = -INFINITY;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                p = max3(p, s[j][2 * u], s[j][2 * u + 1]);
                if constexpr (EIGHT) {
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        w[j][2 * u + x] = fmaf(s[j][2 * u + x], factor[u], vn[2 * j + x]);
                        if (!whole && !(seen[u] >> (2 * j + x) & 1u)) w[j][2 * u + x] = -INFINITY;
                    }
                    m = max3(m, w[j][2 * u], w[j][2 * u + 1]);
                }
            }
            p *= factor[u];
            p = fmaxf(p, __shfl_xor_sync(0xffffffffu, p, 1));
            p = fmaxf(p, __shfl_xor_sync(0xffffffffu, p, 2));
            if constexpr (EIGHT) {
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
            } else {
                m = p;
            }
            const float peak_new = fmaxf(peak[u], p), top_new = fmaxf(top[u], m);
            grown |= peak_new > peak[u] || top_new > top[u];
            // A row that has seen no key yet has maxima of -inf: zero in their place gives weights of zero.
            const float pz = peak_new == -INFINITY ? 0.0f : peak_new, tz = top_new == -INFINITY ? 0.0f : top_new;
            sum[u] *= exp2_fast(peak[u] - pz);
            fade[u] = exp2_fast(top[u] - tz);
            peak[u] = peak_new, top[u] = top_new;
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const float e = exp2_fast(fmaf(s[j][2 * u + x], factor[u], -pz));
                    sum[u] += e;
                    w[j][2 * u + x] = EIGHT ? exp2_fast(w[j][2 * u + x] - (tz - RAISED)) : e;
                }
        }
        if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
            for (int j = 0; j < TILES; ++j) {
                o[j][0] *= fade[0]; o[j][1] *= fade[0]; o[j][2] *= fade[1]; o[j][3] *= fade[1];
            }
        }
        // Weights times values.
        uint32_t pa[PARTS][2][4];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const float w0 = w[2 * h + (x >> 1)][2 * (x & 1)], w1 = w[2 * h + (x >> 1)][2 * (x & 1) + 1];
                if constexpr (EIGHT) {
                    pa[0][h][x] = pack_half(w0, w1);
                    if constexpr (PARTS == 2) {
                        const float2 l = from_halves(pa[0][h][x]);
                        pa[1][h][x] = pack_half(w0 - l.x, w1 - l.y);
                    }
                } else {
                    pa[0][h][x] = pack_bf16(w0, w1);
                }
            }
#pragma unroll
        for (int piece = 0; piece < S::PIECES; ++piece) {
            uint32_t v[4];
            read_transposed(v, stage + S::PLANE + place<S::ROW>(8 * ((lane & 7) >> 1) + 2 * (lane >> 3) + (lane & 1), piece));
            if constexpr (EIGHT) {
                // A register holds values 2g and 2g + 1 of two keys: to the pairs of keys of each.
                uint32_t even[4], odd[4];
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const uint32_t z = __byte_perm(v[x], 0, 0x3120);
                    even[x] = e4m3::halves((unsigned short)(z & 0xffffu));
                    odd[x] = e4m3::halves((unsigned short)(z >> 16));
                }
#pragma unroll
                for (int p = 0; p < PARTS; ++p)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        mma<EIGHT>(o[2 * piece], pa[p][h], even[2 * h], even[2 * h + 1]);
                        mma<EIGHT>(o[2 * piece + 1], pa[p][h], odd[2 * h], odd[2 * h + 1]);
                    }
            } else {
                if (!whole) {
                    // Values that are no numbers, of keys that not every row sees: their products are made one by one for the rows
                    // that do, and zeros take their place (a weight of zero times an infinity is no zero).
                    unsigned bad = 0;
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        if ((v[x] & 0x7F80u) == 0x7F80u) bad |= 1u << (2 * x);
                        if ((v[x] & 0x7F800000u) == 0x7F800000u) bad |= 2u << (2 * x);
                    }
                    if (__any_sync(0xffffffffu, bad)) {
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            // This lane holds value g of keys 8c + 2x, + 1; outputs are of values 2c, + 1 and rows g, g + 8.
#pragma unroll
                            for (int y = 0; y < 2; ++y)
                                for (int cc = 0; cc < 4; ++cc) {
                                    const float we[2] = {__shfl_sync(0xffffffffu, w[x][y], (lane & 28) + cc), __shfl_sync(0xffffffffu, w[x][2 + y], (lane & 28) + cc)};
                                    const unsigned see[2] = {__shfl_sync(0xffffffffu, seen[0], (lane & 28) + cc), __shfl_sync(0xffffffffu, seen[1], (lane & 28) + cc)};
#pragma unroll
                                    for (int d = 0; d < 2; ++d) {
                                        const int source = (2 * c + d) * 4 + cc;
                                        const uint32_t vv = __shfl_sync(0xffffffffu, v[x], source);
                                        const unsigned bb = __shfl_sync(0xffffffffu, bad, source);
                                        const float value = __uint_as_float(y ? vv & 0xffff0000u : vv << 16);
#pragma unroll
                                        for (int u = 0; u < 2; ++u)
                                            if ((bb >> (2 * x + y) & 1u) && (see[u] >> (2 * x + y) & 1u)) o[piece][2 * u + d] = fmaf(we[u], value, o[piece][2 * u + d]);
                                    }
                                }
                        }
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            if (bad >> (2 * x) & 1u) v[x] &= 0xffff0000u;
                            if (bad >> (2 * x + 1) & 1u) v[x] &= 0xffffu;
                        }
                    }
                }
                mma<EIGHT>(o[piece], pa[0][0], v[0], v[1]);
                mma<EIGHT>(o[piece], pa[0][1], v[2], v[3]);
            }
        }
    }
    copies_wait<0>();
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        sum[u] += __shfl_xor_sync(0xffffffffu, sum[u], 1);
        sum[u] += __shfl_xor_sync(0xffffffffu, sum[u], 2);
        if constexpr (!EIGHT) top[u] = peak[u];
    }

    // The groups' states meet in shared memory: [groups][16 RW rows][D + PART] floats.
    __syncthreads();
    float* states = reinterpret_cast<float*>(smem);
    constexpr int ROWF = D + PART;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        float* row = states + ((size_t)run * 16 * RW + rw * 16 + g + 8 * u) * ROWF;
        if (c == 0) row[D] = top[u], row[D + 1] = peak[u], row[D + 2] = sum[u];
        if constexpr (EIGHT) {
#pragma unroll
            for (int p = 0; p < S::PIECES; ++p)
                *reinterpret_cast<float4*>(row + 16 * p + 4 * c) = make_float4(o[2 * p][2 * u], o[2 * p + 1][2 * u], o[2 * p][2 * u + 1], o[2 * p + 1][2 * u + 1]);
        } else {
#pragma unroll
            for (int p = 0; p < S::PIECES; ++p) *reinterpret_cast<float2*>(row + 8 * p + 2 * c) = make_float2(o[p][2 * u], o[p][2 * u + 1]);
        }
    }
    __syncthreads();
    for (int x = threadIdx.x; x < 16 * RW * (D / 4); x += WARPS * 32) {
        const int local = x / (D / 4), d = 4 * (x % (D / 4)), pair = first + local;
        if (pair >= pairs) continue;
        float t = -INFINITY, p = -INFINITY;
#pragma unroll
        for (int n = 0; n < RUNS; ++n) {
            const float* row = states + ((size_t)n * 16 * RW + local) * ROWF;
            t = fmaxf(t, row[D]);
            p = fmaxf(p, row[D + 1]);
        }
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        float l = 0.0f;
#pragma unroll
        for (int n = 0; n < RUNS; ++n) {
            const float* row = states + ((size_t)n * 16 * RW + local) * ROWF;
            const float f = share(row[D], t);
            const float4 v = *reinterpret_cast<const float4*>(row + d);
            acc.x = fmaf(v.x, f, acc.x); acc.y = fmaf(v.y, f, acc.y); acc.z = fmaf(v.z, f, acc.z); acc.w = fmaf(v.w, f, acc.w);
            l = fmaf(row[D + 2], share(row[D + 1], p), l);
        }
        const size_t at = (size_t)(start + pair / ratio) * heads + kv * ratio + pair % ratio;
        if (splits > 1) {
            float* to_row = partial + ((((size_t)r * a.max_rows + pair / ratio) * heads + kv * ratio + pair % ratio) * splits + split) * ROWF;
            *reinterpret_cast<float4*>(to_row + d) = acc;
            if (d == 0) *reinterpret_cast<float4*>(to_row + D) = make_float4(t, p, l, 0.0f);
        } else {
            const float f = l == 0.0f ? 0.0f : (EIGHT ? exp2f(t - p - RAISED) : 1.0f) / l;
            write4(out + at * D + d, l == 0.0f ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(acc.x * f, acc.y * f, acc.z * f, acc.w * f));
        }
    }
}

// Adds up the ranges of keys: a row's D values by D / 4 lanes.
template <typename QT, bool EIGHT, int D>
__global__ void __launch_bounds__(128)
few_rows_merge_kernel(const float* __restrict__ partial, QT* __restrict__ out, Rows a, int heads, int splits) {
    pdl_trigger();
    pdl_wait();
    constexpr int ROWF = D + PART, LANES = D / 4, EACH = 128 / LANES;
    const int r = blockIdx.y, count = a.row_count[r], start = a.row_start[r];
    const long long item = (long long)blockIdx.x * EACH + threadIdx.x / LANES;
    const int row = (int)(item / heads), d = 4 * (threadIdx.x % LANES);
    if (count > a.max_rows || start < 0 || row >= count || start + (long long)row >= a.total_rows) return;
    const size_t at = (size_t)(start + row) * heads + item % heads;
    const float* base = partial + (((size_t)r * a.max_rows + row) * heads + item % heads) * splits * ROWF;
    float t = -INFINITY, p = -INFINITY;
    for (int n = 0; n < splits; ++n) {
        t = fmaxf(t, base[n * ROWF + D]);
        p = fmaxf(p, base[n * ROWF + D + 1]);
    }
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float l = 0.0f;
    for (int n = 0; n < splits; ++n) {
        const float4 v = *reinterpret_cast<const float4*>(base + n * ROWF + d), m = *reinterpret_cast<const float4*>(base + n * ROWF + D);
        const float f = share(m.x, t);
        acc.x = fmaf(v.x, f, acc.x); acc.y = fmaf(v.y, f, acc.y); acc.z = fmaf(v.z, f, acc.z); acc.w = fmaf(v.w, f, acc.w);
        l = fmaf(m.z, share(m.y, p), l);
    }
    const float f = (EIGHT ? exp2f(t - p - RAISED) : 1.0f) / l;
    write4(out + at * D + d, l == 0.0f ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(acc.x * f, acc.y * f, acc.z * f, acc.w * f));
}

}  // namespace mma_pages

