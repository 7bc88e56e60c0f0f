// Attention over pages on the warps' matrix instruction: the kernel of a few rows a request (decoding, drafts).
//
// What bounds it is the cache's bytes: a step of one row a request and R = heads / kv_heads heads that share their keys does 4 R
// operations on every value it reads.  So tiles are 16 rows high (mma.sync m16n8k16: tcgen05's 128 would be padding), a tile's rows
// are a request's (row, head of one group) pairs, and each of a block's WARPS warps streams keys and values of its own: 32 keys at a
// time into its ring of STAGES stages by 16-byte asynchronous copies, without a barrier among the warps.  Where a request brings
// more rows than a tile holds, RW warps work on the same keys, each on 16 rows of its own, and share the ring.
//
// The work is cut evenly: the tiles of 32 keys of all (request, tile of rows, key/value head) items in a row, every block of the grid
// an equal share of them (Walk), however unlike the requests' lengths.  An item that lies within a block is written at once; one that is
// cut leaves a state in each block's slots, and a second kernel adds those up.
//
// Codes become halves in registers (exact) and meet queries as halves, which carry a power of two a row so that every one of them
// is exact that is not 2^-28 of the row's largest; a key's power of two multiplies its finished score.  A value's power joins its
// key's score instead, before the exponential: with s the scores and n the values' exponents (both to base 2)
//     w = 2^(s + n - max (s + n)),   o = sum w code / sum 2^(s - max s) * 2^(max (s + n) - max s),
// so that weights fit halves whatever the values' sizes, with both maxima and the sum in 32 bits.  A row of zeros, whose power is 1, would
// set that maximum and leave small values no bits: it counts with 2^-127, as a page that is not there.  Queries in
// 32 bits, and their weights, are two halves each.  Over bfloat16 pages queries, keys, values and weights are bfloat16.
//
// Measured with the kernel that adds up (32 heads of 128 over 8, bfloat16 queries): 8 x 8,192 keys 31.7 us, 4.3 TB/s (32 alone and cold: 244 registers,
// so eight warps an SM, 37 % of issue slots, tensor pipe 24 %: what bounds the tiles is the length of a warp's chain); 1 x 32,768 23.1 us.
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
// Tiles that an item's beginning and end take as long as (512 items of 64 ragged requests of up to 4,096 keys: 4 73 us, 8 63, 12 59,
// 18 60; 8 x 8,192 keys 33.8, 32.7, 31.9, 32.0; asking for the next item's tiles before an item's states meet, or for its pages and
// queries an item ahead, changes neither these times nor where they are least).
constexpr int OPEN = 12;
constexpr int MOST_KEYS = 1 << 30;   // of a request: places are counted in 32 bits
// Weights are 2^10 times themselves over codes, so that small ones lie above a half's steps; the maxima that the exponentials use are
// raised only when a row's true one has grown by more than 2^5 (2^15 is a half, and most tiles then leave the sums alone).
constexpr float RAISED = 10.0f, BEHIND = 5.0f;

struct Rows {                        // whose rows these are and where their keys lie
    const int* row_start;
    const int* row_count;
    const int* history;
    const int* tables;               // [requests, table_stride]
    int table_stride, total_rows, pages, page_size, window;
    const unsigned* tree;            // [rows, tree_words] or null
    int tree_words;
    unsigned run_pages;              // 2^31 / (page_size / 16), rounded up: t / page_size = (t / 16) * run_pages >> 31 for t < 2^30
    int max_tiles;                   // the most tiles of keys of a request
    int max_rows;                    // the most rows of a request of this call; one with more is another's
};

template <bool EIGHT, int D>
struct Shape {
    static constexpr int ROW = EIGHT ? D : 2 * D;              // bytes of a key
    static constexpr int PIECES = ROW / 16;
    static constexpr int PLANE = TILE * ROW;
    static constexpr int STAGE = 2 * PLANE + (EIGHT ? 256 : 0);      // planes, exponents; whole 256s, so that pieces' bits can be flipped in addresses
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

// The state of a row over some keys: o (the sum of weights and codes), relative to 2^top; the sum of 2^(s - peak).
constexpr int PART = 4;              // floats beside a row's D: top, peak, sum, one unused (16-byte rows)
// A state's weight in a state with the maximum `most`: none for one without keys; NaN stays.
__device__ __forceinline__ float share(float mine, float most) { return mine == -INFINITY ? 0.0f : exp2_fast(mine - most); }

// A row's output from its whole state.  Nothing seen: zeros.
template <bool EIGHT>
__device__ __forceinline__ float4 finished(float4 acc, float top, float peak, float sum) {
    if (sum == 0.0f) return make_float4(0.f, 0.f, 0.f, 0.f);
    const float f = (EIGHT ? exp2f(top - peak) : 1.0f) / sum;
    return make_float4(acc.x * f, acc.y * f, acc.z * f, acc.w * f);
}

// Which of a stage's rows, a lane each, at `at` are zeros (of either sign) throughout; it stops at the piece that says so.  (8 x 8,192 keys
// whose values all have a row of zeros' byte 32.0 -> 35.0 us, 39.3 without stopping; all of zeros 41.4.)
template <int ROW>
__device__ __forceinline__ unsigned rows_of_zeros(uint32_t at) {
    uint32_t any = 0;
    unsigned zeros = 0xffffffffu;
#pragma unroll 1
    for (int piece = 0; piece < ROW / 16 && zeros; ++piece) {
        const uint4 v = read16(at + place<ROW>(threadIdx.x & 31, piece));
        any |= (v.x | v.y | v.z | v.w) & 0x7F7F7F7Fu;
        zeros = __ballot_sync(0xffffffffu, any == 0);
    }
    return zeros;
}

// bfloat16 values that are no numbers, of keys that not every row sees: their products are added one by one for the rows that do, and
// zeros take their place (a weight of zero times an infinity is no zero).  This lane holds value g of keys 8c + 2x, + 1 in v[x];
// its outputs are of values 2c, + 1 and rows g, g + 8.
__device__ __forceinline__ void add_no_numbers(float (&o)[4], uint32_t (&v)[4], const float (&w)[4][4], const unsigned (&seen)[2]) {
    const int lane = threadIdx.x & 31, c = lane & 3;
    unsigned bad = 0;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
        if ((v[x] & 0x7F80u) == 0x7F80u) bad |= 1u << (2 * x);
        if ((v[x] & 0x7F800000u) == 0x7F800000u) bad |= 2u << (2 * x);
    }
    if (!__any_sync(0xffffffffu, bad)) return;
#pragma unroll
    for (int n = 0; n < 8; ++n)
        for (int cc = 0; cc < 4; ++cc) {
            const int quad = (lane & 28) + cc;
            const float we[2] = {__shfl_sync(0xffffffffu, w[n >> 1][n & 1], quad), __shfl_sync(0xffffffffu, w[n >> 1][2 + (n & 1)], quad)};
            const unsigned see[2] = {__shfl_sync(0xffffffffu, seen[0], quad), __shfl_sync(0xffffffffu, seen[1], quad)};
#pragma unroll
            for (int d = 0; d < 2; ++d) {
                const int source = (2 * c + d) * 4 + cc;
                const uint32_t vv = __shfl_sync(0xffffffffu, v[n >> 1], source);
                const unsigned bb = __shfl_sync(0xffffffffu, bad, source);
                const float value = __uint_as_float(n & 1 ? vv & 0xffff0000u : vv << 16);
#pragma unroll
                for (int u = 0; u < 2; ++u)
                    if ((bb >> n & 1u) && (see[u] >> n & 1u)) o[2 * u + d] = fmaf(we[u], value, o[2 * u + d]);
            }
        }
#pragma unroll
    for (int x = 0; x < 4; ++x) {
        if (bad >> (2 * x) & 1u) v[x] &= 0xffff0000u;
        if (bad >> (2 * x + 1) & 1u) v[x] &= 0xffffu;
    }
}

// ---- the work, cut evenly ----
// An item (a tile of a request's rows and a key/value head) has a request's tiles of KEYS keys, and takes OPEN tiles' time more to begin
// and to end.  So items lie in a row with OPEN + tiles places each, and block b of `blocks` has the places all * b / blocks up to
// all * (b + 1) / blocks.  What a block has of an item whose places it shares with others goes to its first slot where the item began
// before the block's places, else to its second.  Places are counted in 32 bits: a request's tiles are cut off at `max_tiles`, by
// which the host knows that they suffice.
struct Request {
    int count, history, start, pairs, low, end, tile0, tiles, row_tiles;
};
template <int KEYS>
__device__ __forceinline__ Request request_of(const Rows& a, int r, int ratio, int tile_rows) {
    Request q;
    q.count = a.row_count[r], q.history = min(max(a.history[r], 0), MOST_KEYS), q.start = a.row_start[r];
    const bool ours = q.count > 0 && q.count <= a.max_rows && q.start >= 0 && q.start < a.total_rows;
    q.count = ours ? min(q.count, a.total_rows - q.start) : 0;
    q.pairs = q.count * ratio;
    const int reach = (int)min((long long)a.table_stride * a.page_size, (long long)MOST_KEYS);
    q.end = min(reach, q.history + (a.tree ? min(q.count, 32 * a.tree_words) : q.count));
    q.low = a.window > 0 ? max(0, q.history - a.window + 1) : 0;
    q.tile0 = q.low / KEYS;
    // (At least one tile, so that rows that see nothing are written too.)
    q.tiles = ours ? min(max((q.end + KEYS - 1) / KEYS - q.tile0, 1), a.max_tiles) : 0;
    q.row_tiles = (q.pairs + tile_rows - 1) / tile_rows;
    return q;
}
// A request's items and places.
template <int KEYS, int OPEN>
__device__ __forceinline__ int places_of(const Rows& a, int r, int requests, int ratio, int tile_rows, int kv_heads, int& items) {
    items = 0;
    if (r >= requests) return 0;
    const Request q = request_of<KEYS>(a, r, ratio, tile_rows);
    items = q.row_tiles * kv_heads;
    return items * (q.tiles + OPEN);
}
// The places and items of all requests, and the places of the first `stop`.  By whole warps.
template <int KEYS, int OPEN>
__device__ __forceinline__ int all_places(const Rows& a, int requests, int ratio, int tile_rows, int kv_heads, int& items, int stop, int& before) {
    const int lane = threadIdx.x & 31;
    unsigned all = 0, of = 0, first = 0;
    for (int r = lane; r - lane < requests; r += 32) {
        int n;
        const unsigned places = places_of<KEYS, OPEN>(a, r, requests, ratio, tile_rows, kv_heads, n);
        all += places, of += n;
        if (r < stop) first += places;
    }
    items = (int)__reduce_add_sync(0xffffffffu, of);
    before = (int)__reduce_add_sync(0xffffffffu, first);
    return (int)__reduce_add_sync(0xffffffffu, all);
}
// The request that place `x` falls in, and the places before it.  By whole warps.
template <int KEYS, int OPEN>
__device__ __forceinline__ int request_at_place(const Rows& a, int requests, int ratio, int tile_rows, int kv_heads, int x, int& before) {
    const int lane = threadIdx.x & 31;
    before = 0;
    for (int r0 = 0; r0 < requests; r0 += 32) {
        int items, upto = places_of<KEYS, OPEN>(a, r0 + lane, requests, ratio, tile_rows, kv_heads, items);
        const int n = upto, sum = (int)__reduce_add_sync(0xffffffffu, (unsigned)n);
        if (x < before + sum) {
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += v;
            }
            const int in = __ffs(__ballot_sync(0xffffffffu, x < before + upto)) - 1;
            before += __shfl_sync(0xffffffffu, upto - n, in);
            return r0 + in;
        }
        before += sum;
    }
    return requests;
}
// The blocks that share the work: all of the grid, as far as each gets two tiles a group of warps or an item of its own.
template <int OPEN>
__device__ __forceinline__ int working_blocks(int all, int items, int blocks, int runs) { return min(blocks, max(items, (all - items * OPEN) / (2 * runs))); }
__device__ __forceinline__ int share_begins(int all, int blocks, int b) {
    return all < 1 << 20 ? (int)((unsigned)all * b / blocks) : (int)((unsigned long long)all * b / blocks);      // (blocks are a few hundred)
}

// A block's items one after another.
template <int KEYS, int OPEN>
struct Walk {
    Request rq;
    int r, kv, first, from, tiles, slot;     // request, head, first pair; the tiles of the item that are the block's (none: go on); slot for its state
    bool whole;                              // all of the item's
    int at, until, request_at, tile_rows, kv_heads, ratio;
    __device__ __forceinline__ Walk(const Rows& a, int requests, int ratio_, int tile_rows_, int kv_heads_, int grid, int runs)
        : tile_rows(tile_rows_), kv_heads(kv_heads_), ratio(ratio_) {
        int items, unused;
        const int all = all_places<KEYS, OPEN>(a, requests, ratio, tile_rows, kv_heads, items, 0, unused), blocks = working_blocks<OPEN>(all, items, grid, runs);
        const bool works = (int)blockIdx.x < blocks;
        at = works ? share_begins(all, blocks, blockIdx.x) : 0;
        until = works ? share_begins(all, blocks, blockIdx.x + 1) : 0;
        r = request_at_place<KEYS, OPEN>(a, requests, ratio, tile_rows, kv_heads, at, request_at);
        if (at < until) rq = request_of<KEYS>(a, r, ratio, tile_rows);
    }
    __device__ __forceinline__ bool next(const Rows& a) {
        do {
            if (at >= until) return false;
            int places = rq.row_tiles * kv_heads * (rq.tiles + OPEN);
            while (at >= request_at + places) {
                request_at += places;
                rq = request_of<KEYS>(a, ++r, ratio, tile_rows);
                places = rq.row_tiles * kv_heads * (rq.tiles + OPEN);
            }
            const int each = rq.tiles + OPEN, item = (at - request_at) / each, item_at = request_at + item * each, upto = min(until, item_at + each);
            kv = item % kv_heads, first = item / kv_heads * tile_rows;
            const int skipped = max(at - item_at - OPEN, 0);
            tiles = max(upto - item_at - OPEN, 0) - skipped;
            from = rq.tile0 + skipped;
            whole = tiles == rq.tiles;
            slot = at > item_at ? 0 : 1;
            at = upto;
        } while (tiles == 0);
        return true;
    }
};

template <typename QT, bool EIGHT, int D, int RW>
__global__ void __launch_bounds__(WARPS * 32)
few_rows_kernel(const QT* __restrict__ q, const uint8_t* __restrict__ cache, const uint8_t* __restrict__ exponents, QT* __restrict__ out,
                float* __restrict__ partial, Rows a, int requests, int heads, int kv_heads, float scale_log2) {
    using S = Shape<EIGHT, D>;
    constexpr int STAGES = S::STAGES, RUNS = WARPS / RW;         // groups of warps that each walk keys of their own
    constexpr int PARTS = EIGHT && sizeof(QT) == 4 ? 2 : 1;
    constexpr int STEPS = D / 16, TILES = D / 8, TILE_ROWS = 16 * RW, ROWF = D + PART;
    pdl_wait();
    pdl_trigger();                       // (in this order: the merge reads the requests' counts without waiting)
    extern __shared__ __align__(256) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const int run = warp / RW, rw = warp % RW;
    const int ratio = heads / kv_heads;

    Walk<TILE, OPEN> walk(a, requests, ratio, TILE_ROWS, kv_heads, gridDim.x, RUNS);

    // Where this lane's pieces lie: what it copies, keys (by the two, or four, quarters of a row's bytes), values.
    const uint32_t ring_at = shared_address(smem) + run * (STAGES * S::STAGE);
    const uint32_t to_lane = place<S::ROW>((rw * 32 + lane) / S::PIECES, (rw * 32 + lane) % S::PIECES);
    const uint32_t key_lane = place<S::ROW>(8 * (g >> 1) + (g & 1), c);
    const uint32_t value_lane = S::PLANE + place<S::ROW>(8 * ((lane & 7) >> 1) + 2 * (lane >> 3) + (lane & 1), 0);
    constexpr int EACH = TILE * S::PIECES / (32 * RW);           // pieces of a plane for a lane
    const int runs_a_page = a.page_size >> 4;
    const unsigned plane = (unsigned)kv_heads * a.page_size;     // rows of a plane of a page
    auto page_of = [&](int sixteenth) { return (int)(((uint64_t)(unsigned)sixteenth * a.run_pages) >> 31); };

    while (walk.next(a)) {
        const int history = walk.rq.history, start = walk.rq.start, pairs = walk.rq.pairs, end = walk.rq.end, low = walk.rq.low;
        const int from = walk.from, first = walk.first, kv = walk.kv, r = walk.r;
        const int mine = max(0, (walk.tiles - run + RUNS - 1) / RUNS);             // tiles of this group: from + run, + RUNS, ...

        const int* table = a.tables + (size_t)r * a.table_stride;
        // A tile's keys lie in two runs of 16, each within a page.  Lookups are made one tile ahead of the copies.
        int page_a = -1, page_b = -1;
        auto look_up = [&](int i) {
            const int n = 2 * (from + run + i * RUNS);
            page_a = i < mine && n * 16 < end ? table[page_of(n)] : -1;
            page_b = i < mine && (n + 1) * 16 < end ? table[page_of(n + 1)] : -1;
        };
        auto fetch = [&](int i) {
            const int n = 2 * (from + run + i * RUNS), t = n * 16;
            const uint32_t stage = ring_at + (i % STAGES) * S::STAGE;
            const bool in_a = (unsigned)page_a < (unsigned)a.pages, in_b = (unsigned)page_b < (unsigned)a.pages;
            const unsigned row_a = ((unsigned)(in_a ? page_a : 0) * 2 * kv_heads + kv) * a.page_size + (n - page_of(n) * runs_a_page) * 16;
            const unsigned row_b = ((unsigned)(in_b ? page_b : 0) * 2 * kv_heads + kv) * a.page_size + (n + 1 - page_of(n + 1) * runs_a_page) * 16;
            if (in_a && in_b && t >= low && t + TILE <= end) {
                // A run's rows follow one another, and 512 bytes of them are one warp's copy.
#pragma unroll
                for (int p = 0; p < 2; ++p) {
                    const uint8_t* lower = cache + (size_t)(row_a + p * plane) * S::ROW + (rw * 32 + lane) * 16;
                    const uint8_t* upper = cache + (size_t)(row_b + p * plane) * S::ROW + (rw * 32 + lane) * 16;
#pragma unroll
                    for (int j = 0; j < EACH; ++j) {
                        constexpr int HALF = 16 * S::ROW;        // bytes of a run
                        const int by = j * RW * 512;
                        const uint32_t dst = stage + p * S::PLANE + (to_lane ^ (uint32_t)(((by / S::ROW) >> 3) << 4)) + by;
                        if constexpr (EACH == 1) copy16(dst, rw >= RW / 2 ? upper - HALF : lower);
                        else copy16(dst, by >= HALF ? upper + (by - HALF) : lower + by);
                    }
                }
            } else {
#pragma unroll
                for (int p = 0; p < 2; ++p)
#pragma unroll
                    for (int j = 0; j < EACH; ++j) {
                        const int piece = (j * RW + rw) * 32 + lane, row = piece / S::PIECES, col = piece % S::PIECES;
                        const bool upper = row >= 16, real = (upper ? in_b : in_a) && t + row < end && t + row >= low;
                        const size_t src = (upper ? row_b + (row - 16) : row_a + row) + p * plane;
                        copy16_or_zeros(stage + p * S::PLANE + place<S::ROW>(row, col), cache + (real ? src * S::ROW + col * 16 : 0), real);
                    }
            }
            if (EIGHT && rw == 0 && lane < 4) {                  // exponents: keys' 32, values' 32
                const bool upper = lane & 1, real = upper ? in_b : in_a;
                const size_t src = (upper ? row_b : row_a) + (lane >> 1) * plane;
                copy16_or_zeros(stage + 2 * S::PLANE + (lane >> 1) * TILE + (lane & 1) * 16, exponents + (real ? src : 0), real);
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
        float factor[2];                                        // what a score over codes is multiplied by
        int position[2];                                        // history + row; -1: no row
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int pair = pair0 + g + 8 * u;
            const bool real = pair < pairs;
            const int row = real ? pair / ratio : 0;
            position[u] = real ? history + row : -1;
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
                const int e = max((int)(most >> 23) - 127, -100);        // the row's largest lies in 2^e .. 2^(e + 1): to 2^14 .. 2^15
                const float f = __int_as_float((127 + 14 - e) << 23);
                factor[u] = fmaxf(__int_as_float((127 - 14 + e) << 23) * scale_log2, 1.0e-44f);      // (not zero: a masked score stays -inf)
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
        // The keys that all of the warp's rows see: from `all_from` to before `all_to`.
        const int warp_row0 = pair0 / ratio, warp_row1 = max(warp_row0, (min(pair0 + 16, pairs) - 1) / ratio);
        const int all_to = a.tree ? min(history, end) : min(history + warp_row0 + 1, end);
        const int all_from = a.window > 0 ? max(history + warp_row1 - a.window + 1, 0) : 0;

        float o[TILES][4];
#pragma unroll
        for (int j = 0; j < TILES; ++j)
#pragma unroll
            for (int x = 0; x < 4; ++x) o[j][x] = 0.0f;
        // What the exponentials are relative to (-inf: no key yet, and zero is subtracted), and the sum of this lane's keys.
        float top[2] = {-INFINITY, -INFINITY}, peak[2] = {-INFINITY, -INFINITY}, sum[2] = {0.0f, 0.0f};

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
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int x = 0; x < 4; ++x) s[j][x] = 0.0f;
#pragma unroll
            for (int h = 0; h < S::PIECES / 4; ++h) {
                const uint32_t keys = stage + (key_lane ^ (uint32_t)(h << 6));
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint4 k = read16(keys + j * 2 * S::ROW);
                    if constexpr (EIGHT) {
                        const uint32_t w[4] = {k.x, k.y, k.z, k.w};
                        uint32_t b0[4], b1[4];
#pragma unroll
                        for (int x = 0; x < 4; ++x) b0[x] = e4m3::halves((unsigned short)(w[x] & 0xffffu)), b1[x] = e4m3::halves((unsigned short)(w[x] >> 16));
                        // (The small part first: the instruction cuts its sums off, at the size that they have by then.)
#pragma unroll
                        for (int p = PARTS - 1; p >= 0; --p)
#pragma unroll
                            for (int x = 0; x < 4; ++x) mma<EIGHT>(s[j], qa[p][4 * h + x], b0[x], b1[x]);
                    } else {
                        mma<EIGHT>(s[j], qa[0][2 * h], k.x, k.y);
                        mma<EIGHT>(s[j], qa[0][2 * h + 1], k.z, k.w);
                    }
                }
            }
            float w[4][4];                                       // over codes: scores with the values' powers; then weights
            uint32_t vb[2];
            auto value_power = [&](int n) { return __uint_as_float(__byte_perm(vb[n >> 2], 0x4B000000u, 0x7440 | (n & 3))) - (8388608.0f + 127.0f); };
            if constexpr (EIGHT) {
                uint32_t kb[2];
                asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(kb[0]), "=r"(kb[1]) : "r"(stage + 2 * S::PLANE + 8 * c) : "memory");
                asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(vb[0]), "=r"(vb[1]) : "r"(stage + 2 * S::PLANE + TILE + 8 * c) : "memory");
#pragma unroll
                for (int n = 0; n < 8; ++n) {
                    // Keys' powers: 255 becomes an infinity, which makes NaN of its codes' zeros.
                    const float k = __uint_as_float(__byte_perm(kb[n >> 2], 0, 0x0444 | (n & 3) << 12) >> 1);
                    const float v = value_power(n);
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        float& z = s[n >> 1][2 * u + (n & 1)];
                        z *= k;
                        w[n >> 1][2 * u + (n & 1)] = fmaf(z, factor[u], v);
                    }
                }
                // Values that have the byte of a row of zeros, 127, or of one that is no numbers, 255.
                if (__any_sync(0xffffffffu, __vcmpeq4(vb[0] | 0x80808080u, 0xffffffffu) | __vcmpeq4(vb[1] | 0x80808080u, 0xffffffffu))) {
                    const unsigned zeros = rows_of_zeros<S::ROW>(stage + S::PLANE) >> (8 * c);
#pragma unroll
                    for (int n = 0; n < 8; ++n) {
                        const unsigned byte = vb[n >> 2] >> (8 * (n & 3)) & 255u;
                        const bool nothing = byte == 127u && (zeros >> n & 1u);
                        if (nothing) vb[n >> 2] &= ~(255u << (8 * (n & 3)));
#pragma unroll
                        for (int u = 0; u < 2; ++u) {
                            float& x = w[n >> 1][2 * u + (n & 1)];
                            if (byte == e4m3::NOT_NUMBERS) x = NAN;
                            else if (nothing) x = fmaf(s[n >> 1][2 * u + (n & 1)], factor[u], -127.0f);
                        }
                    }
                }
            }
            // Who sees what, where that is not everyone everything.
            const bool whole = t0 >= all_from && t0 + TILE <= all_to;
            unsigned seen[2] = {0xffffu, 0xffffu};               // bit 2j + x: key 8c + 2j + x
            if (!whole) {
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    seen[u] = 0;
                    const unsigned* bits = a.tree + (a.tree ? (size_t)(start + max(position[u] - history, 0)) * a.tree_words : 0);
#pragma unroll
                    for (int n = 0; n < 8; ++n) {
                        const int t = t0 + 8 * c + n;
                        bool ok = position[u] >= 0 && t < end && t >= low;
                        if (a.tree) ok = ok && (t < history || (bits[(t - history) >> 5] >> ((t - history) & 31) & 1u));
                        else ok = ok && t <= position[u] && (a.window <= 0 || t > position[u] - a.window);
                        if (ok) seen[u] |= 1u << n;
                        else s[n >> 1][2 * u + (n & 1)] = w[n >> 1][2 * u + (n & 1)] = -INFINITY;
                    }
                }
            }
            float p[2], m[2];                                    // the rows' true maxima in this tile
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                p[u] = fmaxf(max3(fmaxf(s[0][2 * u], s[0][2 * u + 1]), s[1][2 * u], s[1][2 * u + 1]),
                             max3(fmaxf(s[2][2 * u], s[2][2 * u + 1]), s[3][2 * u], s[3][2 * u + 1])) * factor[u];
                p[u] = fmaxf(p[u], __shfl_xor_sync(0xffffffffu, p[u], 1));
                p[u] = fmaxf(p[u], __shfl_xor_sync(0xffffffffu, p[u], 2));
                if constexpr (EIGHT) {
                    m[u] = fmaxf(max3(fmaxf(w[0][2 * u], w[0][2 * u + 1]), w[1][2 * u], w[1][2 * u + 1]),
                                 max3(fmaxf(w[2][2 * u], w[2][2 * u + 1]), w[3][2 * u], w[3][2 * u + 1]));
                    m[u] = fmaxf(m[u], __shfl_xor_sync(0xffffffffu, m[u], 1));
                    m[u] = fmaxf(m[u], __shfl_xor_sync(0xffffffffu, m[u], 2));
                } else {
                    m[u] = p[u];
                }
            }
            if (__any_sync(0xffffffffu, p[0] > peak[0] + BEHIND || p[1] > peak[1] + BEHIND || m[0] > top[0] + BEHIND || m[1] > top[1] + BEHIND)) {
                float fade[2];
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const float peak_new = fmaxf(peak[u], p[u]), top_new = fmaxf(top[u], m[u]);
                    sum[u] *= share(peak[u], peak_new);
                    fade[u] = share(top[u], top_new);
                    peak[u] = peak_new, top[u] = top_new;
                }
#pragma unroll
                for (int j = 0; j < TILES; ++j) {
                    o[j][0] *= fade[0]; o[j][1] *= fade[0]; o[j][2] *= fade[1]; o[j][3] *= fade[1];
                }
            }
            uint32_t pa[PARTS][2][4];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const float pz = peak[u] == -INFINITY ? 0.0f : peak[u], tz = (top[u] == -INFINITY ? 0.0f : top[u]) - RAISED;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const float e = exp2_fast(fmaf(s[j][2 * u + x], factor[u], -pz));
                        sum[u] += e;
                        if constexpr (PARTS == 2) {
                            // In 32 bits a score and its value's power are not rounded together before the reference is taken off (scores
                            // of 16 to 32 would cost 2^-20 of a weight); what is masked or no number stays what it is.
                            const float both = w[j][2 * u + x];
                            w[j][2 * u + x] = exp2_fast(fabsf(both) < INFINITY ? fmaf(s[j][2 * u + x], factor[u], value_power(2 * j + x) - tz) : both);
                        } else {
                            w[j][2 * u + x] = EIGHT ? exp2_fast(w[j][2 * u + x] - tz) : e;
                        }
                    }
                    const float w0 = w[j][2 * u], w1 = w[j][2 * u + 1];
                    uint32_t& to = pa[0][j >> 1][2 * (j & 1) + u];
                    if constexpr (EIGHT) {
                        to = pack_half(w0, w1);
                        if constexpr (PARTS == 2) {
                            const float2 l = from_halves(to);
                            pa[1][j >> 1][2 * (j & 1) + u] = pack_half(w0 - l.x, w1 - l.y);
                        }
                    } else {
                        to = pack_bf16(w0, w1);
                    }
                }
            }
            // Weights times values.
#pragma unroll
            for (int piece = 0; piece < S::PIECES; ++piece) {
                uint32_t v[4];
                read_transposed(v, stage + (value_lane ^ (uint32_t)(piece << 4)));
                if constexpr (EIGHT) {
                    // A register holds values 2g and 2g + 1 of two keys: to the pairs of keys of each.
                    uint32_t even[4], odd[4];
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const uint32_t z = __byte_perm(v[x], 0, 0x3120);
                        even[x] = e4m3::halves((unsigned short)(z & 0xffffu));
                        odd[x] = e4m3::halves((unsigned short)(z >> 16));
                    }
                    if constexpr (PARTS == 2) {
                        // In 32 bits a tile's sums are made by themselves and added by a rounded addition (with the scores' order and the
                        // weights' references above: 1.1e-6 -> 0.55e-6 off, of the whole, at heads of 64; 4 x 2,001 keys 14.1 -> 15.0 us).
                        float of_even[4] = {0.f, 0.f, 0.f, 0.f}, of_odd[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int part = 1; part >= 0; --part)
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                mma<EIGHT>(of_even, pa[part][h], even[2 * h], even[2 * h + 1]);
                                mma<EIGHT>(of_odd, pa[part][h], odd[2 * h], odd[2 * h + 1]);
                            }
#pragma unroll
                        for (int x = 0; x < 4; ++x) o[2 * piece][x] += of_even[x], o[2 * piece + 1][x] += of_odd[x];
                    } else {
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            mma<EIGHT>(o[2 * piece], pa[0][h], even[2 * h], even[2 * h + 1]);
                            mma<EIGHT>(o[2 * piece + 1], pa[0][h], odd[2 * h], odd[2 * h + 1]);
                        }
                    }
                } else {
                    if (!whole) add_no_numbers(o[piece], v, w, seen);
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
        }

        // The groups' states meet in shared memory: [groups][rows][D + PART] floats.
        __syncthreads();
        float* states = reinterpret_cast<float*>(smem);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            float* row = states + ((size_t)run * TILE_ROWS + rw * 16 + g + 8 * u) * ROWF;
            if (c == 0) row[D] = EIGHT ? top[u] - RAISED : top[u], row[D + 1] = peak[u], row[D + 2] = sum[u];
            if constexpr (EIGHT) {
#pragma unroll
                for (int n = 0; n < S::PIECES; ++n)
                    *reinterpret_cast<float4*>(row + 16 * n + 4 * c) = make_float4(o[2 * n][2 * u], o[2 * n + 1][2 * u], o[2 * n][2 * u + 1], o[2 * n + 1][2 * u + 1]);
            } else {
#pragma unroll
                for (int n = 0; n < S::PIECES; ++n) *reinterpret_cast<float2*>(row + 8 * n + 2 * c) = make_float2(o[n][2 * u], o[n][2 * u + 1]);
            }
        }
        __syncthreads();
        float* slot = partial + (2 * (size_t)blockIdx.x + walk.slot) * TILE_ROWS * ROWF;
        for (int x = threadIdx.x; x < TILE_ROWS * (D / 4); x += WARPS * 32) {
            const int local = x / (D / 4), d = 4 * (x % (D / 4)), pair = first + local;
            if (pair >= pairs) continue;
            float t = -INFINITY, most = -INFINITY;
#pragma unroll
            for (int n = 0; n < RUNS; ++n) {
                const float* row = states + ((size_t)n * TILE_ROWS + local) * ROWF;
                t = fmaxf(t, row[D]);
                most = fmaxf(most, row[D + 1]);
            }
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
            float l = 0.0f;
#pragma unroll
            for (int n = 0; n < RUNS; ++n) {
                const float* row = states + ((size_t)n * TILE_ROWS + local) * ROWF;
                const float f = share(row[D], t);
                const float4 v = *reinterpret_cast<const float4*>(row + d);
                acc.x = fmaf(v.x, f, acc.x); acc.y = fmaf(v.y, f, acc.y); acc.z = fmaf(v.z, f, acc.z); acc.w = fmaf(v.w, f, acc.w);
                l = fmaf(row[D + 2], share(row[D + 1], most), l);
            }
            if (walk.whole) {
                write4(out + ((size_t)(start + pair / ratio) * heads + kv * ratio + pair % ratio) * D + d, finished<EIGHT>(acc, t, most, l));
            } else {
                *reinterpret_cast<float4*>(slot + (size_t)local * ROWF + d) = acc;
                if (d == 0) *reinterpret_cast<float4*>(slot + (size_t)local * ROWF + D) = make_float4(t, most, l, 0.0f);
            }
        }
        __syncthreads();
    }
}

// Adds up the items that blocks share, one warp for 128 of a (row, head)'s values (two rows of 64).  Which blocks those are follows
// from the same counts as in the kernel before.
template <typename QT, bool EIGHT, int D, int TILE_ROWS, int KEYS, int OPEN, int RUNS>
__global__ void __launch_bounds__(128)
merge_kernel(const float* __restrict__ partial, QT* __restrict__ out, Rows a, int requests, int heads, int kv_heads, int grid) {
    pdl_trigger();
    constexpr int ROWF = D + PART, LANES = D / 4, EACH = 128 / LANES;
    const int r = blockIdx.y, ratio = heads / kv_heads;
    // The kernel before let this one start when the kernels before it had ended: the requests' counts stand.  Every thread waits before
    // it returns all the same: who waits for this kernel waits for that one by it.
    const Request rq = request_of<KEYS>(a, r, ratio, TILE_ROWS);
    const long long first_item = (long long)blockIdx.x * EACH;
    if (first_item >= (long long)rq.count * heads) return pdl_wait();
    // (The place of this request's items: before it lie those of the requests 0 .. r - 1.)
    int items, request_at;
    const int all = all_places<KEYS, OPEN>(a, requests, ratio, TILE_ROWS, kv_heads, items, r, request_at), blocks = working_blocks<OPEN>(all, items, grid, RUNS);
    const long long item = first_item + threadIdx.x / LANES;
    if (item >= (long long)rq.count * heads) return pdl_wait();
    const int row = (int)item / heads, head = (int)item % heads, kv = head / ratio, pair = row * ratio + head % ratio, d = 4 * (threadIdx.x % LANES);
    const int x0 = request_at + (pair / TILE_ROWS * kv_heads + kv) * (rq.tiles + OPEN), x1 = x0 + rq.tiles + OPEN;
    auto block_of = [&](int x) { return (int)(((unsigned long long)(x + 1) * blocks - 1) / all); };
    const int b0 = block_of(x0 + OPEN), b1 = block_of(x1 - 1);       // of the first tile and the last
    pdl_wait();
    if (b0 == b1) return;
    const int slot0 = 2 * b0 + (share_begins(all, blocks, b0) > x0 ? 0 : 1);
    const float* base = partial + (size_t)(pair % TILE_ROWS) * ROWF;
    auto state = [&](int b) { return base + (size_t)(b == b0 ? slot0 : 2 * b) * TILE_ROWS * ROWF; };
    // A lane has the maxima and sum of one of LANES states, and its four values of all of them, AT_ONCE asked for at one time: what this
    // takes is the trips to memory.  Sixteen where few rows share many blocks (37 states a row of 1 x 32,768 keys: the call 23.5 us,
    // with eight 24.3, with every lane reading all states' maxima first 26.0), but their registers cost where many rows share a few
    // (8 x 4,096 keys of 64 pairs: 56 us, with eight 52.5).
    constexpr int AT_ONCE = TILE_ROWS == 16 ? 16 : 8;
    const int lane = threadIdx.x % LANES;
    const unsigned together = LANES == 32 ? 0xffffffffu : 0xffffu << (threadIdx.x & 16);
    float4 v[AT_ONCE];
    auto ask = [&](int b) {
#pragma unroll
        for (int n = 0; n < AT_ONCE; ++n)
            if (b + n <= b1) v[n] = *reinterpret_cast<const float4*>(state(b + n) + d);
    };
    auto ends = [&](int b) { return b + lane <= b1 ? *reinterpret_cast<const float4*>(state(b + lane) + D) : make_float4(-INFINITY, -INFINITY, 0.f, 0.f); };
    const float4 mine = ends(b0);
    ask(b0);
    float t = mine.x, most = mine.y;
    for (int b = b0 + LANES; b <= b1; b += LANES) {
        const float4 m = ends(b);
        t = fmaxf(t, m.x), most = fmaxf(most, m.y);
    }
#pragma unroll
    for (int o = 1; o < LANES; o <<= 1) t = fmaxf(t, __shfl_xor_sync(together, t, o)), most = fmaxf(most, __shfl_xor_sync(together, most, o));
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float l = 0.0f;
    for (int b = b0; b <= b1; b += LANES) {
        const float4 m = b == b0 ? mine : ends(b);
        const float f = share(m.x, t);
        l = fmaf(m.z, share(m.y, most), l);
#pragma unroll
        for (int k = 0; k < LANES; k += AT_ONCE) {
            if (b + k > b1) break;
#pragma unroll
            for (int n = 0; n < AT_ONCE; ++n) {
                const float fn = __shfl_sync(together, f, k + n, LANES);
                if (b + k + n <= b1) acc.x = fmaf(v[n].x, fn, acc.x), acc.y = fmaf(v[n].y, fn, acc.y), acc.z = fmaf(v[n].z, fn, acc.z), acc.w = fmaf(v[n].w, fn, acc.w);
            }
            ask(b + k + AT_ONCE);
        }
    }
#pragma unroll
    for (int o = 1; o < LANES; o <<= 1) l += __shfl_xor_sync(together, l, o);
    write4(out + ((size_t)(rq.start + row) * heads + head) * D + d, finished<EIGHT>(acc, t, most, l));
}

}  // namespace mma_pages
