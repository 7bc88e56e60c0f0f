// Attention over pages on the tensor cores of tcgen05: few rows a request, heads of 128; trees of drafted tokens over bfloat16 pages, and
// over eight bits more than 32 (row, head) pairs.
//
// The warp form (attention_pages_mma.cuh) spends its time on turning codes into halves, again for every 16 rows, and moving them through
// registers.  Here neither keys nor values pass through registers at all: TMA brings 128 keys of a head to shared memory as they lie in their pages, and the
// matrix instruction reads codes (kind::f8f6f4; bfloat16 pages: kind::f16) from there, keys and values on its 128-row side:
//     S^T [128 keys, rows] = K Q^T           K as it lies, K-major
//     O^T [128 values, rows] += V^T W^T      V as it lies, MN-major; W^T [keys, rows] written by the softmax warps, MN-major
// A request's rows are the narrow side, 16 at a time: what is idle is not the instruction's 128 rows but its columns, which cost
// nothing.  A softmax thread has one key and all rows, so that a key's power of two is its thread's own.
//
// Eight bits on both sides: a query is two codes that add up to it, q = (q1 + q2 / 32) 2^e (bfloat16 has 8 bits, a code 4: exact down
// to 2^-22 of the row's largest), a weight, by then a half (11 bits), three, w = w1 + w2 / 32 + w3 / 1024 (down to 2^-20 of the largest):
// columns of their own, whose sums are added up in 32 bits.  As in the warp form a value's power of two belongs to its key's weight; a row of zeros and a page
// that is not there count with 2^-126.
//
//   warps 0, 10     page lookups and copies, STAGES tiles ahead, every other tile each: 16 keys and their values a copy (a warp issues
//                   one in some 100 clocks, which by itself would be less than memory gives)
//   warp 1          matrix instructions, whichever can be made next: S^T of tiles ahead, O^T
//   warp 11         an item's queries, while the item before is worked on (the first item's are the softmax warps' work)
//   warps 2 .. 9    two units of four warps: exponentials, weights to shared memory.  A tile takes a unit much longer than it takes to
//                   copy, most of it in waits for one thing after another, so the units have every other tile each (SHARED: a
//                   tile's rows are R; their states meet at the item's end), or half of the rows each (2 R)
// The maxima that the exponentials use are those of the first tile; a tile in which some weight would pass 2^8 of them (or a sum's exponential
// 2^96, where values are so small that its weight does not) has the unit raise them, and its sums and outputs (in tensor memory)
// scaled.  Every wait is bounded; the softmax warps go on through their
// barriers without waiting once one has run out.
//
// Work is cut evenly as in the warp form, one block an SM, tiles of 128 keys.
//
// Measured with the kernel that adds up (32 heads over 8): trees of 16 tokens for 8 requests after 4,096 keys of eight bits 52.5 us, one of 63 after
// 8,191 of bfloat16 46, one token each after 8 x 8,191 of bfloat16 60 (4.5 TB/s).  A tile of 64 rows over eight bits takes 3,300 clocks: 500 until a
// unit has begun, 650 to read scores, 800 for exponentials and weights, 1,000 to store these, the rest between (barriers, sums); the tensor pipe is 8 % busy, and two softmax warps a
// scheduler are what registers allow (four units of 16 rows, 96 registers a thread: 57 and 52 us).
#pragma once
#include "attention_pages_mma.cuh"
#include "attn_common.cuh"

namespace tc_pages {

using mma_pages::copy16;
using mma_pages::exp2_fast;
using mma_pages::max3;
using mma_pages::PART;
using mma_pages::Rows;

constexpr int KEYS = 128, D = 128;
constexpr int OPEN = 5;                 // tiles that an item's beginning and end take as long as
constexpr int UNIT_WARPS = 4, LOADER = 10, QUERIES = 11;
// The exponentials' references.  A weight is 1 at the maximum, and up to 2^8 before that is raised (what a code leaves of it is then 8 at
// most, of which 32 is a code again); over bfloat16, which has the exponents, up to 2^60.  The sum's exponentials are 2^64 at the
// maximum: a weight is made from one by its value's power and its row's, which may be 2^120 apart, and must not be lost before.
constexpr float ROOM = 64.0f;
constexpr float NONE = -1.0e30f;        // a maximum of no keys
// What values of nothing count as, to base 2, in the weights' reference: little enough to leave values their bits beside a key of zeros that
// is 2^(126 - 60) times as heavy, and a row's power (up to 2^(126 - ROOM)) times a key's (up to 2^60) is within 32 bits.
constexpr int NOTHING = -126;
enum : int { ERR_PAGES_PRODUCER = 501, ERR_PAGES_MMA = 502, ERR_PAGES_SOFTMAX = 503 };

template <bool EIGHT, bool SHARED, int R>
struct Shape {
    static constexpr int U = 2;
    static constexpr int THREADS = 128 + U * UNIT_WARPS * 32;
    // A stage: eight keys, their values, the next eight keys, ..., rows of 128 bytes; bfloat16: such a half for the rows' first 64 values
    // and one for the others.
    static constexpr int HALF = 2 * KEYS * 128, STAGE = EIGHT ? HALF : 2 * HALF;
    // As many stages as there is room for: a stage is taken for some 5,000 clocks, a third of them until its copies have come, and
    // memory gives one in 1,000.
    static constexpr int STAGES = EIGHT ? 5 : 2;
    // A tile's weights: rows of 128 bytes a key, of which a unit has one half (bfloat16), or all.
    static constexpr int WEIGHTS = KEYS * 128;
    static constexpr bool HALVES = !EIGHT;
    static_assert(!EIGHT || !SHARED, "few rows over eight bits are the warp form's");
    static constexpr int ROWS = SHARED ? R : U * R;             // of an item
    static constexpr int Q_BYTES = 2 * R * D;                   // R rows' queries: two codes each, or bfloat16
    static constexpr int Q_BUFFERS = SHARED ? 2 : 1;            // (two would not fit)
    static constexpr int S_COLS = EIGHT ? 2 * R : R, O_COLS = EIGHT ? 3 * R : R, U_COLS = 2 * S_COLS + O_COLS;
    static constexpr int TMEM = U * U_COLS <= 64 ? 64 : U * U_COLS <= 128 ? 128 : U * U_COLS <= 256 ? 256 : 512;
    static constexpr int AT_WEIGHTS = STAGES * STAGE, AT_QUERIES = AT_WEIGHTS + (HALVES ? 1 : U) * WEIGHTS, AT_EXPONENTS = AT_QUERIES + Q_BUFFERS * (ROWS / R) * Q_BYTES;
    // What a unit's threads tell each other, in floats: minus the sum's reference, the weights' beside it, what raising scales the two by,
    // what the item's end scales its outputs and the other unit's by, 2^(the second) [R]; maxima and sums of warps [2][4][R]; the least
    // 2^(the second) (and three unused).
    static constexpr int UNIT_FLOATS = 7 * R + 2 * UNIT_WARPS * R + 4;
    static constexpr float LIMIT = EIGHT ? 256.0f : 0x1p60f, SUM_LIMIT = 0x1p96f;
    static constexpr int AT_FLOATS = AT_EXPONENTS + STAGES * 256;
    // What the queries' warp tells, of an item's rows: factors, positions, rows of the output (-1: none).
    static constexpr int AT_ROWS = AT_FLOATS + U * UNIT_FLOATS * 4;
    static constexpr int AT_STRAY = AT_ROWS + Q_BUFFERS * 3 * ROWS * 4;                 // [rows][D] products with values that are no numbers
    static constexpr int AT_BARRIERS = AT_STRAY + (EIGHT ? 0 : U * R * D * 4);
    static constexpr int BYTES = AT_BARRIERS + 512 + 1024;                              // and to the next 1024
};

// MN-major operand of bytes or 16-bit values under the 128-byte swizzle: 128 bytes of the MN dimension in a row, rows of the K dimension 128
// bytes apart, groups of eight `eight_rows`, the MN dimension's next 128 bytes `block` further.
__device__ __forceinline__ uint64_t desc_mn(uint32_t at, uint32_t block, uint32_t eight_rows) {
    return (uint64_t)((at & 0x3FFFFu) >> 4) | ((uint64_t)(block >> 4) << 16) | ((uint64_t)(eight_rows >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// K-major, rows of 128 bytes, groups of eight 2048 bytes apart (a stage's keys).
__device__ __forceinline__ uint64_t desc_keys(uint32_t at) { return (uint64_t)((at & 0x3FFFFu) >> 4) | (1ull << 16) | (128ull << 32) | (1ull << 46) | (2ull << 61); }
constexpr uint32_t TRANSPOSED = (1u << 15) | (1u << 16);
// kind::f8f6f4, e4m3 on both sides, 32-bit sums.
__host__ __device__ constexpr uint32_t instruction_e4m3(int m, int n) { return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24); }
__device__ __forceinline__ void mma_e4m3(uint32_t d, uint64_t a, uint64_t b, uint32_t instruction, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(instruction), "r"(accumulate)
        : "memory");
}
// An arrival once this thread's asynchronous copies so far have landed (one of those that the barrier counts).
__device__ __forceinline__ void arrive_after_copies(uint64_t* bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(tc::smem_u32(bar)) : "memory");
}
__device__ __forceinline__ bool is_done(uint64_t* bar, uint32_t parity) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(tc::smem_u32(bar)), "r"(parity)
        : "memory");
    return done != 0;
}
__device__ __forceinline__ float warp_most(float v) {            // NaN aside
    float r;
    asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float warp_least(float v) {
    float r;
    asm("redux.sync.min.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}
// A barrier of a unit's threads; true for all if it is for one.
__device__ __forceinline__ bool unit_any(int unit, bool mine) {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.u32 p, %1, 0;\n\t"
        "barrier.cta.red.or.pred q, %2, 128, p;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(r)
        : "r"((uint32_t)mine), "r"(1 + unit)
        : "memory");
    return r != 0;
}
__device__ __forceinline__ void units_barrier() { asm volatile("barrier.cta.sync 7, 256;" ::: "memory"); }      // of both units
__device__ __forceinline__ void unit_barrier(int unit) { asm volatile("barrier.cta.sync %0, 128;" ::"r"(1 + unit) : "memory"); }

__device__ __forceinline__ float4 shared4(uint32_t at) {
    float4 v;
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ float shared1(uint32_t at) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ void to_shared1(uint32_t at, float v) { asm volatile("st.shared.f32 [%0], %1;" ::"r"(at), "f"(v) : "memory"); }
__device__ __forceinline__ void to_shared4(uint32_t at, uint4 v) {
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ unsigned shared_byte(uint32_t at) {
    unsigned v;
    asm volatile("ld.shared.u8 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ float at4(const float4& v, int k) { return k == 0 ? v.x : k == 1 ? v.y : k == 2 ? v.z : v.w; }
// Value d of a bfloat16 row of a stage, its two halves apart, pieces of 16 bytes exchanged by the row's place.
template <int HALF>
__device__ __forceinline__ unsigned short* value_in(uint8_t* row, int key, int d) {
    return reinterpret_cast<unsigned short*>(row + (d >> 6) * HALF + (((d >> 3 & 7) ^ (key & 7)) << 4) + 2 * (d & 7));
}

// Two halves to two codes, the second value in the upper byte.
__device__ __forceinline__ uint32_t codes2(uint32_t halves) {
    unsigned short r;
    asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(r) : "r"(halves));
    return r;
}
// 16 halves (pairs) as 16 codes, and what is left of them times 32.
__device__ __forceinline__ uint4 take_codes(uint32_t (&h)[8], bool more) {
    uint32_t c[8];
    const __half2 scale = __floats2half2_rn(32.0f, 32.0f);
#pragma unroll
    for (int n = 0; n < 8; ++n) {
        c[n] = codes2(h[n]);
        if (more) {
            const uint32_t back = e4m3::halves((unsigned short)c[n]);
            const __half2 left = __hmul2(__hsub2(*reinterpret_cast<const __half2*>(&h[n]), *reinterpret_cast<const __half2*>(&back)), scale);
            h[n] = *reinterpret_cast<const uint32_t*>(&left);
        }
    }
    return make_uint4(c[0] | c[1] << 16, c[2] | c[3] << 16, c[4] | c[5] << 16, c[6] | c[7] << 16);
}

template <bool EIGHT, bool SHARED, int R>
__global__ void __launch_bounds__(Shape<EIGHT, SHARED, R>::THREADS, 1)
pages_kernel(const __grid_constant__ CUtensorMap map, const __nv_bfloat16* __restrict__ q, const uint8_t* __restrict__ exponents,
             __nv_bfloat16* __restrict__ out, float* __restrict__ partial, Rows a, int requests, int heads, int kv_heads, float scale_log2,
             int* error_word) {
    using S = Shape<EIGHT, SHARED, R>;
    constexpr int U = S::U, TILE_ROWS = SHARED ? R : U * R, ROWF = D + PART, STAGES = S::STAGES, CHUNKS = R / 16;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint64_t* full = (uint64_t*)(smem + S::AT_BARRIERS);        // [STAGES]
    uint64_t* empty = full + STAGES;                            // [STAGES]
    uint64_t* q_full = empty + STAGES;                          // [Q_BUFFERS]
    uint64_t* q_free = q_full + 2;                              // [Q_BUFFERS]
    uint64_t* s_full = q_free + 2;                              // [U][2]
    uint64_t* s_free = s_full + 2 * U;                          // [U][2]
    uint64_t* w_full = s_free + 2 * U;                          // [U]
    uint64_t* o_done = w_full + U;                              // [U]: O^T with these weights
    uint32_t* tmem_slot = (uint32_t*)(o_done + U);
    volatile int* abort_flag = (volatile int*)(tmem_slot + 1);
    volatile int* live = abort_flag + 1;                        // [STAGES]: which of the stage's runs of 16 keys are in the cache
    volatile int* stray_flag = live + STAGES;                   // [U]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int ratio = heads / kv_heads;

    if (threadIdx.x == 0) {
        for (int i = 0; i < STAGES; ++i) tc::mbar_init(&full[i], EIGHT ? 17 : 1), tc::mbar_init(&empty[i], 1);     // (copies' bytes; 16 lanes' exponents)
        for (int u = 0; u < U; ++u) {
            tc::mbar_init(&q_full[u], 1);
            tc::mbar_init(&q_free[u], 1 + U * UNIT_WARPS);
            for (int i = 0; i < 2; ++i) {
                tc::mbar_init(&s_full[2 * u + i], 1);
                tc::mbar_init(&s_free[2 * u + i], UNIT_WARPS);
            }
            tc::mbar_init(&w_full[u], UNIT_WARPS);
            tc::mbar_init(&o_done[u], 1);
            stray_flag[u] = 0;
        }
        *abort_flag = 0;
        tc::fence_barrier_init();
        tc::tma_prefetch_desc(&map);
    }
    if (warp == 1) {
        tc::tmem_alloc(tmem_slot, S::TMEM);
        tc::tmem_relinquish();
    }
    if constexpr (!EIGHT)
        for (int i = threadIdx.x; i < U * R * D / 4; i += S::THREADS) reinterpret_cast<float4*>(smem + S::AT_STRAY)[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    tc::fence_proxy_async();
    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    // Dependents may start only now that this block holds its tensor memory (they must not take what it waits for) and the kernels before
    // have ended (the merge reads the requests' counts without waiting).
    pdl_wait();
    pdl_trigger();

    // ---- the work, which every role walks alike
    mma_pages::Walk<KEYS, OPEN> sg(a, requests, ratio, TILE_ROWS, kv_heads, gridDim.x, 1);
    const int runs_a_page = a.page_size >> 4;
    auto page_of = [&](int sixteenth) { return (int)(((uint64_t)(unsigned)sixteenth * a.run_pages) >> 31); };

    // 16 of an item's rows' queries, two lanes a row, and what is to be known of the rows.
    auto lay_out = [&](int buffer, int row0) {
        float* info = reinterpret_cast<float*>(smem + S::AT_ROWS) + buffer * 3 * S::ROWS;
        const int part = lane & 1;
        const int item_row = row0 + (lane >> 1), row = item_row % R, pair = sg.first + item_row;
        const bool real = pair < sg.rq.pairs;
        const int token = real ? pair / ratio : 0, to_row = (sg.rq.start + token) * heads + sg.kv * ratio + (real ? pair - token * ratio : 0);
        const __nv_bfloat16* src = q + (size_t)to_row * D + part * 64;
        uint8_t* queries = smem + S::AT_QUERIES + (buffer * (S::ROWS / R) + item_row / R) * S::Q_BYTES;
        uint4 x[8];
#pragma unroll
        for (int n = 0; n < 8; ++n) x[n] = real ? reinterpret_cast<const uint4*>(src)[n] : make_uint4(0, 0, 0, 0);
        float f = scale_log2;
        if constexpr (EIGHT) {
            unsigned most = 0;                           // magnitudes of bfloat16 compare as their bits do
#pragma unroll
            for (int n = 0; n < 8; ++n) {
                const unsigned v[4] = {x[n].x, x[n].y, x[n].z, x[n].w};
#pragma unroll
                for (int k = 0; k < 4; ++k) most = max(most, max(v[k] & 0x7FFFu, v[k] >> 16 & 0x7FFFu));
            }
            most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
            const int e = min(max((int)(most >> 7) - 127, -100), 127);     // the row's largest lies in 2^e .. 2^(e + 1): to 2^7 .. 2^8
            const float up = __int_as_float((127 + 7 - e) << 23);
            f = fmaxf(__int_as_float((127 - 7 + e) << 23) * scale_log2, 1.0e-44f);     // (not zero: a masked score stays -inf)
            const bool bad = most >= 0x7F80u;            // a row with an infinity or a NaN: codes that are NaN
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                uint32_t one[4], two[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const uint4& from = x[2 * n + (k >> 1)];
                    const unsigned w0 = k & 1 ? from.z : from.x, w1 = k & 1 ? from.w : from.y;
                    const float v[4] = {__uint_as_float(w0 << 16) * up, __uint_as_float(w0 & 0xffff0000u) * up, __uint_as_float(w1 << 16) * up,
                                        __uint_as_float(w1 & 0xffff0000u) * up};
                    const unsigned c0 = e4m3::pack2(v[0], v[1]), c1 = e4m3::pack2(v[2], v[3]);
                    const float2 b0 = mma_pages::from_halves(e4m3::halves((unsigned short)c0)), b1 = mma_pages::from_halves(e4m3::halves((unsigned short)c1));
                    one[k] = bad ? 0x7F7F7F7Fu : c0 | c1 << 16;
                    two[k] = e4m3::pack2((v[0] - b0.x) * 32.0f, (v[1] - b0.y) * 32.0f) | e4m3::pack2((v[2] - b1.x) * 32.0f, (v[3] - b1.y) * 32.0f) << 16;
                }
                const int piece = part * 4 + n, r1 = (row >> 4) * 32 + (row & 15), r2 = r1 + 16;
                *reinterpret_cast<uint4*>(queries + r1 * 128 + ((piece ^ (r1 & 7)) << 4)) = make_uint4(one[0], one[1], one[2], one[3]);
                *reinterpret_cast<uint4*>(queries + r2 * 128 + ((piece ^ (r2 & 7)) << 4)) = make_uint4(two[0], two[1], two[2], two[3]);
            }
        } else {
#pragma unroll
            for (int n = 0; n < 8; ++n) *reinterpret_cast<uint4*>(queries + part * (R * 128) + row * 128 + ((n ^ (row & 7)) << 4)) = x[n];
        }
        if (part == 0) {
            info[item_row] = f;
            reinterpret_cast<int*>(info)[S::ROWS + item_row] = real ? sg.rq.history + token : -1;
            reinterpret_cast<int*>(info)[2 * S::ROWS + item_row] = real ? to_row : -1;
        }
    };

    if (warp == 0 || warp == LOADER) {
        const int p = lane & 7, plane = (lane >> 3) & 1;          // a run of 16 keys; for exponents, keys' or values'
        uint32_t use = 0;
        bool ok = true;
        while (ok && sg.next(a)) {
            const int* table = a.tables + (size_t)sg.r * a.table_stride;
            // The pages of four tiles' 32 runs at a time, a lane each, asked for four tiles ahead: a lookup takes as long as a tile.
            auto look_up = [&](int i) {
                const int n = (sg.from + i) * (KEYS / 16) + lane;
                return i + lane / 8 < sg.tiles && n * 16 < sg.rq.end && n * 16 + 16 > sg.rq.low ? table[page_of(n)] : -1;
            };
            int four = look_up(0), next_four = look_up(4);
            for (int i = 0; i < sg.tiles; ++i, ++use) {
                const int stage = use % STAGES, n = (sg.from + i) * (KEYS / 16) + p, page = __shfl_sync(0xffffffffu, four, (i & 3) * 8 + p);
                if ((i & 3) == 3) four = next_four, next_four = look_up(i + 5);
                if ((use & 1) != (warp == LOADER)) continue;
                const bool real = (unsigned)page < (unsigned)a.pages;
                const unsigned runs = __ballot_sync(0xffffffffu, real) & 0xffu;
                const int off = (n - page_of(n) * runs_a_page) * 16;
                ok = tc::mbar_wait_warp(&empty[stage], ((use / STAGES) & 1u) ^ 1u, abort_flag, error_word, ERR_PAGES_PRODUCER);
                if (!ok) break;
                if (lane == 0) {
                    live[stage] = (int)runs;
                    tc::mbar_expect_tx(&full[stage], (uint32_t)__popc(runs) * 2 * 16 * D * (EIGHT ? 1 : 2));
                }
                __syncwarp();
                // One lane makes all copies, from operands that are there before the first: waits between them would be as long as the copies.
                uint8_t* to = smem + stage * S::STAGE;
                const int eights = (sg.kv * a.page_size + off) >> 3;
                int y[8], at_page[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) y[k] = __shfl_sync(0xffffffffu, eights, k), at_page[k] = __shfl_sync(0xffffffffu, page, k);
                if (lane == 0) {
                    if (runs == 0xffu) {
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            tc::tma_load_5d(to + k * 4096, &map, 0, 0, 0, y[k], at_page[k], &full[stage]);
                            if (!EIGHT) tc::tma_load_5d(to + S::HALF + k * 4096, &map, 64, 0, 0, y[k], at_page[k], &full[stage]);
                        }
                    } else {
#pragma unroll
                        for (int k = 0; k < 8; ++k)
                            if (runs >> k & 1u) {
                                tc::tma_load_5d(to + k * 4096, &map, 0, 0, 0, y[k], at_page[k], &full[stage]);
                                if (!EIGHT) tc::tma_load_5d(to + S::HALF + k * 4096, &map, 64, 0, 0, y[k], at_page[k], &full[stage]);
                            }
                    }
                }
                __syncwarp();
                if (EIGHT && lane < 16) {
                    const unsigned row = (((unsigned)(real ? page : 0) * 2 + plane) * kv_heads + sg.kv) * a.page_size + off;
                    if (real) copy16(tc::smem_u32(smem + S::AT_EXPONENTS + stage * 256 + plane * KEYS + p * 16), exponents + row);
                    arrive_after_copies(&full[stage]);
                }
            }
        }
    } else if (warp == QUERIES) {
        // An item's queries while the one before it is worked on: two lanes a row.
        uint32_t segment = 0;
        bool ok = true;
        for (; sg.next(a); ++segment) {
            if (segment == 0) continue;                          // (the softmax warps lay out the first)
            const int buffer = segment % S::Q_BUFFERS;
            ok = tc::mbar_wait_warp(&q_free[buffer], ((segment / S::Q_BUFFERS) & 1u) ^ 1u, abort_flag, error_word, ERR_PAGES_PRODUCER);
            if (!ok) break;
            for (int row0 = 0; row0 < S::ROWS; row0 += 16) lay_out(buffer, row0);
            tc::fence_proxy_async();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(&q_full[buffer]);
        }
    } else if (warp == 1) {
        if (tc::elect_one()) {
            uint32_t use = 0, segments = 0, scored[U] = {0, 0}, weighed[U] = {0, 0};       // tiles so far; units' S^T and O^T so far
            bool ok = true;
            while (ok && sg.next(a)) {
                const int q_buffer = segments % S::Q_BUFFERS;
                ok = tc::mbar_wait(&q_full[q_buffer], (segments / S::Q_BUFFERS) & 1u, abort_flag, error_word, ERR_PAGES_MMA);
                ++segments;
                tc::tc_fence_after();
                // S^T of tile `next`, O^T of `tile` (of unit `turn`, where both units have every tile): whichever finds what it needs.
                int next = 0, tile = 0, turn = 0;
                unsigned long long since = 0;
                for (uint32_t idle = 0; tile < sg.tiles && ok;) {
                    bool made = false;
                    if (next < sg.tiles) {
                        const int stage = (use + next) % STAGES, u0 = SHARED ? next & 1 : 0, u1 = SHARED ? u0 : U - 1;
                        bool ready = is_done(&full[stage], ((use + next) / STAGES) & 1u);
                        for (int u = u0; u <= u1; ++u) ready = ready && is_done(&s_free[2 * u + (scored[u] & 1)], ((scored[u] >> 1) & 1u) ^ 1u);
                        if (ready) {
                            tc::tc_fence_after();
                            const uint32_t keys = tc::smem_u32(smem + stage * S::STAGE);
                            for (int u = u0; u <= u1; ++u) {
                                const int buffer = scored[u]++ & 1;
                                const uint32_t queries = tc::smem_u32(smem + S::AT_QUERIES + (q_buffer * (S::ROWS / R) + (SHARED ? 0 : u)) * S::Q_BYTES), d = tmem + u * S::U_COLS + buffer * S::S_COLS;
                                if constexpr (EIGHT) {
#pragma unroll
                                    for (int k = 0; k < D / 32; ++k)
                                        mma_e4m3(d, desc_keys(keys + k * 32), tc::smem_desc_k_sw128(queries + k * 32), instruction_e4m3(KEYS, 2 * R),
                                                 k > 0);
                                } else {
#pragma unroll
                                    for (int k = 0; k < D / 16; ++k)
                                        tc::mma_bf16_ss(d, desc_keys(keys + (k >> 2) * S::HALF + (k & 3) * 32),
                                                        tc::smem_desc_k_sw128(queries + (k >> 2) * (R * 128) + (k & 3) * 32), tc::instr_desc_bf16(KEYS, R), k > 0);
                                }
                                tc::mma_commit(&s_full[2 * u + buffer]);
                            }
                            if (++next == sg.tiles) tc::mma_commit(&q_free[q_buffer]);
                            made = true;
                        }
                    }
                    if (tile < next) {
                        const int u = SHARED ? tile & 1 : turn, stage = (use + tile) % STAGES;
                        if (is_done(&w_full[u], weighed[u] & 1u)) {
                            tc::tc_fence_after();
                            const uint32_t values = tc::smem_u32(smem + stage * S::STAGE + 1024), d = tmem + u * S::U_COLS + 2 * S::S_COLS;
                            const uint32_t weights = tc::smem_u32(smem + S::AT_WEIGHTS + u * (S::HALVES ? 64 : S::WEIGHTS));
                            const bool begun = SHARED ? tile > 1 : tile > 0;
                            if constexpr (EIGHT) {
#pragma unroll
                                for (int k = 0; k < KEYS / 32; ++k)
                                    mma_e4m3(d, desc_mn(values + k * 8192, S::HALF, 2048), desc_mn(weights + k * 4096, S::WEIGHTS, 1024),
                                             instruction_e4m3(D, 3 * R) | TRANSPOSED, begun || k > 0);
                            } else {
#pragma unroll
                                for (int k = 0; k < KEYS / 16; ++k)
                                    tc::mma_bf16_ss(d, desc_mn(values + k * 4096, S::HALF, 2048), desc_mn(weights + k * 2048, S::WEIGHTS, 1024),
                                                    tc::instr_desc_bf16(D, R) | TRANSPOSED, begun || k > 0);
                            }
                            ++weighed[u];
                            const bool last = SHARED || turn == U - 1;
                            if (last) tc::mma_commit(&empty[stage]);
                            tc::mma_commit(&o_done[u]);
                            turn = last ? 0 : turn + 1;
                            tile += last;
                            made = true;
                        }
                    }
                    if (made) {
                        idle = 0;
                    } else if ((++idle & 255u) == 0) {
                        const unsigned long long now = tc::global_ns();
                        if (idle == 256) since = now;
                        if (*abort_flag) ok = false;
                        else if (now - since > tc::WAIT_LIMIT_NS) {
                            *abort_flag = 1;
                            if (error_word) atomicCAS(error_word, 0, ERR_PAGES_MMA);
                            ok = false;
                        }
                    }
                }
                use += sg.tiles;
            }
        }
    } else {
        const int unit = (warp - 2) / UNIT_WARPS, quarter = warp & 3, key = quarter * 32 + lane;
        const int thread = ((warp - 2) % UNIT_WARPS) * 32 + lane;               // of the unit, for what is shared out among its threads
        const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
        const uint32_t s_at = tmem + unit * S::U_COLS + lanes, o_at = s_at + 2 * S::S_COLS;
        float* shared = reinterpret_cast<float*>(smem + S::AT_FLOATS) + unit * S::UNIT_FLOATS;
        float *minus_peak = shared, *shift = shared + R, *fade_sum = shared + 2 * R, *fade_o = shared + 3 * R, *own_scale = shared + 4 * R,
              *given_scale = shared + 5 * R, *power = shared + 6 * R, *warp_peak = shared + 7 * R, *warp_top = warp_peak + UNIT_WARPS * R,             // [4][R]
              *least_power = warp_top + UNIT_WARPS * R;
        float* strays = reinterpret_cast<float*>(smem + S::AT_STRAY) + unit * R * D;
        const uint32_t live_at = tc::smem_u32((const void*)live), rows_at = tc::smem_u32(shared), exponents_at = tc::smem_u32(smem + S::AT_EXPONENTS);
        const uint32_t weights_at = tc::smem_u32(smem + S::AT_WEIGHTS + (S::HALVES ? 0 : unit * S::WEIGHTS)) + key * 128;
        const float* rows_info = reinterpret_cast<const float*>(smem + S::AT_ROWS) + (SHARED ? 0 : unit * R);
        uint32_t before = 0, mine = 0, segment = 0;             // tiles of the items before; this unit's so far; items
        bool ok = true;
        for (; sg.next(a); before += sg.tiles, ++segment) {
            const int first = sg.first + (SHARED ? 0 : unit * R), pairs = sg.rq.pairs, history = sg.rq.history, start = sg.rq.start;
            const int q_buffer = segment % S::Q_BUFFERS;
            if (segment == 0) {
                if (warp - 2 < S::ROWS / 16) lay_out(0, 16 * (warp - 2));
                tc::fence_proxy_async();
                units_barrier();
                if (warp == 2 && lane == 0) tc::mbar_arrive(&q_full[0]);
            }
            if (ok) ok = tc::mbar_wait_warp(&q_full[q_buffer], (segment / S::Q_BUFFERS) & 1u, abort_flag, error_word, ERR_PAGES_SOFTMAX);
            const float* factor = rows_info + q_buffer * 3 * S::ROWS;
            const int *position = reinterpret_cast<const int*>(factor) + S::ROWS, *out_row = position + S::ROWS;
            const uint32_t factors_at = tc::smem_u32(factor);
            const int row0 = first / ratio, row1 = max(row0, (min(first + R, pairs) - 1) / ratio);
            const int all_to = a.tree ? min(history, sg.rq.end) : min(history + row0 + 1, sg.rq.end);
            const int all_from = a.window > 0 ? max(history + row1 - a.window + 1, 0) : 0;

            float sum[R];
#pragma unroll
            for (int n = 0; n < R; ++n) sum[n] = 0.0f;
            for (int i = SHARED ? unit : 0; i < sg.tiles; i += SHARED ? 2 : 1, ++mine) {
                const bool opening = i < (SHARED ? 2 : 1);       // the unit's first tile of the item
                const uint32_t use = before + i;
                const int stage = use % STAGES, s_buffer = mine & 1;
                const int t0 = (sg.from + i) * KEYS, t = t0 + key;
                // The tile's copies, its scores, and whether the weights' place is free again (which is not needed yet): asked for together,
                // since an answer takes long.
                bool free_again = mine == 0;
                if (ok) {
                    const bool a0 = is_done(&full[stage], (use / STAGES) & 1u), a1 = is_done(&s_full[2 * unit + s_buffer], (mine >> 1) & 1u);
                    free_again = __all_sync(0xffffffffu, free_again || is_done(&o_done[unit], (mine & 1u) ^ 1u));
                    if (!__all_sync(0xffffffffu, a0 && a1)) {
                        ok = tc::mbar_wait_warp(&full[stage], (use / STAGES) & 1u, abort_flag, error_word, ERR_PAGES_SOFTMAX);
                        if (ok) ok = tc::mbar_wait_warp(&s_full[2 * unit + s_buffer], (mine >> 1) & 1u, abort_flag, error_word, ERR_PAGES_SOFTMAX);
                    }
                }
                auto weights_place = [&]() {                     // every O^T that has been asked for has been made
                    if (!free_again && ok) ok = tc::mbar_wait_warp(&o_done[unit], (mine & 1u) ^ 1u, abort_flag, error_word, ERR_PAGES_SOFTMAX);
                    free_again = true;
                    tc::tc_fence_after();
                };
                tc::tc_fence_after();
                int runs;
                asm volatile("ld.shared.s32 %0, [%1];" : "=r"(runs) : "r"(live_at + 4 * stage) : "memory");
                const bool dead = !(runs >> (key >> 4) & 1);     // a page that is not in the cache: a key of zeros
                float k_power = 1.0f, v_power = 1.0f, v_exponent = 0.0f;
                if constexpr (EIGHT) {
                    const uint32_t b = exponents_at + stage * 256 + key;
                    const unsigned kb = shared_byte(b), vb = shared_byte(b + KEYS);
                    bool nothing = dead;
                    if (!dead && vb == 127) {                    // the byte of a row of zeros
                        unsigned any = 0;
#pragma unroll 1
                        for (int n = 0; n < 8 && !any; ++n) {
                            const uint4 v = *reinterpret_cast<const uint4*>(smem + stage * S::STAGE + (key >> 3) * 2048 + 1024 + (key & 7) * 128 + n * 16);
                            any = (v.x | v.y | v.z | v.w) & 0x7F7F7F7Fu;
                        }
                        nothing = !any;
                    }
                    // A value that is no number makes its key none: NaN for the rows that see it.
                    k_power = dead ? 0.0f : vb == e4m3::NOT_NUMBERS ? NAN : e4m3::up(kb);
                    const int n = nothing ? NOTHING : vb == e4m3::NOT_NUMBERS ? 0 : (int)vb - 127;
                    v_power = __uint_as_float((unsigned)(n + 127) << 23);
                    v_exponent = (float)n;
                }
                const bool whole = t0 >= all_from && t0 + KEYS <= all_to && runs == 0xff;
                const bool in_reach = t >= sg.rq.low && t < sg.rq.end;
                uint8_t* value_row = smem + stage * S::STAGE + (key >> 3) * 2048 + 1024 + (key & 7) * 128;
                bool stray = false;
                unsigned hidden = 0;                             // rows that do not see this key
                if (!whole) {
                    if (dead || !in_reach) {
                        // Values that nobody sees must be numbers, those of a page that is not there zeros.
#pragma unroll
                        for (int n = 0; n < (EIGHT ? 8 : 16); ++n)
                            *reinterpret_cast<uint4*>(value_row + (n >> 3) * S::HALF + (n & 7) * 16) = make_uint4(0, 0, 0, 0);
                    } else if (!EIGHT && a.tree && t >= history) {
                        // Values that are no numbers, of a key that not every row sees: their products are added up beside the others, for
                        // the rows that do, and zeros take their place (a weight of zero times an infinity is no zero).
#pragma unroll
                        for (int n = 0; n < 16; ++n) {
                            const uint4 v = *reinterpret_cast<const uint4*>(value_row + (n >> 3) * S::HALF + (n & 7) * 16);
                            const unsigned x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                            for (int k = 0; k < 4; ++k) stray |= (x[k] & 0x7F80u) == 0x7F80u || (x[k] & 0x7F800000u) == 0x7F800000u;
                        }
                    }
                    for (int n = 0; n < R; ++n) {
                        const int pos = position[n];
                        bool sees = in_reach && pos >= 0;
                        if (a.tree) {
                            if (sees && t >= history)
                                sees = (a.tree[(size_t)(start + pos - history) * a.tree_words + ((t - history) >> 5)] >> ((t - history) & 31)) & 1u;
                        } else {
                            sees = sees && t <= pos && (a.window <= 0 || t > pos - a.window);
                        }
                        if (!sees) hidden |= 1u << n;
                    }
                }
                // ---- what the sum's exponentials are of: scores, less the row's reference
                float x[R];
                auto scores = [&](bool raw) {
#pragma unroll
                    for (int c = 0; c < CHUNKS; ++c) {
                        float z[16];
                        if constexpr (EIGHT) {
                            uint32_t v[32];
                            tc::tmem_ld_32x32(s_at + s_buffer * S::S_COLS + 32 * c, v);
                            tc::tmem_wait_ld();
#pragma unroll
                            for (int n = 0; n < 16; ++n) z[n] = fmaf(__uint_as_float(v[16 + n]), 1.0f / 32.0f, __uint_as_float(v[n])) * k_power;
                        } else {
                            uint32_t v[16];
                            tc::tmem_ld_32x16(s_at + s_buffer * S::S_COLS + 16 * c, v);
                            tc::tmem_wait_ld();
#pragma unroll
                            for (int n = 0; n < 16; ++n) z[n] = __uint_as_float(v[n]);
                        }
                        if (!whole) {
#pragma unroll
                            for (int n = 0; n < 16; ++n) z[n] = hidden >> (16 * c + n) & 1u ? -INFINITY : dead ? 0.0f : z[n];
                        }
#pragma unroll
                        for (int n = 0; n < 16; n += 4) {
                            const float4 f = shared4(factors_at + 4 * (16 * c + n)),
                                         mp = raw ? make_float4(0.f, 0.f, 0.f, 0.f) : shared4(rows_at + 4 * (16 * c + n));
                            x[16 * c + n] = fmaf(z[n], f.x, mp.x), x[16 * c + n + 1] = fmaf(z[n + 1], f.y, mp.y);
                            x[16 * c + n + 2] = fmaf(z[n + 2], f.z, mp.z), x[16 * c + n + 3] = fmaf(z[n + 3], f.w, mp.w);
                        }
                    }
                };
                scores(opening);                                 // (the first tile has no references yet)
                // ---- exponentials (in place of what they are of) and weights, two halves (bfloat16 values) to a register
                uint32_t h[R / 2];
                auto weights = [&]() -> float {                  // the largest weight
                    float most = 0.0f;
#pragma unroll
                    for (int n = 0; n < R; n += 4) {
                        float w[4];
                        const float4 s = EIGHT ? shared4(rows_at + 4 * (6 * R + n)) : make_float4(1.f, 1.f, 1.f, 1.f);
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            x[n + k] = exp2_fast(x[n + k]);
                            w[k] = EIGHT ? x[n + k] * (at4(s, k) * v_power) : x[n + k];
                        }
                        most = max3(max3(most, w[0], w[1]), w[2], w[3]);
#pragma unroll
                        for (int k = 0; k < 4; k += 2) h[(n + k) / 2] = EIGHT ? mma_pages::pack_half(w[k], w[k + 1]) : mma_pages::pack_bf16(w[k], w[k + 1]);
                    }
                    return most;
                };
                bool raise = opening;
                if (!opening) {
                    bool over = weights() > S::LIMIT;
                    // (Weights up to the limit are of exponentials up to the sums' wherever their factor is no less than the limits' ratio.)
                    if (EIGHT && v_power * *least_power < S::LIMIT / S::SUM_LIMIT)
#pragma unroll
                        for (int n = 0; n < R; ++n) over |= x[n] > S::SUM_LIMIT;
                    raise = unit_any(unit, over);
                    if (raise) scores(true);
                }
                if (raise) {
                    // ---- the references rise to this tile's maxima
#pragma unroll
                    for (int n = 0; n < R; ++n) {
                        const float p = warp_most(x[n]), w = EIGHT ? warp_most(x[n] + v_exponent) : p;
                        if (lane == 0) warp_peak[quarter * R + n] = p, warp_top[quarter * R + n] = w;
                    }
                    unit_barrier(unit);
                    if (thread < R) {
                        const int n = thread;
                        float p = NONE, w = NONE;
#pragma unroll
                        for (int k = 0; k < UNIT_WARPS; ++k) p = fmaxf(p, warp_peak[k * R + n]), w = fmaxf(w, warp_top[k * R + n]);
                        const float old = opening ? NONE : -minus_peak[n], now = fmaxf(old, EIGHT && p > NONE ? p - ROOM : p);
                        const float top_old = opening ? NONE : old - shift[n], top_now = EIGHT ? fmaxf(top_old, w) : now;
                        fade_sum[n] = exp2_fast(old - now);
                        fade_o[n] = EIGHT ? exp2_fast(top_old - top_now) : fade_sum[n];
                        minus_peak[n] = -now, shift[n] = now - top_now, power[n] = exp2_fast(now - top_now);
                        if constexpr (EIGHT) {
                            static_assert(R == 32, "one warp has a unit's rows");
                            const float least = warp_least(power[n]);
                            if (lane == 0) *least_power = least;
                        }
                    }
                    unit_barrier(unit);
#pragma unroll
                    for (int n = 0; n < R; n += 4) {
                        const float4 mp = shared4(rows_at + 4 * n);
                        x[n] += mp.x, x[n + 1] += mp.y, x[n + 2] += mp.z, x[n + 3] += mp.w;
                    }
                    weights();
                    if (!opening) {
                        weights_place();
#pragma unroll
                        for (int n = 0; n < R; ++n) sum[n] *= fade_sum[n];
#pragma unroll
                        for (int c = 0; c < S::O_COLS / 16; ++c) {
                            uint32_t v[16];
                            tc::tmem_ld_32x16(o_at + 16 * c, v);
                            tc::tmem_wait_ld();
#pragma unroll
                            for (int n = 0; n < 16; ++n) v[n] = __float_as_uint(__uint_as_float(v[n]) * fade_o[(EIGHT ? c / 3 : c) * 16 + n]);
                            tc::tmem_st_32x16(o_at + 16 * c, v);
                        }
                        tc::tmem_wait_st();
                    }
                }
                tc::tc_fence_before();
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(&s_free[2 * unit + s_buffer]);
                // ---- the weights to shared memory
                weights_place();
                constexpr int SKIP = S::HALVES ? 4 : 0;          // pieces of 16 bytes to the second unit's half
#pragma unroll
                for (int n = 0; n < R; ++n) sum[n] += x[n];
                if constexpr (!EIGHT)
                    if (stray) {
#pragma unroll
                        for (int row = 0; row < R; ++row) {
                            if (hidden >> row & 1u) continue;
                            for (int d = 0; d < D; ++d) {
                                const unsigned v = *value_in<S::HALF>(value_row, key, d);
                                if ((v & 0x7F80u) == 0x7F80u) atomicAdd(strays + row * D + d, x[row] * __uint_as_float(v << 16));
                            }
                        }
                        stray_flag[unit] = 1;
                    }
#pragma unroll
                for (int c = 0; c < CHUNKS; ++c) {
                    if constexpr (EIGHT) {
                        uint32_t left[8];
#pragma unroll
                        for (int n = 0; n < 8; ++n) left[n] = h[8 * c + n];
#pragma unroll
                        for (int k = 0; k < 3; ++k) to_shared4(weights_at + (((SKIP * unit + 3 * c + k) ^ (key & 7)) << 4), take_codes(left, k < 2));
                    } else {
#pragma unroll
                        for (int k = 0; k < 2; ++k)
                            to_shared4(weights_at + (((SKIP * unit + 2 * c + k) ^ (key & 7)) << 4),
                                       make_uint4(h[8 * c + 4 * k], h[8 * c + 4 * k + 1], h[8 * c + 4 * k + 2], h[8 * c + 4 * k + 3]));
                    }
                }
                if constexpr (!EIGHT)
                    if (a.tree && t0 + KEYS > history) {
                        // No unit takes such values away before all have read them.
                        if (!SHARED) units_barrier();
                        if (stray)
                            for (int d = 0; d < D; ++d) {
                                unsigned short* x = value_in<S::HALF>(value_row, key, d);
                                if ((*x & 0x7F80u) == 0x7F80u) *x = 0;
                            }
                    }
                tc::fence_proxy_async();
                tc::tc_fence_before();
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(&w_full[unit]);
            }

            // ---- the item's sums over this block's keys: a thread has one of the 128 values of every row
            const bool any_tile = !SHARED || unit < sg.tiles;    // (an item of one tile leaves the second unit none)
            const uint32_t last = mine - 1;
#pragma unroll
            for (int n = 0; n < R; ++n) {
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) sum[n] += __shfl_xor_sync(0xffffffffu, sum[n], o);
                if (lane == 0) warp_peak[quarter * R + n] = sum[n];
            }
            if (ok && any_tile) ok = tc::mbar_wait_warp(&o_done[unit], last & 1u, abort_flag, error_word, ERR_PAGES_SOFTMAX);
            tc::tc_fence_after();
            if (SHARED) units_barrier();
            else unit_barrier(unit);
            const bool any_stray = !EIGHT && stray_flag[unit], both = SHARED && sg.tiles > 1;
            // The second unit's sums go to the first by way of the weights' place, for which both have no more use.
            const uint32_t given_at = tc::smem_u32(smem + S::AT_WEIGHTS);
            float* slot = partial + ((2 * (size_t)blockIdx.x + sg.slot) * TILE_ROWS + (SHARED ? 0 : unit * R)) * ROWF;
            auto outputs = [&](int c, float (&o)[16]) {
                uint32_t v[16];
                tc::tmem_ld_32x16(o_at + (EIGHT ? 48 : 16) * c, v);
                tc::tmem_wait_ld();
#pragma unroll
                for (int n = 0; n < 16; ++n) o[n] = __uint_as_float(v[n]);
                if constexpr (EIGHT) {
                    tc::tmem_ld_32x16(o_at + 48 * c + 16, v);
                    tc::tmem_wait_ld();
#pragma unroll
                    for (int n = 0; n < 16; ++n) o[n] = fmaf(__uint_as_float(v[n]), 1.0f / 32.0f, o[n]);
                    tc::tmem_ld_32x16(o_at + 48 * c + 32, v);
                    tc::tmem_wait_ld();
#pragma unroll
                    for (int n = 0; n < 16; ++n) o[n] = fmaf(__uint_as_float(v[n]), 1.0f / 1024.0f, o[n]);
                }
                if (any_stray)
#pragma unroll
                    for (int n = 0; n < 16; ++n) o[n] += strays[(16 * c + n) * D + key];
            };
            if (SHARED && unit == 1) {
                if (both)
#pragma unroll
                    for (int c = 0; c < CHUNKS; ++c) {
                        float o[16];
                        outputs(c, o);
#pragma unroll
                        for (int n = 0; n < 16; ++n) to_shared1(given_at + ((16 * c + n) * D + key) * 4, o[n]);
                    }
            } else if (thread < R) {
                // A row's sum, and what its outputs are to be multiplied by.
                const int row = thread;
                auto total_of = [&](uint32_t sums) {
                    return (shared1(sums + 4 * row) + shared1(sums + 4 * (R + row))) + (shared1(sums + 4 * (2 * R + row)) + shared1(sums + 4 * (3 * R + row)));
                };
                float total = total_of(rows_at + 28 * R), peak = -shared1(rows_at + 4 * row), top = peak - shared1(rows_at + 4 * (R + row)), f = 1.0f, g = 0.0f;
                if (both) {
                    const uint32_t theirs = rows_at + S::UNIT_FLOATS * 4;
                    const float peak2 = -shared1(theirs + 4 * row), top2 = peak2 - shared1(theirs + 4 * (R + row)), p = fmaxf(peak, peak2), t = fmaxf(top, top2);
                    total = fmaf(total, exp2_fast(peak - p), total_of(theirs + 28 * R) * exp2_fast(peak2 - p));
                    f = exp2_fast(top - t), g = exp2_fast(top2 - t);
                    peak = p, top = t;
                }
                if (sg.whole) {
                    const float s = total == 0.0f ? 0.0f : __fdividef(EIGHT ? exp2_fast(top - peak) : 1.0f, total);
                    f *= s, g *= s;
                } else if (out_row[row] >= 0) {
                    float* to = slot + (size_t)row * ROWF + D;
                    to[0] = top, to[1] = peak, to[2] = total;
                }
                own_scale[row] = f, given_scale[row] = g;
            }
            if (SHARED) units_barrier();
            else unit_barrier(unit);
            if (!SHARED || unit == 0) {
#pragma unroll
                for (int c = 0; c < CHUNKS; ++c) {
                    float o[16];
                    outputs(c, o);
#pragma unroll
                    for (int n = 0; n < 16; n += 4) {
                        const int row = 16 * c + n;
                        const float4 f = shared4(rows_at + 4 * (4 * R + row)), g = shared4(rows_at + 4 * (5 * R + row)), to = shared4(factors_at + 4 * (2 * S::ROWS + row));
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            o[n + k] *= at4(f, k);
                            if (both) o[n + k] = fmaf(shared1(given_at + ((row + k) * D + key) * 4), at4(g, k), o[n + k]);
                            const int to_row = __float_as_int(at4(to, k));
                            if (to_row < 0) continue;
                            if (sg.whole) out[(size_t)to_row * D + key] = __float2bfloat16_rn(o[n + k]);
                            else slot[(size_t)(row + k) * ROWF + key] = o[n + k];
                        }
                    }
                }
            }
            tc::tc_fence_before();
            if (SHARED) units_barrier();                         // before the next item's rows take this one's places
            else unit_barrier(unit);
            if (lane == 0) tc::mbar_arrive(&q_free[q_buffer]);
            if (any_stray) {
                for (int n = thread; n < R * D; n += 128) strays[n] = 0.0f;
                stray_flag[unit] = 0;
                unit_barrier(unit);
            }
        }
    }
    tc::tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc::tc_fence_after();
        tc::tmem_dealloc(tmem, S::TMEM);
    }
}

}  // namespace tc_pages
