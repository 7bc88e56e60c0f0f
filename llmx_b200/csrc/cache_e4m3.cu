// Keys and values into a cache of eight bits, and back.
//
// The cache of G heads of D values: codes [pages, 2, G, page, D] (keys, then values) and exponent bytes [pages, 2, G, page]; what
// they stand for and how they are made is in e4m3.cuh.  A row's slot is page * page size + place.
#include "e4m3.cuh"
#include <cuda_fp16.h>

namespace {

constexpr int WARPS = 4;
constexpr int MAX_WIDTH = 256;      // values of a row: eight a lane

// ---- writing: bound by the bytes of the rows (a code for two or four of them is little) ----
// 16 bytes of a row a lane: LANES of them are a row, and a warp has EACH * 32 / LANES rows, whose loads are all asked for before the
// first is used.  Items are (row, plane, head), heads of a row next to one another.
__device__ __forceinline__ void read16(const float* p, float (&x)[4]) {
    const float4 v = *reinterpret_cast<const float4*>(p);
    x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
}
__device__ __forceinline__ void read16(const __nv_bfloat16* p, float (&x)[8]) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    const unsigned w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) x[2 * i] = __uint_as_float(w[i] << 16), x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
}

template <typename T, int LANES, int EACH>
__global__ void __launch_bounds__(WARPS * 32)
quantize_wide_kernel(const T* __restrict__ k, long long k_stride, const T* __restrict__ v, long long v_stride, const int* __restrict__ slots,
                     uint8_t* __restrict__ codes, uint8_t* __restrict__ exponents, int items, int kv_heads, int page_size, long long total_slots) {
    pdl_trigger();
    pdl_wait();
    constexpr int VALUES = 16 / sizeof(T), D = LANES * VALUES, ROWS = 32 / LANES;
    const int lane = threadIdx.x & 31, part = lane % LANES;
    const int first = (blockIdx.x * WARPS + (threadIdx.x >> 5)) * (ROWS * EACH) + lane / LANES;
    float x[EACH][VALUES];
    int slot[EACH], head[EACH];
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
        const int item = first + e * ROWS, row = item / (2 * kv_heads), rest = item - row * 2 * kv_heads, plane = rest >= kv_heads, g = rest - plane * kv_heads;
        head[e] = rest;
        slot[e] = -1;
        if (item < items) {
            slot[e] = slots[row];
            read16((plane ? v + row * v_stride : k + row * k_stride) + g * D + part * VALUES, x[e]);
        } else {
#pragma unroll
            for (int i = 0; i < VALUES; ++i) x[e][i] = 0.0f;
        }
    }
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
        unsigned peak = 0;
#pragma unroll
        for (int i = 0; i < VALUES; ++i) peak = max(peak, __float_as_uint(x[e][i]) & 0x7FFFFFFFu);
        if constexpr (LANES == 32) peak = __reduce_max_sync(0xffffffffu, peak);
        else
#pragma unroll
            for (int o = 1; o < LANES; o <<= 1) peak = max(peak, __shfl_xor_sync(0xffffffffu, peak, o));
        const unsigned byte = e4m3::exponent_byte(peak);
        const float f = byte == e4m3::NOT_NUMBERS ? 0.0f : e4m3::down(byte);
        unsigned w[VALUES / 4];
#pragma unroll
        for (int i = 0; i < VALUES / 4; ++i)
            w[i] = byte == e4m3::NOT_NUMBERS ? 0u : e4m3::pack2(x[e][4 * i] * f, x[e][4 * i + 1] * f) | e4m3::pack2(x[e][4 * i + 2] * f, x[e][4 * i + 3] * f) << 16;
        if (slot[e] < 0 || slot[e] >= total_slots) continue;
        const int page = slot[e] / page_size;
        const size_t at = ((size_t)page * 2 * kv_heads + head[e]) * page_size + (slot[e] - page * page_size);
        if (part == 0) exponents[at] = (uint8_t)byte;
        if constexpr (VALUES == 4) *reinterpret_cast<unsigned*>(codes + at * D + 4 * part) = w[0];
        else *reinterpret_cast<uint2*>(codes + at * D + 8 * part) = make_uint2(w[0], w[1]);
    }
}

// Any width, rows that start anywhere: one warp an item, 32 values at a time.  The row stays in registers between its maximum and its
// codes.
template <typename T>
__global__ void __launch_bounds__(WARPS * 32)
quantize_kernel(const T* __restrict__ k, long long k_stride, const T* __restrict__ v, long long v_stride, const int* __restrict__ slots,
                uint8_t* __restrict__ codes, uint8_t* __restrict__ exponents, int rows, int kv_heads, int head_dim, int page_size,
                long long total_slots) {
    pdl_trigger();
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const long long item = (long long)blockIdx.x * WARPS + (threadIdx.x >> 5);
    if (item >= (long long)rows * 2 * kv_heads) return;
    const int row = (int)(item / (2 * kv_heads)), rest = (int)(item % (2 * kv_heads)), plane = rest / kv_heads, g = rest % kv_heads;
    const int slot = slots[row];
    if (slot < 0 || slot >= total_slots) return;
    const T* src = (plane ? v + row * v_stride : k + row * k_stride) + g * head_dim;
    float x[MAX_WIDTH / 32];
    unsigned peak = 0;
#pragma unroll
    for (int i = 0; i < MAX_WIDTH / 32; ++i) {
        const int d = lane + 32 * i;
        x[i] = d < head_dim ? to_float(src[d]) : 0.0f;
        peak = max(peak, __float_as_uint(x[i]) & 0x7FFFFFFFu);
    }
    const unsigned byte = e4m3::exponent_byte(__reduce_max_sync(0xffffffffu, peak));
    const size_t at = (((size_t)(slot / page_size) * 2 + plane) * kv_heads + g) * page_size + slot % page_size;
    if (lane == 0) exponents[at] = (uint8_t)byte;
    const float f = e4m3::down(byte);
#pragma unroll
    for (int i = 0; i < MAX_WIDTH / 32; ++i) {
        const int d = lane + 32 * i;
        if (d < head_dim) codes[at * head_dim + d] = byte == e4m3::NOT_NUMBERS ? 0 : (uint8_t)e4m3::pack2(x[i] * f, 0.0f);
    }
}

// ---- writing a step's rows as the q/k/v product leaves them: per-head norm, rotation, queries out, keys and values into their slots ----
// The arithmetic of head_norm_rope_kernel (rowwise.cu), operation for operation, with a head's row in registers at its end, where it is
// given its exponent.  One warp a (row, head): a query head, or a key head with its value.  Bound by latency and, of many rows, by loads in
// flight, a row a warp at a time (32 heads of 128 over 8, beside the same into bfloat16 pages: 8 rows 2.2 / 1.8 us, 2,048 25.5 / 22.1, whose
// bytes take 10.9).
struct HeadsIn {
    const float* qkv;                 // [rows, stride]: q heads, then k heads at k_offset, v heads at v_offset
    int stride, k_offset, v_offset;
    const float* q_weight;            // [head_dim] or null
    const float* k_weight;
    float eps;
    const float* cos_table;           // [positions, rot_half] or null
    const float* sin_table;
    int rot_half;
    const int* positions;
    const int* slots;
    int rows, heads, kv_heads, head_dim, page_size;
    long long total_slots;
};
__device__ __forceinline__ void write4(float* p, float4 v) { *reinterpret_cast<float4*>(p) = v; }
__device__ __forceinline__ void write4(__nv_bfloat16* p, float4 v) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
    *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const unsigned*>(&a), *reinterpret_cast<const unsigned*>(&b));
}

template <typename QT>
__global__ void __launch_bounds__(WARPS * 32)
head_norm_rope_kernel(HeadsIn a, QT* __restrict__ q_out, uint8_t* __restrict__ codes, uint8_t* __restrict__ exponents) {
    pdl_trigger();
    pdl_wait();
    __shared__ float smem[WARPS][MAX_WIDTH];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, per_row = a.heads + a.kv_heads, D = a.head_dim;
    const long long item = (long long)blockIdx.x * WARPS + warp;
    if (item >= (long long)a.rows * per_row) return;
    const int row = (int)(item / per_row), j = (int)(item % per_row);
    const bool is_q = j < a.heads;
    const int g = is_q ? 0 : j - a.heads;
    const int slot = is_q ? 0 : a.slots[row];
    if (slot < 0 || (!is_q && slot >= a.total_slots)) return;
    float* buf = smem[warp];
    const float* src = a.qkv + (size_t)row * a.stride + (is_q ? j * D : a.k_offset + g * D);
    const float* weight = is_q ? a.q_weight : a.k_weight;
    float s = 0.0f;
    for (int d = lane; d < D; d += 32) {
        const float v = src[d];
        buf[d] = v;
        s = fmaf(v, v, s);
    }
    if (weight) {
        s = warp_sum(s);
        const float rr = 1.0f / sqrtf(s / (float)D + a.eps);
        __syncwarp();
        for (int d = lane; d < D; d += 32) buf[d] = buf[d] * (rr * weight[d]);
    }
    __syncwarp();
    const float* cs = a.cos_table ? a.cos_table + (size_t)a.positions[row] * a.rot_half : nullptr;
    const float* sn = a.cos_table ? a.sin_table + (size_t)a.positions[row] * a.rot_half : nullptr;
    float x[MAX_WIDTH / 32];
#pragma unroll
    for (int i = 0; i < MAX_WIDTH / 32; ++i) {
        const int d = lane + 32 * i;
        x[i] = 0.0f;
        if (d >= D) continue;
        if (cs && d < 2 * a.rot_half) {
            const int p = d < a.rot_half ? d : d - a.rot_half;
            const float u = buf[p], v = buf[p + a.rot_half];
            x[i] = d < a.rot_half ? fmaf(-v, sn[p], u * cs[p]) : fmaf(u, sn[p], v * cs[p]);
        } else {
            x[i] = buf[d];
        }
        if (is_q) q_out[(size_t)row * a.heads * D + j * D + d] = from_float<QT>(x[i]);
    }
    if (is_q) return;
    const float* value = a.qkv + (size_t)row * a.stride + a.v_offset + g * D;
#pragma unroll
    for (int plane = 0; plane < 2; ++plane) {
        unsigned peak = 0;
#pragma unroll
        for (int i = 0; i < MAX_WIDTH / 32; ++i) {
            if (plane) x[i] = lane + 32 * i < D ? value[lane + 32 * i] : 0.0f;
            peak = max(peak, __float_as_uint(x[i]) & 0x7FFFFFFFu);
        }
        const unsigned byte = e4m3::exponent_byte(__reduce_max_sync(0xffffffffu, peak));
        const size_t at = (((size_t)(slot / a.page_size) * 2 + plane) * a.kv_heads + g) * a.page_size + slot % a.page_size;
        if (lane == 0) exponents[at] = (uint8_t)byte;
        const float f = e4m3::down(byte);
#pragma unroll
        for (int i = 0; i < MAX_WIDTH / 32; ++i)
            if (lane + 32 * i < D) codes[at * D + lane + 32 * i] = byte == e4m3::NOT_NUMBERS ? 0 : (uint8_t)e4m3::pack2(x[i] * f, 0.0f);
    }
}

// Heads of 128 rotated whole or not at all: four values a lane, a pair's partner 16 lanes away (head_norm_rope_128_kernel's arithmetic).
template <typename QT>
__global__ void __launch_bounds__(WARPS * 32)
head_norm_rope_128_kernel(HeadsIn a, QT* __restrict__ q_out, uint8_t* __restrict__ codes, uint8_t* __restrict__ exponents) {
    pdl_trigger();
    pdl_wait();
    constexpr int D = 128;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, per_row = a.heads + a.kv_heads;
    const unsigned item = blockIdx.x * WARPS + warp;
    if (item >= (unsigned)a.rows * (unsigned)per_row) return;
    const int row = (int)(item / (unsigned)per_row), j = (int)(item - (unsigned)row * (unsigned)per_row);
    const bool is_q = j < a.heads;
    const int g = is_q ? 0 : j - a.heads;
    const int slot = is_q ? 0 : a.slots[row];
    if (slot < 0 || (!is_q && slot >= a.total_slots)) return;
    const float* row_src = a.qkv + (size_t)row * a.stride;
    float4 x = reinterpret_cast<const float4*>(row_src + (is_q ? j * D : a.k_offset + g * D))[lane], value = make_float4(0.f, 0.f, 0.f, 0.f);
    if (!is_q) value = reinterpret_cast<const float4*>(row_src + a.v_offset + g * D)[lane];
    float4 c, sn;
    if (a.cos_table) {
        const size_t base = (size_t)a.positions[row] * 64 + 4 * (lane & 15);
        c = *reinterpret_cast<const float4*>(a.cos_table + base);
        sn = *reinterpret_cast<const float4*>(a.sin_table + base);
    }
    const float* weight = is_q ? a.q_weight : a.k_weight;
    if (weight) {
        float s = fmaf(x.x, x.x, fmaf(x.y, x.y, fmaf(x.z, x.z, x.w * x.w)));
        s = warp_sum(s);
        const float rr = 1.0f / sqrtf(s / (float)D + a.eps);
        const float4 w4 = reinterpret_cast<const float4*>(weight)[lane];
        x.x *= rr * w4.x; x.y *= rr * w4.y; x.z *= rr * w4.z; x.w *= rr * w4.w;
    }
    if (a.cos_table) {
        float4 o;
        o.x = __shfl_xor_sync(0xffffffffu, x.x, 16); o.y = __shfl_xor_sync(0xffffffffu, x.y, 16);
        o.z = __shfl_xor_sync(0xffffffffu, x.z, 16); o.w = __shfl_xor_sync(0xffffffffu, x.w, 16);
        if (lane < 16) {
            x.x = fmaf(-o.x, sn.x, x.x * c.x); x.y = fmaf(-o.y, sn.y, x.y * c.y);
            x.z = fmaf(-o.z, sn.z, x.z * c.z); x.w = fmaf(-o.w, sn.w, x.w * c.w);
        } else {
            x.x = fmaf(o.x, sn.x, x.x * c.x); x.y = fmaf(o.y, sn.y, x.y * c.y);
            x.z = fmaf(o.z, sn.z, x.z * c.z); x.w = fmaf(o.w, sn.w, x.w * c.w);
        }
    }
    if (is_q) {
        write4(q_out + ((size_t)row * a.heads + j) * D + 4 * lane, x);
        return;
    }
    const int page = slot / a.page_size;
#pragma unroll
    for (int plane = 0; plane < 2; ++plane) {
        const float4 y = plane ? value : x;
        const unsigned peak = max(max(__float_as_uint(y.x) & 0x7FFFFFFFu, __float_as_uint(y.y) & 0x7FFFFFFFu),
                                  max(__float_as_uint(y.z) & 0x7FFFFFFFu, __float_as_uint(y.w) & 0x7FFFFFFFu));
        const unsigned byte = e4m3::exponent_byte(__reduce_max_sync(0xffffffffu, peak));
        const float f = e4m3::down(byte);
        const size_t at = (((size_t)page * 2 + plane) * a.kv_heads + g) * a.page_size + (slot - page * a.page_size);
        if (lane == 0) exponents[at] = (uint8_t)byte;
        reinterpret_cast<unsigned*>(codes + at * D)[lane] =
            byte == e4m3::NOT_NUMBERS ? 0u : e4m3::pack2(y.x * f, y.y * f) | e4m3::pack2(y.z * f, y.w * f) << 16;
    }
}

// ---- reading back: bound by the bytes written ----
// 16 bytes of the output a thread (8 codes, or 4), four of them 256 pieces apart, whose loads are all asked for before the first is used; a
// block has up to 1024 pieces of a page.  Pages of 8 heads of 128 and 16 slots as bfloat16: 512 in 11.7 us, 4,096 in 75 (5.4 TB/s; a copy of what
// is written takes 82); 512 as float32 in 19.
__device__ __forceinline__ float code_value(unsigned halves, bool upper) {
    return __half2float(__ushort_as_half((unsigned short)(upper ? halves >> 16 : halves & 0xffffu)));
}
__device__ __forceinline__ uint4 values16(uint2 w, float f, __nv_bfloat16) {
    unsigned r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const unsigned h = e4m3::halves((unsigned short)((i < 2 ? w.x : w.y) >> (16 * (i & 1))));
        const __nv_bfloat162 b = __floats2bfloat162_rn(code_value(h, false) * f, code_value(h, true) * f);
        r[i] = *reinterpret_cast<const unsigned*>(&b);
    }
    return make_uint4(r[0], r[1], r[2], r[3]);
}
__device__ __forceinline__ uint4 values16(uint2 w, float f, float) {
    const unsigned a = e4m3::halves((unsigned short)w.x), b = e4m3::halves((unsigned short)(w.x >> 16));
    return make_uint4(__float_as_uint(code_value(a, false) * f), __float_as_uint(code_value(a, true) * f), __float_as_uint(code_value(b, false) * f),
                      __float_as_uint(code_value(b, true) * f));
}

constexpr int READERS = 256, PIECES = 4;

template <typename T>
__global__ void __launch_bounds__(READERS)
dequantize_wide_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ exponents, const int* __restrict__ pages,
                       const int* __restrict__ used, T* __restrict__ out, int blocks_a_page, int pieces_a_page, int pieces_a_row, int page_size,
                       int total_pages) {
    pdl_trigger();
    pdl_wait();
    constexpr int CODES = 16 / sizeof(T);
    const int i = blockIdx.x / blocks_a_page, first = (blockIdx.x % blocks_a_page) * (READERS * PIECES) + threadIdx.x;
    const int page = pages[i], live = page < 0 || page >= total_pages ? 0 : used ? used[i] : page_size;
    const size_t rows_a_page = pieces_a_page / pieces_a_row;
    uint2 w[PIECES];
    float f[PIECES];
#pragma unroll
    for (int n = 0; n < PIECES; ++n) {
        const int piece = first + n * READERS, row = piece / pieces_a_row;
        w[n] = make_uint2(0, 0);
        f[n] = 0.0f;
        if (piece < pieces_a_page && row % page_size < live) {
            const uint8_t* src = codes + ((size_t)page * pieces_a_page + piece) * CODES;
            if constexpr (CODES == 8) w[n] = *reinterpret_cast<const uint2*>(src);
            else w[n].x = *reinterpret_cast<const unsigned*>(src);
            f[n] = e4m3::up(exponents[page * rows_a_page + row]);
        }
    }
#pragma unroll
    for (int n = 0; n < PIECES; ++n) {
        const int piece = first + n * READERS;
        if (piece < pieces_a_page) reinterpret_cast<uint4*>(out)[(size_t)i * pieces_a_page + piece] = values16(w[n], f[n], T());
    }
}

// Any width: one warp a row of a page.
template <typename T>
__global__ void __launch_bounds__(WARPS * 32)
dequantize_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ exponents, const int* __restrict__ pages,
                  const int* __restrict__ used, T* __restrict__ out, long long rows, int kv_heads, int head_dim, int page_size, int total_pages) {
    pdl_trigger();
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const long long item = (long long)blockIdx.x * WARPS + (threadIdx.x >> 5);
    if (item >= rows) return;
    const int place = (int)(item % page_size);
    const long long head = item / page_size, i = head / (2 * kv_heads);
    const int page = pages[i];
    const bool live = page >= 0 && page < total_pages && (!used || place < used[i]);
    const size_t at = ((size_t)max(page, 0) * 2 * kv_heads + head % (2 * kv_heads)) * page_size + place;
    const float f = live ? e4m3::up(exponents[at]) : 0.0f;
    for (int d = lane; d < head_dim; d += 32)
        out[item * head_dim + d] = from_float<T>(live ? code_value(e4m3::halves(codes[at * head_dim + d]), false) * f : 0.0f);
}

constexpr int EXPANDED = 16, ROW_PIECES = 16;         // slots of an expanded page; pieces of eight of a head's 128 values
constexpr int MOST_PAGES = (1 << 25) - 1;             // of a request (256 GB of one head's)

// Requests' keys and values as bfloat16 pages of 16 slots, for a kernel that reads those: the requests of more than `rows_over` rows, one
// after another without gaps, a block a page, as far as the pages reach (a request whose keys no longer fit is left out).  `out_table` names
// a request's pages, `out_count` has its rows (none for the requests that are left out), `out_list` the requests.  Bound by the bytes: a byte read and two written for each value (8,192 keys of 8 heads: 12 us).
// A value row that is no numbers comes as zeros with its key as NaN: the attention's mask then keeps it from the rows that do
// not see it (a weight of zero would not), and makes NaN of those that do, as it has to.
__global__ void __launch_bounds__(READERS)
expand_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ exponents, const int* __restrict__ row_start,
              const int* __restrict__ row_count, const int* __restrict__ history, const int* __restrict__ tables, int table_stride, int requests,
              int total_rows, int rows_over, int max_rows, int window, int pages,
              int kv_heads, int page_size, __nv_bfloat16* __restrict__ out, int* __restrict__ out_table, int out_stride,
              int* __restrict__ out_count, int* __restrict__ out_list) {
    pdl_trigger();
    pdl_wait();
    // A request's rows, none where it is left out: its reader trusts what it gets, so rows must lie in the output, and keys (up to the
    // end of the last stage of 128) in the request's part of the table.
    auto rows_of = [&](int r) {
        const int n = row_count[r], h = history[r], start = row_start[r];
        return n > rows_over && n <= max_rows && h >= 0 && start >= 0 && (long long)h + n <= (long long)(out_stride - 8) * EXPANDED
                   ? max(min(n, total_rows - start), 0) : 0;
    };
    __shared__ int owner, page_of_owner;
    if (threadIdx.x == 0) owner = -1;
    __syncthreads();
    if (threadIdx.x < 32) {
        // (Counts that overlap may claim more pages than there are: sums stay below 2^31.  The first block walks all requests, for their counts.)
        const int f = blockIdx.x, capacity = gridDim.x;
        int before = 0;
        for (int r0 = 0; r0 < requests && (before <= f || f == 0); r0 += 32) {
            const int r = r0 + threadIdx.x;
            const int rows = r < requests ? rows_of(r) : 0;
            int n = 0, first = 0;
            if (rows > 0) {
                const int keys = history[r] + rows;
                // The reader starts at a whole stage of 128 keys.
                first = window > 0 ? max(0, history[r] - window + 1) / 128 * (128 / EXPANDED) : 0;
                n = min(max(0, min((keys + EXPANDED - 1) / EXPANDED, out_stride) - first), MOST_PAGES);
            }
            int upto = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int x = __shfl_up_sync(0xffffffffu, upto, o);
                if ((int)threadIdx.x >= o) upto += x;
            }
            const int end = before + upto, begin = end - n;
            const bool fits = end <= capacity;
            if (fits && f >= begin && f < end) owner = r, page_of_owner = first + f - begin;
            if (f == 0 && r < requests) out_list[r] = r, out_count[r] = fits ? rows : 0;
            before = min(before + __shfl_sync(0xffffffffu, upto, 31), 32 * MOST_PAGES);
        }
    }
    __syncthreads();
    const int r = owner, j = page_of_owner;
    if (r < 0) return;
    if (threadIdx.x == 0) out_table[(size_t)r * out_stride + j] = blockIdx.x;
    const int keys = (int)min((long long)history[r] + rows_of(r), (long long)table_stride * page_size);
    const int total = 2 * kv_heads * EXPANDED * ROW_PIECES, low = window > 0 ? max(0, history[r] - window + 1) : 0;
    const int* table = tables + (size_t)r * table_stride;
    const size_t plane = (size_t)kv_heads * page_size;
    uint4* to = reinterpret_cast<uint4*>(out) + (size_t)blockIdx.x * total;
    // The run's 16 slots lie in one page where pages are whole 16s.
    const bool together = page_size % EXPANDED == 0;
    const int t0 = j * EXPANDED, run_page = together && t0 < keys ? table[t0 / page_size] : -1, run_off = t0 % page_size;
    // Eight codes a piece; four pieces' loads are asked for before the first is used.
    for (int x0 = threadIdx.x; x0 < total; x0 += PIECES * READERS) {
        uint2 w[PIECES];
        unsigned byte[PIECES], other[PIECES];
#pragma unroll
        for (int n = 0; n < PIECES; ++n) {
            const int x = x0 + n * READERS, piece = x % ROW_PIECES, slot = x / ROW_PIECES % EXPANDED, head = x / (ROW_PIECES * EXPANDED);   // plane * kv_heads + g
            const int t = t0 + slot;
            const bool wanted = x < total && t >= low && t < keys;
            const int page = together ? run_page : wanted ? table[t / page_size] : -1, off = together ? run_off + slot : t % page_size;
            w[n] = make_uint2(0, 0);
            byte[n] = other[n] = 0;
            if (wanted && page >= 0 && page < pages) {
                const size_t at = ((size_t)page * 2 * kv_heads + head) * page_size + off;
                w[n] = *reinterpret_cast<const uint2*>(codes + at * (8 * ROW_PIECES) + piece * 8);
                byte[n] = exponents[at];
                if (head < kv_heads) other[n] = exponents[at + plane];
            }
        }
#pragma unroll
        for (int n = 0; n < PIECES; ++n) {
            const int x = x0 + n * READERS;
            if (x >= total) continue;
            uint4 v = values16(w[n], e4m3::up(byte[n]), __nv_bfloat16());
            if (byte[n] == e4m3::NOT_NUMBERS || other[n] == e4m3::NOT_NUMBERS) {
                const unsigned nan = x < total / 2 ? 0x7FC07FC0u : 0u;
                v = make_uint4(nan, nan, nan, nan);
            }
            to[x] = v;
        }
    }
}

}  // namespace

// Row r's keys and values, [rows, kv_heads, head_dim] of `dtype` with rows `k_stride` and `v_stride` values apart, go to slots[r]
// (below 0 or beyond the cache: not kept).
LLMX_EXPORT int llmx_quantize_kv(const void* k, long long k_stride, const void* v, long long v_stride, int dtype, const int* slots, void* codes,
                                 void* exponents, int rows, int kv_heads, int head_dim, int page_size, int pages, cudaStream_t stream) {
    if (rows <= 0) return 0;
    if (dtype != LLMX_F32 && dtype != LLMX_BF16) return LLMX_ERR_BAD_ARGUMENT;
    if (kv_heads <= 0 || head_dim <= 0 || head_dim > MAX_WIDTH || page_size <= 0 || pages < 0) return LLMX_ERR_UNSUPPORTED;
    const long long items = (long long)rows * 2 * kv_heads, blocks = (items + WARPS - 1) / WARPS;
    if (blocks >= (1ll << 31)) return LLMX_ERR_UNSUPPORTED;
    // Rows in 16-byte pieces where they lie so and a warp's lanes are whole rows.  Few items: one at a time a warp, so that they find more
    // of the device's warps; many: two, for their loads' latency.  In us with one / two / four, rows of 8 heads of 128: 8 of float32 1.3 /
    // 1.5 / 2.0, 256 2.3 / 2.9 / 3.0, 1,024 4.9 / 4.5 / 5.1, 8,192 34 / 23 / 22, 40,000 of bfloat16 84 / 68 / 80.  Warps that stay and ask for
    // the next rows before these are written are no faster (26 and 76).
    const int size = dtype == LLMX_F32 ? 4 : 2, lanes = head_dim * size / 16;
    const bool wide = head_dim * size % 16 == 0 && (lanes == 8 || lanes == 16 || lanes == 32) && !((k_stride | v_stride) * size % 16) &&
                      !(((uintptr_t)k | (uintptr_t)v | (uintptr_t)codes) & 15) && items < (1ll << 30);
    if (wide) {
        const int each = items * lanes >= 148ll * 32 * 64 ? 2 : 1;
        const long long per = (long long)WARPS * (32 / lanes) * each;
#define LLMX_QUANTIZE(T, LANES, EACH)                                                                                                  \
    launch_kernel(quantize_wide_kernel<T, LANES, EACH>, dim3((unsigned)((items + per - 1) / per)), dim3(WARPS * 32), 0, stream, (const T*)k,  \
                  k_stride, (const T*)v, v_stride, slots, (uint8_t*)codes, (uint8_t*)exponents, (int)items, kv_heads, page_size,              \
                  (long long)pages * page_size)
#define LLMX_QUANTIZE_EACH(T, LANES)                   \
    do {                                               \
        if (each == 2) LLMX_QUANTIZE(T, LANES, 2);     \
        else LLMX_QUANTIZE(T, LANES, 1);               \
    } while (0)
        if (dtype == LLMX_F32) {
            if (lanes == 32) LLMX_QUANTIZE_EACH(float, 32);
            else if (lanes == 16) LLMX_QUANTIZE_EACH(float, 16);
            else LLMX_QUANTIZE_EACH(float, 8);
        } else {
            if (lanes == 32) LLMX_QUANTIZE_EACH(__nv_bfloat16, 32);
            else if (lanes == 16) LLMX_QUANTIZE_EACH(__nv_bfloat16, 16);
            else LLMX_QUANTIZE_EACH(__nv_bfloat16, 8);
        }
#undef LLMX_QUANTIZE_EACH
#undef LLMX_QUANTIZE
        return launch_status();
    }
#define LLMX_QUANTIZE(T)                                                                                                            \
    launch_kernel(quantize_kernel<T>, dim3((unsigned)blocks), dim3(WARPS * 32), 0, stream, (const T*)k, k_stride, (const T*)v, v_stride, slots, \
                  (uint8_t*)codes, (uint8_t*)exponents, rows, kv_heads, head_dim, page_size, (long long)pages * page_size)
    if (dtype == LLMX_BF16) LLMX_QUANTIZE(__nv_bfloat16);
    else if (dtype == LLMX_F32) LLMX_QUANTIZE(float);
    else return LLMX_ERR_BAD_ARGUMENT;
#undef LLMX_QUANTIZE
    return launch_status();
}

// out[i] = page pages[i], [2, kv_heads, page_size, head_dim] of `dtype`; places from used[i] on (null: none) and pages outside of the
// cache are zeros.
LLMX_EXPORT int llmx_dequantize_pages(const void* codes, const void* exponents, const int* pages, const int* used, void* out, int dtype, int n,
                                      int kv_heads, int head_dim, int page_size, int total_pages, cudaStream_t stream) {
    if (n <= 0) return 0;
    if (kv_heads <= 0 || head_dim <= 0 || page_size <= 0) return LLMX_ERR_UNSUPPORTED;
    const long long rows = (long long)n * 2 * kv_heads * page_size, blocks = (rows + WARPS - 1) / WARPS;
    if (blocks >= (1ll << 31)) return LLMX_ERR_UNSUPPORTED;
    if (dtype != LLMX_F32 && dtype != LLMX_BF16) return LLMX_ERR_BAD_ARGUMENT;
    const int per = dtype == LLMX_F32 ? 4 : 8;          // codes for 16 bytes
    const long long pieces = (long long)2 * kv_heads * page_size * (head_dim / per), blocks_a_page = (pieces + READERS * PIECES - 1) / (READERS * PIECES);
    if (head_dim % per == 0 && !(((uintptr_t)codes | (uintptr_t)out) & 15) && pieces < (1ll << 30) && n * blocks_a_page < (1ll << 31)) {
#define LLMX_DEQUANTIZE(T)                                                                                                            \
    launch_kernel(dequantize_wide_kernel<T>, dim3((unsigned)(n * blocks_a_page)), dim3(READERS), 0, stream, (const uint8_t*)codes,            \
                  (const uint8_t*)exponents, pages, used, (T*)out, (int)blocks_a_page, (int)pieces, head_dim / per, page_size, total_pages)
        if (dtype == LLMX_BF16) LLMX_DEQUANTIZE(__nv_bfloat16);
        else LLMX_DEQUANTIZE(float);
#undef LLMX_DEQUANTIZE
        return launch_status();
    }
#define LLMX_DEQUANTIZE(T)                                                                                                            \
    launch_kernel(dequantize_kernel<T>, dim3((unsigned)blocks), dim3(WARPS * 32), 0, stream, (const uint8_t*)codes, (const uint8_t*)exponents, \
                  pages, used, (T*)out, rows, kv_heads, head_dim, page_size, total_pages)
    if (dtype == LLMX_BF16) LLMX_DEQUANTIZE(__nv_bfloat16);
    else if (dtype == LLMX_F32) LLMX_DEQUANTIZE(float);
    else return LLMX_ERR_BAD_ARGUMENT;
#undef LLMX_DEQUANTIZE
    return launch_status();
}

// Requests of more than `rows_over` rows (and at most `max_rows`), their keys and values as bfloat16 pages out[0 .. capacity) of [2, kv_heads, 16, 128]: all of
// them, or under a window those from the stage of 128 that the first row's window starts in.  `capacity` pages must hold them.
LLMX_EXPORT int llmx_expand_requests(const void* codes, const void* exponents, const int* row_start, const int* row_count, const int* history,
                                     const int* tables, int table_stride, int requests, int total_rows, int rows_over, int max_rows, int window, int pages,
                                     int kv_heads, int head_dim, int page_size,
                                     void* out, int capacity, int* out_table, int out_stride, int* out_count, int* out_list, cudaStream_t stream) {
    if (requests <= 0 || capacity <= 0) return 0;
    if (kv_heads <= 0 || head_dim != 8 * ROW_PIECES || page_size <= 0 || (((uintptr_t)codes | (uintptr_t)out) & 15)) return LLMX_ERR_UNSUPPORTED;
    launch_kernel(expand_kernel, dim3((unsigned)capacity), dim3(READERS), 0, stream, (const uint8_t*)codes, (const uint8_t*)exponents, row_start,
                  row_count, history, tables, table_stride, requests, total_rows, rows_over, max_rows, window, pages, kv_heads, page_size, (__nv_bfloat16*)out, out_table, out_stride,
                  out_count, out_list);
    return launch_status();
}

// Per-head norm, rotation, queries out and keys and values into their slots, as llmx_head_norm_rope_kv (rowwise.cu) for a cache in eight bits.
LLMX_EXPORT int llmx_head_norm_rope_e4m3(const float* qkv, int qkv_stride, int k_offset, int v_offset, const float* q_weight, const float* k_weight,
                                         float eps, const float* cos_table, const float* sin_table, int rot_half, const int* positions,
                                         const int* slots, void* q_out, int q_dtype, void* codes, void* exponents, long long pages, int rows, int heads,
                                         int kv_heads, int head_dim, int page_size, cudaStream_t stream) {
    if (rows <= 0) return 0;
    if (head_dim <= 0 || rot_half < 0 || 2 * rot_half > head_dim || page_size <= 0 || (q_dtype != LLMX_F32 && q_dtype != LLMX_BF16)) return LLMX_ERR_BAD_ARGUMENT;
    const long long blocks = ((long long)rows * (heads + kv_heads) + WARPS - 1) / WARPS;
    if (head_dim > MAX_WIDTH || blocks >= (1ll << 29)) return LLMX_ERR_UNSUPPORTED;
    const HeadsIn a = {qkv, qkv_stride, k_offset, v_offset, q_weight, k_weight, eps, cos_table, sin_table, rot_half, positions, slots,
                       rows, heads, kv_heads, head_dim, page_size, pages * page_size};
    const bool fast = head_dim == 128 && (!cos_table || rot_half == 64) && !((qkv_stride | k_offset | v_offset) % 4) &&
                      !(((uintptr_t)qkv | (uintptr_t)q_out | (uintptr_t)codes | (uintptr_t)q_weight | (uintptr_t)k_weight | (uintptr_t)cos_table |
                         (uintptr_t)sin_table) & 15);
#define LLMX_HEADS(KERNEL, QT) \
    launch_kernel(KERNEL<QT>, dim3((unsigned)blocks), dim3(WARPS * 32), 0, stream, a, (QT*)q_out, (uint8_t*)codes, (uint8_t*)exponents)
    if (q_dtype == LLMX_BF16) {
        if (fast) LLMX_HEADS(head_norm_rope_128_kernel, __nv_bfloat16);
        else LLMX_HEADS(head_norm_rope_kernel, __nv_bfloat16);
    } else {
        if (fast) LLMX_HEADS(head_norm_rope_128_kernel, float);
        else LLMX_HEADS(head_norm_rope_kernel, float);
    }
#undef LLMX_HEADS
    return launch_status();
}
