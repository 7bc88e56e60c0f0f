// Keys and values into a cache of eight bits, and back.
//
// The cache of G heads of D values: codes [pages, 2, G, page, D] (keys, then values) and exponent bytes [pages, 2, G, page]; what
// they stand for and how they are made is in e4m3.cuh.  A row's slot is page * page size + place.
#include "e4m3.cuh"
#include <cuda_fp16.h>

namespace {

constexpr int WARPS = 4;
constexpr int MAX_WIDTH = 256;      // values of a row: a lane holds an eighth of 64 of them at most

__device__ __forceinline__ float read1(const float* p) { return *p; }
__device__ __forceinline__ float read1(const __nv_bfloat16* p) { return __bfloat162float(*p); }

// One warp a (row, plane, head).  The row stays in registers between its maximum and its codes.
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
        x[i] = d < head_dim ? read1(src + d) : 0.0f;
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

// One warp a row of a page.
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
    for (int d = lane; d < head_dim; d += 32) {
        const unsigned h = live ? e4m3::halves(codes[at * head_dim + d]) : 0u;
        out[item * head_dim + d] = from_float<T>(__half2float(__ushort_as_half((unsigned short)(h & 0xffffu))) * f);
    }
}

constexpr int EXPANDED = 16;         // slots of an expanded page

// Requests' keys and values as bfloat16 pages of 16 slots, for a kernel that reads those: the requests of more than `rows_over` rows, one
// after another without gaps, a block a page.  `out_table` names a request's pages, `out_count` has its rows (none for the requests
// that are left out), `out_list` the requests.  Bound by the bytes: a byte read and two written for each value.
// A value row that is no numbers comes as zeros with its key as NaN: the attention's mask then keeps it from the rows that do
// not see it (a weight of zero would not), and makes NaN of those that do, as it has to.
__global__ void __launch_bounds__(256)
expand_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ exponents, const int* __restrict__ row_count,
              const int* __restrict__ history, const int* __restrict__ tables, int table_stride, int requests, int rows_over, int window, int pages,
              int kv_heads, int head_dim, int page_size, __nv_bfloat16* __restrict__ out, int* __restrict__ out_table, int out_stride,
              int* __restrict__ out_count, int* __restrict__ out_list) {
    pdl_trigger();
    pdl_wait();
    __shared__ int owner, page_of_owner;
    if (threadIdx.x == 0) owner = -1;
    __syncthreads();
    if (blockIdx.x == 0)
        for (int r = threadIdx.x; r < requests; r += blockDim.x) {
            out_list[r] = r;
            out_count[r] = row_count[r] > rows_over ? row_count[r] : 0;
        }
    if (threadIdx.x < 32) {
        const int f = blockIdx.x;
        int before = 0;
        for (int r0 = 0; r0 < requests && before <= f; r0 += 32) {
            const int r = r0 + threadIdx.x;
            int n = 0, first = 0;
            if (r < requests && row_count[r] > rows_over) {
                const int keys = history[r] + row_count[r];
                // The reader starts at a whole stage of 128 keys.
                first = window > 0 ? max(0, history[r] - window + 1) / 128 * (128 / EXPANDED) : 0;
                n = max(0, min((keys + EXPANDED - 1) / EXPANDED, out_stride) - first);
            }
            int upto = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int x = __shfl_up_sync(0xffffffffu, upto, o);
                if ((int)threadIdx.x >= o) upto += x;
            }
            if (f >= before + upto - n && f < before + upto) owner = r, page_of_owner = first + f - (before + upto - n);
            before += __shfl_sync(0xffffffffu, upto, 31);
        }
    }
    __syncthreads();
    const int r = owner, j = page_of_owner;
    if (r < 0) return;
    if (threadIdx.x == 0) out_table[(size_t)r * out_stride + j] = blockIdx.x;
    const int keys = min(history[r] + row_count[r], table_stride * page_size);
    const int pieces = head_dim / 16;
    const int* table = tables + (size_t)r * table_stride;
    const size_t plane = (size_t)kv_heads * page_size;
    for (int x = threadIdx.x; x < 2 * kv_heads * EXPANDED * pieces; x += blockDim.x) {
        const int piece = x % pieces, slot = x / pieces % EXPANDED, head = x / (pieces * EXPANDED);      // head: plane * kv_heads + g
        const int t = j * EXPANDED + slot;
        const int page = t < keys ? table[t / page_size] : -1;
        uint4 lo = make_uint4(0, 0, 0, 0), hi = lo;
        if (page >= 0 && page < pages) {
            const size_t at = ((size_t)page * 2 * kv_heads + head) * page_size + t % page_size;
            const unsigned byte = exponents[at];
            const bool key = head < kv_heads;
            const bool bad = byte == e4m3::NOT_NUMBERS || (key && exponents[at + plane] == e4m3::NOT_NUMBERS);
            if (bad) {
                if (key) lo = hi = make_uint4(0x7FC07FC0u, 0x7FC07FC0u, 0x7FC07FC0u, 0x7FC07FC0u);
            } else {
                const uint4 w = *reinterpret_cast<const uint4*>(codes + at * head_dim + piece * 16);
                const float f = e4m3::up(byte);
                auto four = [&](unsigned c, unsigned& a, unsigned& b) {
                    const unsigned h0 = e4m3::halves((unsigned short)(c & 0xffffu)), h1 = e4m3::halves((unsigned short)(c >> 16));
                    const float2 x0 = __half22float2(*reinterpret_cast<const __half2*>(&h0)), x1 = __half22float2(*reinterpret_cast<const __half2*>(&h1));
                    const __nv_bfloat162 y0 = __floats2bfloat162_rn(x0.x * f, x0.y * f), y1 = __floats2bfloat162_rn(x1.x * f, x1.y * f);
                    a = *reinterpret_cast<const unsigned*>(&y0);
                    b = *reinterpret_cast<const unsigned*>(&y1);
                };
                four(w.x, lo.x, lo.y);
                four(w.y, lo.z, lo.w);
                four(w.z, hi.x, hi.y);
                four(w.w, hi.z, hi.w);
            }
        }
        uint4* to = reinterpret_cast<uint4*>(out + (((size_t)blockIdx.x * 2 * kv_heads + head) * EXPANDED + slot) * head_dim + piece * 16);
        to[0] = lo;
        to[1] = hi;
    }
}

}  // namespace

// Row r's keys and values, [rows, kv_heads, head_dim] of `dtype` with rows `k_stride` and `v_stride` values apart, go to slots[r]
// (below 0 or beyond the cache: not kept).
LLMX_EXPORT int llmx_quantize_kv(const void* k, long long k_stride, const void* v, long long v_stride, int dtype, const int* slots, void* codes,
                                 void* exponents, int rows, int kv_heads, int head_dim, int page_size, int pages, cudaStream_t stream) {
    if (rows <= 0) return 0;
    if (kv_heads <= 0 || head_dim <= 0 || head_dim > MAX_WIDTH || page_size <= 0 || pages < 0) return LLMX_ERR_UNSUPPORTED;
    const long long items = (long long)rows * 2 * kv_heads, blocks = (items + WARPS - 1) / WARPS;
    if (blocks >= (1ll << 31)) return LLMX_ERR_UNSUPPORTED;
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
#define LLMX_DEQUANTIZE(T)                                                                                                            \
    launch_kernel(dequantize_kernel<T>, dim3((unsigned)blocks), dim3(WARPS * 32), 0, stream, (const uint8_t*)codes, (const uint8_t*)exponents, \
                  pages, used, (T*)out, rows, kv_heads, head_dim, page_size, total_pages)
    if (dtype == LLMX_BF16) LLMX_DEQUANTIZE(__nv_bfloat16);
    else if (dtype == LLMX_F32) LLMX_DEQUANTIZE(float);
    else return LLMX_ERR_BAD_ARGUMENT;
#undef LLMX_DEQUANTIZE
    return launch_status();
}

// Requests of more than `rows_over` rows, their keys and values as bfloat16 pages out[0 .. capacity) of [2, kv_heads, 16, head_dim]: all of
// them, or under a window those from the stage of 128 that the first row's window starts in.  `capacity` pages must hold them.
LLMX_EXPORT int llmx_expand_requests(const void* codes, const void* exponents, const int* row_count, const int* history, const int* tables,
                                     int table_stride, int requests, int rows_over, int window, int pages, int kv_heads, int head_dim, int page_size,
                                     void* out, int capacity, int* out_table, int out_stride, int* out_count, int* out_list, cudaStream_t stream) {
    if (requests <= 0 || capacity <= 0) return 0;
    if (kv_heads <= 0 || head_dim <= 0 || head_dim % 16 || page_size <= 0 || (((uintptr_t)codes | (uintptr_t)out) & 15)) return LLMX_ERR_UNSUPPORTED;
    launch_kernel(expand_kernel, dim3((unsigned)capacity), dim3(256), 0, stream, (const uint8_t*)codes, (const uint8_t*)exponents, row_count, history,
                  tables, table_stride, requests, rows_over, window, pages, kv_heads, head_dim, page_size, (__nv_bfloat16*)out, out_table, out_stride,
                  out_count, out_list);
    return launch_status();
}
