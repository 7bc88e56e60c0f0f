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
