// Softmax attention of requests' new rows over pages: of eight bits, under a window or a tree's bits; of bfloat16 and float32 under a tree's.
//
// Request r brings row_count[r] rows, row_start[r] the first, after history[r] keys that the cache holds already; the rows' own keys
// and values follow them there.  Row i sees the keys t with
//     t <= history + i,  t > history + i - window (window > 0)         or, with a tree,
//     t < history  or  bit (t - history) of its words is set (t < history + row_count)
// and   o = sum_t e_t v_t / sum_t e_t,   e_t = exp(scale q . k_t - max),  zeros where a row sees no key (or only such with scores of -inf).
// Query head h reads key/value head h / (heads / kv_heads).  A page that is not in the cache reads as zeros.
//
// Three forms.  Heads of 64 or 128 in pages of 16 to 512 slots by 16 run on matrix instructions, the warps' (attention_pages_mma.cuh) or
// tcgen05's (attention_pages_tc.cuh): queries of either type over eight bits, bfloat16 over bfloat16.  The general form takes any
// width to 256, any page size and any types, one block a (row, head): each warp walks every fourth key in increasing order with a
// running maximum and sum; the four states are merged in warp order, so a row's sums depend on its own keys alone (3.5 ms where the
// warps' form takes 33 us: 8 rows after 8,192 keys, 32 heads of 128 over 8).
#include "attention_pages_mma.cuh"
#include "attention_pages_tc.cuh"

namespace {
constexpr int WARPS = 4;
constexpr int MAX_PER_LANE = 8;     // widths up to 256

using mma_pages::Rows;

struct E4m3 {};                     // the cache's type: codes, exponents beside them

__device__ __forceinline__ float read_value(const float* p) { return *p; }
__device__ __forceinline__ float read_value(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ float read_value(const uint8_t* p) { return __half2float(__ushort_as_half((unsigned short)(e4m3::halves(*p) & 0xffffu))); }

template <typename T> struct Stored { typedef T type; };
template <> struct Stored<E4m3> { typedef uint8_t type; };

template <typename QT, typename KVT>
__global__ void __launch_bounds__(WARPS * 32)
attention_pages_kernel(const QT* __restrict__ q, const void* __restrict__ cache, const uint8_t* __restrict__ exponents, QT* __restrict__ out, Rows a,
                       int heads, int kv_heads, int head_dim, float scale) {
    pdl_trigger();
    pdl_wait();
    typedef typename Stored<KVT>::type S;
    constexpr bool eight = sizeof(S) == 1;
    extern __shared__ float smem[];  // WARPS * (head_dim + 2)
    const int i = blockIdx.x, h = blockIdx.y, r = blockIdx.z;
    const int count = a.row_count[r], history = max(a.history[r], 0);
    const int row = a.row_start[r] + i;
    if (i >= count || count > a.max_rows || row < 0 || row >= a.total_rows) return;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = h / (heads / kv_heads);
    const long long pos = (long long)history + i;
    const long long reach = (long long)a.table_stride * a.page_size;
    const long long end = min(a.tree ? (long long)history + min(count, 32 * a.tree_words) : pos + 1, reach);
    const long long lo = a.window > 0 ? max(0ll, pos - a.window + 1) : 0;
    const int* table = a.tables + (size_t)r * a.table_stride;
    const unsigned* bits = a.tree ? a.tree + (size_t)row * a.tree_words : nullptr;

    float qv[MAX_PER_LANE], acc[MAX_PER_LANE];
    const QT* qrow = q + ((size_t)row * heads + h) * head_dim;
#pragma unroll
    for (int j = 0; j < MAX_PER_LANE; ++j) {
        const int d = lane + 32 * j;
        qv[j] = d < head_dim ? to_float(qrow[d]) : 0.0f;
        acc[j] = 0.0f;
    }
    float m = -INFINITY, l = 0.0f;
    for (long long t = lo + warp; t < end; t += WARPS) {
        if (bits && t >= history && !(bits[(t - history) >> 5] >> ((t - history) & 31) & 1u)) continue;
        const int page = table[t / a.page_size];
        const bool there = page >= 0 && page < a.pages;
        const size_t slot = (((size_t)max(page, 0) * 2) * kv_heads + g) * a.page_size + t % a.page_size;
        const size_t v_slot = slot + (size_t)kv_heads * a.page_size;
        const S* kp = (const S*)cache + slot * head_dim;
        const S* vp = (const S*)cache + v_slot * head_dim;
        float s = 0.0f;
#pragma unroll
        for (int j = 0; j < MAX_PER_LANE; ++j) {
            const int d = lane + 32 * j;
            if (there && d < head_dim) s = fmaf(qv[j], read_value(kp + d), s);
        }
        s = warp_sum(s);
        float vf = 1.0f;
        if (eight && there) {
            s *= e4m3::up(exponents[slot]);
            vf = e4m3::up(exponents[v_slot]);
        }
        s *= scale;
        const float m_new = fmaxf(m, s), base = m_new == -INFINITY ? 0.0f : m_new;      // (a score of -inf weighs nothing, before the first key too)
        const float corr = expf(m - base);   // exp(-inf) = 0 on the first key
        const float e = expf(s - base);
        l = l * corr + e;
#pragma unroll
        for (int j = 0; j < MAX_PER_LANE; ++j) {
            const int d = lane + 32 * j;
            acc[j] = fmaf(e, there && d < head_dim ? read_value(vp + d) * vf : 0.0f, acc[j] * corr);
        }
        m = m_new;
    }
    float* mine = smem + warp * (head_dim + 2);
#pragma unroll
    for (int j = 0; j < MAX_PER_LANE; ++j) {
        const int d = lane + 32 * j;
        if (d < head_dim) mine[d] = acc[j];
    }
    if (lane == 0) {
        mine[head_dim] = m;
        mine[head_dim + 1] = l;
    }
    __syncthreads();
    if (warp) return;
    float mm = -INFINITY, ll = 0.0f, f[WARPS];
    for (int w = 0; w < WARPS; ++w) mm = fmaxf(mm, smem[w * (head_dim + 2) + head_dim]);
    for (int w = 0; w < WARPS; ++w) {
        // A warp without keys has a sum of zero and says nothing; one whose scores are NaN has a NaN there.
        const float lw = smem[w * (head_dim + 2) + head_dim + 1], mw = smem[w * (head_dim + 2) + head_dim];
        f[w] = lw == 0.0f ? 0.0f : expf(mw - (mm == -INFINITY ? 0.0f : mm));
        ll = fmaf(lw, f[w], ll);
    }
    QT* orow = out + ((size_t)row * heads + h) * head_dim;
    for (int d = lane; d < head_dim; d += 32) {
        float o = 0.0f;
        for (int w = 0; w < WARPS; ++w) o = fmaf(smem[w * (head_dim + 2) + d], f[w], o);
        orow[d] = from_float<QT>(ll == 0.0f ? 0.0f : o / ll);
    }
}

int multiprocessors() {
    static const int n = [] {
        int dev = 0, v = 0;
        return cudaGetDevice(&dev) == cudaSuccess && cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess && v > 0 ? v : 148;
    }();
    return n;
}

// How a call is cut up; `rows` 0: only the general form takes these sizes.
struct FewPlan {
    bool tensor = false;                  // tcgen05, else the warps' instruction
    int rows = 0, blocks = 0, max_tiles = 0;      // (row, head) pairs of a tile; tiles of keys of a request at most
    long long bytes(int head_dim) const { return 2ll * blocks * rows * (head_dim + mma_pages::PART) * 4; }      // two states a block
};

FewPlan few_plan(int q_dtype, int cache_dtype, int requests, int max_rows, int max_context, int heads, int kv_heads, int head_dim, int page_size,
                 int window, int general) {
    FewPlan p;
    if (general) return p;
    const bool types = (cache_dtype == LLMX_E4M3 && (q_dtype == LLMX_BF16 || q_dtype == LLMX_F32)) || (cache_dtype == LLMX_BF16 && q_dtype == LLMX_BF16);
    if (!types || (head_dim != 64 && head_dim != 128) || page_size % 16 || page_size > 512) return p;
    const long long pairs = (long long)max_rows * (heads / kv_heads);
    // Over eight bits the warps' form is as fast up to 32 pairs and simpler to feed; from 33 on a tile's keys are turned into halves for too
    // many warps.  In us, warps against tcgen05, each with tiles as high as the pairs ask for (the slower side of each, tcgen05's tiles of 16
    // and 32 rows and the warps' of 64, is no longer built): 1 x 32,768 keys of 4 pairs 25.6 / 26.6, 8 x 8,192 32.6 / 34.3, 64 requests of 2
    // pairs 63 / 70, 8 x 4,096 of 32 pairs 33.2 / 34.4; 8 x 4,096 of 64 pairs 57.6 / 52.4, 1 x 8,191 of 252 54.3 / 43.6, 32 x 1,024 of 64 71 / 74.
    p.tensor = head_dim == 128 && q_dtype == LLMX_BF16 && (cache_dtype == LLMX_BF16 || pairs > 32);
    // As few rows a tile as hold a request's: bfloat16, 8 x 4,096 keys, tiles of 16 / 32 / 64 rows: of 16 pairs 39 / 45 / 49 us, of 32 60 /
    // 46 / 51, of 64 106 / 72 / 54.
    p.rows = pairs <= 16 ? 16 : pairs <= 32 ? 32 : 64;
    // As many blocks as find an SM at one time.  The kernel leaves some of them without work where there is too little.
    const long long items = (pairs + p.rows - 1) / p.rows * kv_heads * requests;
    const long long keys = window > 0 ? min((long long)max_context, (long long)window + max_rows) : max_context;
    p.max_tiles = max_context / (p.tensor ? tc_pages::KEYS : mma_pages::TILE) + 2;
    const long long tiles = items * (keys / (p.tensor ? tc_pages::KEYS : mma_pages::TILE) + 2);
    if (items * (p.max_tiles + mma_pages::OPEN) >= (1ll << 31)) p.rows = 0;      // (places are counted in 32 bits)
    p.blocks = (int)min((p.tensor ? 1ll : 2ll) * multiprocessors(), max(items, tiles / 2));
    return p;
}

template <typename QT, bool EIGHT, int D, int TILE_ROWS, int KEYS, int OPEN, int RUNS>
int merge(const FewPlan& p, void* out, const float* partial, const Rows& a, int requests, int max_rows, int heads, int kv_heads, cudaStream_t stream) {
    const long long rows = (long long)max_rows * heads, blocks = (rows * (D / 4) + 127) / 128;
    launch_kernel(mma_pages::merge_kernel<QT, EIGHT, D, TILE_ROWS, KEYS, OPEN, RUNS>, dim3((unsigned)blocks, (unsigned)requests), dim3(128), 0, stream, partial,
                  (QT*)out, a, requests, heads, kv_heads, p.blocks);
    return launch_status();
}

template <typename QT, bool EIGHT, int D, int RW>
int few_rows(const FewPlan& p, const void* q, const void* cache, const void* exponents, void* out, float* partial, const Rows& a, int requests,
             int max_rows, int heads, int kv_heads, float scale, cudaStream_t stream) {
    using namespace mma_pages;
    constexpr int ring = (WARPS / RW) * Shape<EIGHT, D>::STAGES * Shape<EIGHT, D>::STAGE, states = WARPS * 16 * (D + PART) * 4;
    LLMX_ALLOW_SMEM(few_rows_kernel<QT, EIGHT, D, RW>);
    launch_kernel(few_rows_kernel<QT, EIGHT, D, RW>, dim3((unsigned)p.blocks), dim3(WARPS * 32), (size_t)(ring > states ? ring : states), stream,
                  (const QT*)q, (const uint8_t*)cache, (const uint8_t*)exponents, (QT*)out, partial, a, requests, heads, kv_heads,
                  scale * 1.4426950408889634f);
    if (const int e = launch_status()) return e;
    return merge<QT, EIGHT, D, 16 * RW, TILE, OPEN, WARPS / RW>(p, out, partial, a, requests, max_rows, heads, kv_heads, stream);
}

// The pages as (128 bytes of a row) x (eight rows) x (keys, values) x (eights of a plane) x (page): a copy is 16 keys and their values, eight
// keys, their values, eight keys, ... (bfloat16: of the rows' first or second half).
int pages_map(CUtensorMap* map, const void* cache, bool eight, int pages, int kv_heads, int page_size) {
    llmx_encode_tiled_fn enc = llmx_encode_tiled();
    if (!enc) return 10003;
    const cuuint64_t row = eight ? 128 : 256, plane = row * kv_heads * page_size;
    const cuuint64_t dims[5] = {128, 8, 2, (cuuint64_t)kv_heads * page_size / 8, (cuuint64_t)pages}, strides[4] = {row, plane, 8 * row, 2 * plane};
    const cuuint32_t box[5] = {eight ? 128u : 64u, 8, 2, 2, 1}, elem[5] = {1, 1, 1, 1, 1};
    return enc(map, eight ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 5, const_cast<void*>(cache), dims, strides, box, elem,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
               ? 0
               : 10003;
}

template <bool EIGHT, bool SHARED, int R>
int tensor_rows(const FewPlan& p, const void* q, const void* cache, const void* exponents, void* out, float* partial, const Rows& a, int requests,
                int max_rows, int heads, int kv_heads, float scale, int* error_word, cudaStream_t stream) {
    using namespace tc_pages;
    CUtensorMap map;
    if (const int e = pages_map(&map, cache, EIGHT, a.pages, kv_heads, a.page_size)) return e;
    LLMX_ALLOW_SMEM(pages_kernel<EIGHT, SHARED, R>);
    launch_kernel(pages_kernel<EIGHT, SHARED, R>, dim3((unsigned)p.blocks), dim3(tc_pages::Shape<EIGHT, SHARED, R>::THREADS),
                  (size_t)tc_pages::Shape<EIGHT, SHARED, R>::BYTES, stream, map, (const __nv_bfloat16*)q, (const uint8_t*)exponents, (__nv_bfloat16*)out, partial, a,
                  requests, heads, kv_heads, scale * 1.4426950408889634f, error_word);
    if (const int e = launch_status()) return e;
    return merge<__nv_bfloat16, EIGHT, 128, SHARED ? R : 2 * R, KEYS, OPEN, 1>(p, out, partial, a, requests, max_rows, heads, kv_heads, stream);
}
}  // namespace

// The bytes that `workspace` needs.
LLMX_EXPORT int llmx_attention_pages_workspace(int q_dtype, int cache_dtype, int requests, int max_rows, int max_context, int heads, int kv_heads,
                                               int head_dim, int page_size, int window, int general, long long* bytes) {
    *bytes = 0;
    if (requests <= 0 || max_rows <= 0 || kv_heads <= 0 || page_size <= 0) return 0;
    const FewPlan p = few_plan(q_dtype, cache_dtype, requests, max_rows, max_context, heads, kv_heads, head_dim, page_size, window, general);
    if (p.rows) *bytes = p.bytes(head_dim);
    return 0;
}

// q/out [total_rows, heads, head_dim] of `q_dtype`; the cache [pages, 2, kv_heads, page_size, head_dim] of `cache_dtype`, with `exponents`
// [pages, 2, kv_heads, page_size] where that is LLMX_E4M3.  Requests of more than `max_rows` rows are left out; none has more than
// `max_context` keys.  `general`: the general form, whose sums do not depend on what a row is batched with.  Rows that no request names are left as they are.
LLMX_EXPORT int llmx_attention_pages(const void* q, int q_dtype, const void* cache, const void* exponents, int cache_dtype, void* out,
                                     const int* row_start, const int* row_count, const int* history, const int* tables, int table_stride,
                                     const void* tree, int tree_words, int requests, int total_rows, int max_rows, int max_context, int pages,
                                     int heads, int kv_heads, int head_dim, int page_size, int window, int general, float scale, void* workspace,
                                     long long workspace_bytes, int* error_word, cudaStream_t stream) {
    if (requests <= 0 || total_rows <= 0 || max_rows <= 0) return 0;
    if (head_dim <= 0 || head_dim > 32 * MAX_PER_LANE || kv_heads <= 0 || heads % kv_heads || heads > 65535 || requests > 65535 || page_size <= 0)
        return LLMX_ERR_UNSUPPORTED;
    Rows a = {row_start, row_count, history, tables, table_stride, total_rows, pages, page_size, window, (const unsigned*)tree, tree_words,
                    ((1u << 31) + (unsigned)max(page_size / 16, 1) - 1) / (unsigned)max(page_size / 16, 1), 0, max_rows};
    if (!(scale > 0.0f)) return LLMX_ERR_BAD_ARGUMENT;
    if (!tree && cache_dtype != LLMX_E4M3) return LLMX_ERR_UNSUPPORTED;      // (the forms over bfloat16 look among drafted tokens alone for infinities)
    const FewPlan p = few_plan(q_dtype, cache_dtype, requests, max_rows, max_context, heads, kv_heads, head_dim, page_size, window, general);
    a.max_tiles = p.max_tiles;
    if (p.rows && pages > 0 && (long long)total_rows * heads < (1ll << 31) && !(((uintptr_t)q | (uintptr_t)out | (uintptr_t)cache | (uintptr_t)exponents) & 15) &&
        (long long)pages * 2 * kv_heads * page_size < (1ll << 31)) {
        if (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < p.bytes(head_dim)) return LLMX_ERR_BAD_ARGUMENT;
#define LLMX_FEW_ARGS p, q, cache, exponents, out, (float*)workspace, a, requests, max_rows, heads, kv_heads, scale
        if (p.tensor) {
            if (cache_dtype == LLMX_E4M3) return tensor_rows<true, false, 32>(LLMX_FEW_ARGS, error_word, stream);
            if (p.rows == 16) return tensor_rows<false, true, 16>(LLMX_FEW_ARGS, error_word, stream);
            if (p.rows == 32) return tensor_rows<false, true, 32>(LLMX_FEW_ARGS, error_word, stream);
            return tensor_rows<false, false, 32>(LLMX_FEW_ARGS, error_word, stream);
        }
#define LLMX_FEW_ROWS(QT, EIGHT, D)                                                         \
    do {                                                                                    \
        if (p.rows == 16) return few_rows<QT, EIGHT, D, 1>(LLMX_FEW_ARGS, stream);          \
        if (p.rows == 32) return few_rows<QT, EIGHT, D, 2>(LLMX_FEW_ARGS, stream);          \
        return few_rows<QT, EIGHT, D, 4>(LLMX_FEW_ARGS, stream);                            \
    } while (0)
        if (cache_dtype == LLMX_BF16) LLMX_FEW_ROWS(__nv_bfloat16, false, 64);
        if (q_dtype == LLMX_BF16 && head_dim == 64) LLMX_FEW_ROWS(__nv_bfloat16, true, 64);
        if (q_dtype == LLMX_BF16 && p.rows == 16) return few_rows<__nv_bfloat16, true, 128, 1>(LLMX_FEW_ARGS, stream);
        if (q_dtype == LLMX_BF16) return few_rows<__nv_bfloat16, true, 128, 2>(LLMX_FEW_ARGS, stream);
        if (head_dim == 64) LLMX_FEW_ROWS(float, true, 64);
        LLMX_FEW_ROWS(float, true, 128);
#undef LLMX_FEW_ARGS
#undef LLMX_FEW_ROWS
    }
    const size_t shmem = (size_t)WARPS * (head_dim + 2) * sizeof(float);
    const dim3 grid((unsigned)max_rows, (unsigned)heads, (unsigned)requests);
#define LLMX_PAGES(QT, KVT)                                                                                                               \
    launch_kernel(attention_pages_kernel<QT, KVT>, grid, dim3(WARPS * 32), shmem, stream, (const QT*)q, cache, (const uint8_t*)exponents, (QT*)out, \
                  a, heads, kv_heads, head_dim, scale)
#define LLMX_PAGES_Q(KVT)                                    \
    do {                                                     \
        if (q_dtype == LLMX_BF16) LLMX_PAGES(__nv_bfloat16, KVT); \
        else if (q_dtype == LLMX_F32) LLMX_PAGES(float, KVT); \
        else return LLMX_ERR_BAD_ARGUMENT;                   \
    } while (0)
    if (cache_dtype == LLMX_E4M3) LLMX_PAGES_Q(E4m3);
    else if (cache_dtype == LLMX_BF16) LLMX_PAGES_Q(__nv_bfloat16);
    else if (cache_dtype == LLMX_F32) LLMX_PAGES_Q(float);
    else return LLMX_ERR_BAD_ARGUMENT;
#undef LLMX_PAGES_Q
#undef LLMX_PAGES
    return launch_status();
}
