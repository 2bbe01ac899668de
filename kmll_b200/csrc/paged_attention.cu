// Attention over the paged 8-bit cache: rows of requests of unequal length, each over its own pages.
#include <climits>

#include "internal.cuh"
#include "paged.cuh"

namespace kmll {
namespace {

__device__ inline int code_at(uint4 u, int i) {
    const uint32_t w = i < 4 ? u.x : i < 8 ? u.y : i < 12 ? u.z : u.w;
    return (int)(int8_t)(w >> (8 * (i & 3)));
}

// ---- any head size: a block of four warps per (row, kv head), a warp per query head ------------------------------------------
// A lane has one key of 32 (codes of a 16-byte group against q in shared memory), then one column of the values in turn.  f32 throughout.  For head
// sizes other than 64 and 128, and rows that are not aligned to 16 bytes.  Bound: the latency of its loads, one tile of 32 keys after the other (32
// query heads over 8 of size 80, 16 requests of 2048 tokens: 238 us for 42 MB; a prompt of 512: 195 us).
template <typename T>
__global__ void __launch_bounds__(128) paged_rows_kernel(const PagedArgs a) {
    __shared__ __align__(16) float s_q[4][256];
    __shared__ __align__(16) float s_p[4][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, t = blockIdx.x, h = blockIdx.y, hd = a.head_dim, group = a.heads / a.kv_heads;
    pdl_wait();
    int lo = 0, hi = a.requests;  // the last request that starts at or before t
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.query_start[mid] <= t) lo = mid;
        else hi = mid;
    }
    const PagedRequest rq = PagedRequest::of(a, lo);
    if (t < rq.first || t >= rq.first + rq.rows || (long long)rq.rows * group <= a.skip_rows) return;
    const int pos = min(rq.pos0 + (t - rq.first), rq.hi - 1), start = window_start(rq.pos0 + (t - rq.first), a.window);
    const int32_t* const table = a.table + (size_t)lo * a.width;
    for (int g = warp; g < group; g += 4) {
        const size_t row = ((size_t)t * a.heads + (size_t)h * group + g) * hd;
        __syncwarp();
        for (int d = lane; d < hd; d += 32) s_q[warp][d] = row_entry<T>(a.query, row + d) * a.scale2;
        __syncwarp();
        float m = -INFINITY, l = 0.0f, acc[8] = {};
        for (int j0 = start & ~31; j0 <= pos; j0 += 32) {
            const int j = j0 + lane, page = j <= pos ? table[j / a.block] : -1;
            const bool there = j >= start && j <= pos && page >= 0 && page < a.pages;
            float s = -INFINITY, vs = 0.0f;
            if (there) {
                const size_t ph = (size_t)page * a.kv_heads + h;
                const uint4* const k = reinterpret_cast<const uint4*>(a.k_codes + ph * a.block * hd) + j % a.block;
                float dot = 0.0f;
                for (int c = 0; c < hd / 16; ++c) {
                    const uint4 u = k[(size_t)c * a.block];
#pragma unroll
                    for (int i = 0; i < 16; ++i) dot = fmaf((float)code_at(u, i), s_q[warp][c * 16 + i], dot);
                }
                s = dot * a.k_scales[ph];
                vs = a.v_scales[ph];
            }
            const float top = fmaxf(m, warp_max(s)), base = top == -INFINITY ? 0.0f : top;
            const float p = there ? exp2f(s - base) : 0.0f, turn = exp2f(m - base);
            m = top;
            l = l * turn + warp_sum(p);
            __syncwarp();
            s_p[warp][lane] = p * vs;
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 8; ++i) acc[i] *= turn;
            for (int half = 0; half < 2; ++half) {
                const int jj = j0 + half * 16, pg = jj <= pos && jj + 15 >= start ? table[jj / a.block] : -1;
                if (pg < 0 || pg >= a.pages) continue;
                const uint4* const v = reinterpret_cast<const uint4*>(a.v_codes + ((size_t)pg * a.kv_heads + h) * a.block * hd) + (size_t)(jj % a.block / 16) * hd;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int d = lane + 32 * i;
                    if (d >= hd) break;
                    const uint4 u = v[d];
#pragma unroll
                    for (int e = 0; e < 16; ++e) acc[i] = fmaf((float)code_at(u, e), s_p[warp][half * 16 + e], acc[i]);
                }
            }
        }
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // (a row that attends nothing is zero)
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (lane + 32 * i < hd) store_row(static_cast<T*>(a.out) + row + lane + 32 * i, acc[i] * inv);
    }
}

}  // namespace
}  // namespace kmll

using namespace kmll;

// Rows up to which a request goes to the kernel for few rows.  Eight take half of the registers of sixteen (three blocks on a multiprocessor for two); sixteen are for
// calls that have no more, and for heads in groups of more than eight, whose single tokens need them.
static int few_rows(long long max_rows, int group) { return max_rows <= 8 || (max_rows > kPagedDecodeRows && group <= 8) ? 8 : kPagedDecodeRows; }

extern "C" size_t kmll_paged_attention_workspace_bytes(int heads, int kv_heads, int head_dim, int requests, int tokens, int max_query, int max_context) {
    if (heads <= 0 || kv_heads <= 0 || requests <= 0 || tokens <= 0 || max_query <= 0 || !paged_decode_serves(head_dim)) return 0;
    const long long max_rows = (long long)max_query * (heads / kv_heads);
    const size_t few = kPagedZeroBytes + paged_decode_scratch_bytes(head_dim, few_rows(max_rows, heads / kv_heads));
    return max_rows <= kPagedDecodeRows ? few : (few + 255) / 256 * 256 + paged_prompt_scratch_bytes(heads, kv_heads, head_dim, requests, tokens);
}

extern "C" int kmll_paged_attention(kmll_stream_t stream, const void* query, int is_f32, const int32_t* query_start, const int32_t* context, const int32_t* block_table,
                                    int table_width, int requests, int tokens, int max_query, int max_context, int heads, const int8_t* k_codes, const float* k_scales,
                                    const int8_t* v_codes, const float* v_scales, int pages, int block, int kv_heads, int head_dim, float scale, int window,
                                    void* workspace, void* out) {
    KMLL_TRY_RC(check_paged_cache("paged attention", k_codes, k_scales, v_codes, v_scales, pages, block, kv_heads, head_dim));
    KMLL_REQUIRE(requests >= 0 && tokens >= 0 && max_query >= 0 && max_context >= 0 && table_width >= 0, "paged attention: negative size");
    KMLL_REQUIRE(heads > 0 && heads <= 65535 && heads % kv_heads == 0, "paged attention: %d query heads over %d kv heads", heads, kv_heads);
    KMLL_REQUIRE((long long)table_width * block <= INT_MAX - 1024, "paged attention: a table of %d pages of %d tokens: positions are 32 bits", table_width, block);
    KMLL_REQUIRE(scale > 0.0f && scale < INFINITY, "paged attention: scale must be positive and finite");
    KMLL_REQUIRE(window >= 0, "paged attention: negative window");
    if (requests == 0 || tokens == 0 || max_query == 0) return KMLL_OK;
    KMLL_REQUIRE_PTR(query);
    KMLL_REQUIRE_PTR(query_start);
    KMLL_REQUIRE_PTR(context);
    KMLL_REQUIRE_PTR(block_table);
    KMLL_REQUIRE_PTR(out);
    PagedArgs a = {query, query_start, context, block_table, table_width, requests, tokens, heads, kv_heads, head_dim, block, pages, k_codes, v_codes,
                   k_scales, v_scales, scale * 1.4426950408889634f, window, out, max_query, 0};
    const long long max_rows = (long long)max_query * (heads / kv_heads);
    if (paged_decode_serves(head_dim) && (reinterpret_cast<uintptr_t>(query) & 15u) == 0) {
        KMLL_REQUIRE_PTR(workspace);
        KMLL_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 15u) == 0, "paged attention: the workspace must be 16-byte aligned");
        const int limit = few_rows(max_rows, heads / kv_heads);
        if ((long long)requests * kv_heads > kPagedCounters)
            return fail(KMLL_ERR_CAPACITY, "paged attention: %d requests of %d kv heads, at most %d together", requests, kv_heads, kPagedCounters);
        int* const counters = static_cast<int*>(workspace);
        unsigned char* const scratch = static_cast<unsigned char*>(workspace) + kPagedZeroBytes;
        unsigned char* const rest = static_cast<unsigned char*>(workspace) + (kPagedZeroBytes + paged_decode_scratch_bytes(head_dim, limit) + 255) / 256 * 256;
        const bool many = max_rows > kPagedDecodeRows && paged_prompt_serves(a);
        if (many && !paged_prompt_fits(a)) return fail(KMLL_ERR_CAPACITY, "paged attention: %d tokens of %d heads in one call", tokens, heads);
        a.skip_rows = limit;
        KMLL_TRY_RC(paged_decode_launch(as_stream(stream), a, is_f32 != 0, limit, max_context, counters, scratch,
                                        many ? paged_prompt_order(a, rest) : PagedOrder{nullptr, 0, 0}));
        if (max_rows <= kPagedDecodeRows) return check_launch("paged attention");
        if (many) {
            KMLL_TRY_RC(paged_prompt_launch(as_stream(stream), a, is_f32 != 0, counters + kPagedCounters, rest));
            return check_launch("paged attention");
        }
    }
    const cudaError_t e = is_f32 ? launch(paged_rows_kernel<float>, dim3(tokens, kv_heads), dim3(128), 0, as_stream(stream), true, a)
                                 : launch(paged_rows_kernel<uint16_t>, dim3(tokens, kv_heads), dim3(128), 0, as_stream(stream), true, a);
    if (e != cudaSuccess) return fail(KMLL_ERR_CUDA, "paged attention: %s", cudaGetErrorString(e));
    return check_launch("paged attention");
}
