// The paged 8-bit cache of requests of unequal length: the pages of a step, rotation and storage of its rows, reading rows back.
//
// A page holds `block` tokens of every kv head, as int8 codes and one f32 scale for each (page, head): value = code * scale, scale = (largest
// magnitude written to the page so far) / 127, the rule of the RS-I8 weights.  Codes lie the way the products read them, in groups of 16
// bytes along the axis that is summed over: keys [page][head][dim / 16][token][16], values [page][head][token / 16][dim][16].  Both are
// operand rows of the 8-bit tensor-core instructions as they lie (a contraction runs along the bytes of a group), eight groups are 128
// bytes without bank conflicts, and a page of a head is one run of block * head_dim bytes.
#include <climits>

#include "internal.cuh"
#include "paged.cuh"

namespace kmll {
namespace {

// ---- pages of a step ------------------------------------------------------------------------------------------------------
constexpr int kPlanThreads = 512;
constexpr int kPlanMaxRequests = 8192;

struct PlanArgs {
    const int32_t *lengths, *new_tokens;
    int requests, block;
    int32_t* table;
    int width;
    const int32_t* free_blocks;
    int free_capacity;
    const int32_t* free_count;
    int capacity;
    int32_t *context, *query_start, *positions, *slots, *free_count_out, *status;
};

// Sums over the threads in front of this one, and over all of them.
__device__ inline longlong2 plan_scan(longlong2 v, longlong2& whole, longlong2* scratch) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    longlong2 s = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long a = __shfl_up_sync(0xffffffffu, s.x, o), b = __shfl_up_sync(0xffffffffu, s.y, o);
        if (lane >= o) { s.x += a; s.y += b; }
    }
    if (lane == 31) scratch[warp] = s;
    __syncthreads();
    longlong2 before = make_longlong2(0, 0);
    whole = before;
    for (int w = 0; w < kPlanThreads / 32; ++w) {
        if (w == warp) before = whole;
        whole.x += scratch[w].x;
        whole.y += scratch[w].y;
    }
    return make_longlong2(before.x + s.x - v.x, before.y + s.y - v.y);
}

// Every block of the cluster sums all requests (a few loads each), then takes its share of the tokens; nothing is written before all blocks
// have read, so the outputs may be the inputs' own buffers.  Latency: one load, one scan, one dependent load (the page), one store.
__global__ void __launch_bounds__(kPlanThreads) paged_plan_kernel(const PlanArgs a) {
    extern __shared__ int32_t plan_smem[];
    __shared__ longlong2 scratch[kPlanThreads / 32];
    int32_t* const s_len = plan_smem;
    int32_t* const s_start = s_len + a.requests;      // tokens in front of the request
    int32_t* const s_taken = s_start + a.requests + 1;  // pages taken in front of it
    const int tid = threadIdx.x, blocks = (int)gridDim.x;
    const int per = (a.requests + kPlanThreads - 1) / kPlanThreads;
    pdl_wait();
    const long long count = *a.free_count;
    longlong2 mine = make_longlong2(0, 0);
    int bad = 0;
    for (int i = 0; i < per; ++i) {
        const int r = tid * per + i;
        if (r >= a.requests) break;
        const long long c = a.lengths[r], n = a.new_tokens[r];
        if (c < 0 || n < 0) { bad = max(bad, 3); continue; }
        if (c + n > (long long)a.width * a.block) { bad = max(bad, 2); continue; }
        mine.x += n;
        mine.y += (c + n + a.block - 1) / a.block - (c + a.block - 1) / a.block;
    }
    longlong2 whole;
    longlong2 at = plan_scan(mine, whole, scratch);
    bad = __syncthreads_or(bad == 3) ? 3 : __syncthreads_or(bad == 2) ? 2 : 0;
    if (bad == 0 && (count < 0 || count > a.free_capacity || whole.x > a.capacity)) bad = 3;
    if (bad == 0 && whole.y > count) bad = 1;
    for (int i = 0; i < per; ++i) {
        const int r = tid * per + i;
        if (r >= a.requests) break;
        const int c = a.lengths[r], n = bad ? 0 : a.new_tokens[r];
        s_len[r] = c;
        s_start[r] = bad ? 0 : (int)at.x;
        s_taken[r] = bad ? 0 : (int)at.y;
        if (bad) continue;
        at.x += n;
        at.y += (c + n + a.block - 1) / a.block - (c + a.block - 1) / a.block;
    }
    const int total = bad ? 0 : (int)whole.x;
    if (tid == 0) s_start[a.requests] = total;
    __syncthreads();
    if (blocks > 1) {
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
    for (int r = blockIdx.x * kPlanThreads + tid; r <= a.requests; r += blocks * kPlanThreads) {
        a.query_start[r] = s_start[r];
        if (r < a.requests) a.context[r] = s_len[r] + s_start[r + 1] - s_start[r];
    }
    if (blockIdx.x == 0 && tid == 0) {
        *a.free_count_out = (int32_t)(bad ? count : count - whole.y);
        *a.status = bad;
    }
    for (int t = blockIdx.x * kPlanThreads + tid; t < a.capacity; t += blocks * kPlanThreads) {
        int pos = 0, slot = -1;
        if (t < total) {
            int lo = 0, hi = a.requests - 1;  // the last request that starts at or before t (those without tokens in between start there too)
            while (lo < hi) {
                const int mid = (lo + hi + 1) >> 1;
                if (s_start[mid] <= t) lo = mid;
                else hi = mid - 1;
            }
            pos = s_len[lo] + t - s_start[lo];
            const int held = (s_len[lo] + a.block - 1) / a.block, b = pos / a.block;
            int32_t* const entry = a.table + (size_t)lo * a.width + b;
            int page;
            if (b >= held) {
                page = a.free_blocks[(int)count - 1 - (s_taken[lo] + b - held)];
                if (pos % a.block == 0) *entry = page;
            } else {
                page = *entry;
            }
            slot = page * a.block + pos % a.block;
        }
        a.positions[t] = pos;
        a.slots[t] = slot;
    }
}

// Pages of the requests that have ended go back on the stack, request after request, first page first.
__global__ void __launch_bounds__(kPlanThreads) paged_release_kernel(const int32_t* context, const int32_t* ended, int requests, int block, int32_t* table, int width,
                                                                     int32_t* free_blocks, int free_capacity, const int32_t* free_count, int32_t* context_out,
                                                                     int32_t* free_count_out, int32_t* status) {
    extern __shared__ int32_t plan_smem[];
    __shared__ longlong2 scratch[kPlanThreads / 32];
    int32_t* const s_pages = plan_smem;
    int32_t* const s_at = s_pages + requests;
    const int tid = threadIdx.x, per = (requests + kPlanThreads - 1) / kPlanThreads;
    pdl_wait();
    const long long count = *free_count;
    longlong2 mine = make_longlong2(0, 0);
    int bad = 0;
    for (int i = 0; i < per; ++i) {
        const int r = tid * per + i;
        if (r >= requests) break;
        const long long c = context[r], n = (c + block - 1) / block;
        if (c < 0 || n > width) bad = 1;
        s_pages[r] = ended[r] != 0 && c >= 0 && n <= width ? (int)n : 0;
        mine.x += s_pages[r];
    }
    longlong2 whole;
    long long at = plan_scan(mine, whole, scratch).x;
    bad = __syncthreads_or(bad) ? 3 : count < 0 || count + whole.x > free_capacity ? 1 : 0;
    for (int i = 0; i < per; ++i) {
        const int r = tid * per + i;
        if (r >= requests) break;
        s_at[r] = (int)(count + at);
        at += s_pages[r];
        context_out[r] = !bad && ended[r] != 0 ? 0 : context[r];
    }
    __syncthreads();
    if (tid == 0) {
        *free_count_out = (int32_t)(bad ? count : count + whole.x);
        *status = bad;
    }
    if (bad) return;
    for (int r = tid >> 5; r < requests; r += kPlanThreads / 32)
        for (int i = tid & 31; i < s_pages[r]; i += 32) {
            int32_t* const entry = table + (size_t)r * width + i;
            free_blocks[s_at[r] + i] = *entry;
            *entry = -1;
        }
}

// ---- rotation and storage -------------------------------------------------------------------------------------------------
// sin and cos of x >= 0 in 64 bits: x less the nearest multiple of pi / 2 (pi / 2 as a sum of two doubles), then Taylor's series, whose
// first term left out is below 1e-15 on [-pi / 4, pi / 4].  Half of the instructions of the library's sincos, which keeps a path for huge
// arguments; positions are 31 bits.
__device__ inline double2 sin_cos(double x) {
    constexpr double kPi2Hi = 1.5707963267948966, kPi2Lo = 6.123233995736766e-17;
    const double k = rint(x * (1.0 / kPi2Hi));
    const double r = fma(-k, kPi2Lo, fma(-k, kPi2Hi, x)), z = r * r;
    double s = -1.0 / 1307674368000.0, c = -1.0 / 87178291200.0;  // 15!, 14!
    s = fma(s, z, 1.0 / 6227020800.0);
    c = fma(c, z, 1.0 / 479001600.0);
    s = fma(s, z, -1.0 / 39916800.0);
    c = fma(c, z, -1.0 / 3628800.0);
    s = fma(s, z, 1.0 / 362880.0);
    c = fma(c, z, 1.0 / 40320.0);
    s = fma(s, z, -1.0 / 5040.0);
    c = fma(c, z, -1.0 / 720.0);
    s = fma(s, z, 1.0 / 120.0);
    c = fma(c, z, 1.0 / 24.0);
    s = fma(s, z, -1.0 / 6.0);
    c = fma(c, z, -0.5);
    s = fma(s * z, r, r);
    c = fma(c, z, 1.0);
    const int quarter = (int)((long long)k & 3);
    const double a = quarter & 1 ? c : s, b = quarter & 1 ? s : c;
    return make_double2(quarter & 2 ? -a : a, quarter == 1 || quarter == 2 ? -b : b);
}

struct PrepareArgs {
    const void *query, *key, *value;
    int f32;
    size_t ldq, ldk, ldv;
    const float* freqs;
    int n_freqs;
    const int32_t *positions, *slots;
    int tokens, heads, kv_heads, head_dim;
    void* query_rot;
    int8_t *k_codes, *v_codes;
    float *k_scales, *v_scales;
    int pages, block, group;  // group: tokens whose runs a block of threads takes
};

template <typename T>
__device__ inline float load_as_f32(const T* p);
template <>
__device__ inline float load_as_f32<float>(const float* p) { return *p; }
template <>
__device__ inline float load_as_f32<uint16_t>(const uint16_t* p) { return bf16_bits_to_f32(*p); }

// The nearest whole number to v * inv = v / scale, ties to even as the quotient itself has them: where the product is within its rounding
// error of a tie the quotient decides.
__device__ inline int code_of(double v, double scale, double inv) {
    if (inv == 0.0) return 0;  // (a page of zeros)
    const double t = v * inv, n = rint(t);
    const double c = fabs(fabs(t - n) - 0.5) < 1e-9 ? rint(v / scale) : n;
    return (int)fmin(fmax(c, -127.0), 127.0);
}
// A value that is not finite must not spoil its page: an infinity takes the largest code, NaN counts as 0.
__device__ inline bool is_finite(double v) { return fabs(v) < 1e300; }

constexpr int kPrepareThreads = 128;

// Blocks (x, y): y < kv_heads keys, y < 2 * kv_heads values of one head, above that query heads.  A run is a stretch of tokens with ascending
// slots in one page; the thread block whose tokens hold the first of a run takes all of it, so that a page's scale is known in one place.
template <typename T>
__global__ void __launch_bounds__(kPrepareThreads) prepare_paged_kernel(const PrepareArgs a) {
    __shared__ float scratch[33];
    const int tid = threadIdx.x, t0 = blockIdx.x * a.group, t1 = min(a.tokens, t0 + a.group), hd = a.head_dim, half = a.n_freqs;
    const int y = blockIdx.y;
    pdl_wait();
    const int limit = a.pages * a.block;
    if (y >= 2 * a.kv_heads) {
        const int h = y - 2 * a.kv_heads, items = half + (hd - 2 * half);
        for (int i = tid; i < (t1 - t0) * items; i += kPrepareThreads) {
            const int t = t0 + i / items, d = i % items;
            const int slot = a.slots[t];
            if (slot < 0 || slot >= limit) continue;
            const T* src = static_cast<const T*>(a.query) + (size_t)t * a.ldq + (size_t)h * hd;
            T* dst = static_cast<T*>(a.query_rot) + ((size_t)t * a.heads + h) * hd;
            if (d >= half) {
                dst[d + half] = src[d + half];
                continue;
            }
            const double2 sc = sin_cos((double)a.positions[t] * (double)a.freqs[d]);
            const double u = load_as_f32(src + d), v = load_as_f32(src + d + half);
            const float p = (float)(u * sc.y - v * sc.x), q = (float)(u * sc.x + v * sc.y);
            if constexpr (sizeof(T) == 4) {
                dst[d] = p;
                dst[d + half] = q;
            } else {
                dst[d] = f32_to_bf16_bits(p);
                dst[d + half] = f32_to_bf16_bits(q);
            }
        }
        return;
    }
    const bool keys = y < a.kv_heads;
    const int h = keys ? y : y - a.kv_heads;
    const T* const in = static_cast<const T*>(keys ? a.key : a.value) + (size_t)h * hd;
    const size_t ld = keys ? a.ldk : a.ldv;
    const int turned = keys ? half : 0;
    // entries d and (for d < turned) d + turned of token t
    auto pair = [&](int t, int d, double& u, double& v) {
        const T* src = in + (size_t)t * ld;
        if (d >= turned) {
            u = load_as_f32(src + d + turned);
            v = 0.0;
            return;
        }
        const double2 sc = sin_cos((double)a.positions[t] * (double)a.freqs[d]);
        const double p = load_as_f32(src + d), q = load_as_f32(src + d + turned);
        u = p * sc.y - q * sc.x;
        v = p * sc.x + q * sc.y;
    };
    const int items = hd - turned;
    for (int t = t0; t < t1; ++t) {
        const int slot = a.slots[t];
        if (slot < 0 || slot >= limit) continue;
        const int at = slot % a.block, page = slot / a.block;
        if (at != 0 && t > 0 && a.slots[t - 1] == slot - 1) continue;
        int n = 1;
        while (at + n < a.block && t + n < a.tokens && a.slots[t + n] == slot + n) ++n;
        double largest = 0.0;
        for (int i = tid; i < n * items; i += kPrepareThreads) {
            double u, v;
            pair(t + i / items, i % items, u, v);
            if (is_finite(u)) largest = fmax(largest, fabs(u));
            if (is_finite(v)) largest = fmax(largest, fabs(v));
        }
        const float top = block_max((float)(largest / 127.0), scratch);
        float* const scale_at = (keys ? a.k_scales : a.v_scales) + (size_t)page * a.kv_heads + h;
        int8_t* const codes = (keys ? a.k_codes : a.v_codes) + ((size_t)page * a.kv_heads + h) * a.block * hd;
        auto place = [&](int token, int d) { return keys ? ((d >> 4) * a.block + token) * 16 + (d & 15) : ((token >> 4) * hd + d) * 16 + (token & 15); };
        const float before = at == 0 ? 0.0f : *scale_at, scale = fmaxf(top, before);
        const double s = scale, inv = scale > 0.0f ? 1.0 / s : 0.0;
        __syncthreads();  // (all have read the scale)
        if (tid == 0) *scale_at = scale;
        if (scale > before && at > 0) {
            for (int i = tid; i < at * hd; i += kPrepareThreads) {
                int8_t* const c = codes + place(i / hd, i % hd);
                *c = (int8_t)code_of((double)*c * (double)before, s, inv);
            }
        }
        for (int i = tid; i < n * items; i += kPrepareThreads) {
            double u, v;
            const int d = i % items, token = at + i / items;
            pair(t + i / items, d, u, v);
            if (!(u == u)) u = 0.0;
            if (!(v == v)) v = 0.0;
            if (d < turned) {
                codes[place(token, d)] = (int8_t)code_of(u, s, inv);
                codes[place(token, d + turned)] = (int8_t)code_of(v, s, inv);
            } else {
                codes[place(token, d + turned)] = (int8_t)code_of(u, s, inv);
            }
        }
        __syncthreads();
    }
}

// Rows of the cache as f32; slots outside of it leave their row as it is.
__global__ void paged_cache_rows_kernel(const int8_t* k_codes, const float* k_scales, const int8_t* v_codes, const float* v_scales, int pages, int block, int kv_heads,
                                        int head_dim, const int32_t* slots, int count, float* k, float* v) {
    pdl_wait();
    const int row_len = kv_heads * head_dim;
    for (int r = blockIdx.x; r < count; r += gridDim.x) {
        const int slot = slots[r];
        if (slot < 0 || slot >= pages * block) continue;
        const int page = slot / block, at = slot % block;
        for (int i = threadIdx.x; i < row_len; i += blockDim.x) {
            const int h = i / head_dim, d = i % head_dim;
            const size_t ph = (size_t)page * kv_heads + h, base = ph * block * head_dim;
            k[(size_t)r * row_len + i] = (float)k_codes[base + ((d >> 4) * block + at) * 16 + (d & 15)] * k_scales[ph];
            v[(size_t)r * row_len + i] = (float)v_codes[base + ((at >> 4) * head_dim + d) * 16 + (at & 15)] * v_scales[ph];
        }
    }
}

}  // namespace

int check_paged_cache(const char* who, const void* k_codes, const void* k_scales, const void* v_codes, const void* v_scales, int pages, int block, int kv_heads, int head_dim) {
    if (k_codes == nullptr || k_scales == nullptr || v_codes == nullptr || v_scales == nullptr) return fail(KMLL_ERR_NULL, "%s: null cache pointer", who);
    KMLL_REQUIRE(block == 16 || block == 32 || block == 64 || block == 128, "%s: a page holds 16, 32, 64 or 128 tokens, got %d", who, block);
    KMLL_REQUIRE(pages > 0 && (long long)pages * block <= INT_MAX, "%s: %d pages of %d tokens: slots are 32 bits", who, pages, block);
    KMLL_REQUIRE(kv_heads > 0 && kv_heads <= 1024, "%s: %d kv heads", who, kv_heads);
    KMLL_REQUIRE(head_dim >= 16 && head_dim <= 256 && head_dim % 16 == 0, "%s: head size %d is not a multiple of 16 up to 256", who, head_dim);
    KMLL_REQUIRE(((reinterpret_cast<uintptr_t>(k_codes) | reinterpret_cast<uintptr_t>(v_codes)) & 15u) == 0, "%s: codes must be 16-byte aligned", who);
    return KMLL_OK;
}

}  // namespace kmll

using namespace kmll;

extern "C" int kmll_paged_plan(kmll_stream_t stream, const int32_t* lengths, const int32_t* new_tokens, int requests, int block, int32_t* block_table, int table_width,
                               const int32_t* free_blocks, int free_capacity, const int32_t* free_count, int token_capacity, int32_t* context, int32_t* query_start,
                               int32_t* positions, int32_t* slots, int32_t* free_count_out, int32_t* status) {
    KMLL_REQUIRE(requests >= 0 && token_capacity >= 0 && table_width >= 0 && free_capacity >= 0, "paged plan: negative size");
    if (requests > kPlanMaxRequests) return fail(KMLL_ERR_CAPACITY, "paged plan: %d requests, at most %d", requests, kPlanMaxRequests);
    KMLL_REQUIRE(block == 16 || block == 32 || block == 64 || block == 128, "paged plan: a page holds 16, 32, 64 or 128 tokens, got %d", block);
    KMLL_REQUIRE((long long)table_width * block <= INT_MAX, "paged plan: a table of %d pages of %d tokens: positions are 32 bits", table_width, block);
    KMLL_REQUIRE_PTR(free_count);
    KMLL_REQUIRE_PTR(query_start);
    KMLL_REQUIRE_PTR(free_count_out);
    KMLL_REQUIRE_PTR(status);
    if (requests > 0) {
        KMLL_REQUIRE_PTR(lengths);
        KMLL_REQUIRE_PTR(new_tokens);
        KMLL_REQUIRE_PTR(block_table);
        KMLL_REQUIRE_PTR(context);
    }
    if (free_capacity > 0) KMLL_REQUIRE_PTR(free_blocks);
    if (token_capacity > 0) {
        KMLL_REQUIRE_PTR(positions);
        KMLL_REQUIRE_PTR(slots);
    }
    const PlanArgs a = {lengths, new_tokens, requests, block, block_table, table_width, free_blocks, free_capacity, free_count, token_capacity, context, query_start,
                        positions, slots, free_count_out, status};
    const int cluster = token_capacity > 2 * kPlanThreads ? 8 : 1;
    cudaError_t e = allow_all_dynamic_smem(paged_plan_kernel);
    if (e == cudaSuccess)
        e = launch_cluster(paged_plan_kernel, dim3(cluster), cluster, dim3(kPlanThreads), (3 * (size_t)requests + 2) * 4, as_stream(stream), true, a);
    if (e != cudaSuccess) return fail(KMLL_ERR_CUDA, "paged plan: %s", cudaGetErrorString(e));
    return check_launch("paged plan");
}

extern "C" int kmll_paged_release(kmll_stream_t stream, const int32_t* context, const int32_t* ended, int requests, int block, int32_t* block_table, int table_width,
                                  int32_t* free_blocks, int free_capacity, const int32_t* free_count, int32_t* context_out, int32_t* free_count_out, int32_t* status) {
    KMLL_REQUIRE(requests >= 0 && table_width >= 0 && free_capacity >= 0, "paged release: negative size");
    if (requests > kPlanMaxRequests) return fail(KMLL_ERR_CAPACITY, "paged release: %d requests, at most %d", requests, kPlanMaxRequests);
    KMLL_REQUIRE(block == 16 || block == 32 || block == 64 || block == 128, "paged release: a page holds 16, 32, 64 or 128 tokens, got %d", block);
    KMLL_REQUIRE_PTR(free_count);
    KMLL_REQUIRE_PTR(free_count_out);
    KMLL_REQUIRE_PTR(status);
    if (requests > 0) {
        KMLL_REQUIRE_PTR(context);
        KMLL_REQUIRE_PTR(ended);
        KMLL_REQUIRE_PTR(block_table);
        KMLL_REQUIRE_PTR(context_out);
    }
    if (free_capacity > 0) KMLL_REQUIRE_PTR(free_blocks);
    cudaError_t e = allow_all_dynamic_smem(paged_release_kernel);
    if (e == cudaSuccess)
        e = launch(paged_release_kernel, dim3(1), dim3(kPlanThreads), 2 * (size_t)requests * 4, as_stream(stream), true, context, ended, requests, block, block_table,
                   table_width, free_blocks, free_capacity, free_count, context_out, free_count_out, status);
    if (e != cudaSuccess) return fail(KMLL_ERR_CUDA, "paged release: %s", cudaGetErrorString(e));
    return check_launch("paged release");
}

extern "C" int kmll_prepare_paged_attention(kmll_stream_t stream, const void* query, int ld_query, const void* key, int ld_key, const void* value, int ld_value, int is_f32,
                                            const float* freqs, int n_freqs, const int32_t* positions, const int32_t* slots, int tokens, int heads, int kv_heads,
                                            int head_dim, void* query_rot, int8_t* k_codes, float* k_scales, int8_t* v_codes, float* v_scales, int pages, int block) {
    KMLL_REQUIRE(tokens >= 0, "prepare paged attention: negative token count");
    KMLL_TRY_RC(check_paged_cache("prepare paged attention", k_codes, k_scales, v_codes, v_scales, pages, block, kv_heads, head_dim));
    KMLL_REQUIRE(heads >= 0 && heads <= 4096, "prepare paged attention: %d query heads", heads);
    KMLL_REQUIRE(n_freqs >= 0 && 2 * n_freqs <= head_dim, "prepare paged attention: frequency count %d exceeds half the head size %d", n_freqs, head_dim);
    KMLL_REQUIRE(query_rot != query || ld_query == heads * head_dim || tokens <= 1, "prepare paged attention: rows that do not lie together cannot turn in place");
    KMLL_REQUIRE(ld_query >= heads * head_dim && ld_key >= kv_heads * head_dim && ld_value >= kv_heads * head_dim, "prepare paged attention: rows overlap");
    if (tokens == 0) return KMLL_OK;
    KMLL_REQUIRE_PTR(key);
    KMLL_REQUIRE_PTR(value);
    KMLL_REQUIRE_PTR(slots);
    if (heads > 0) {
        KMLL_REQUIRE_PTR(query);
        KMLL_REQUIRE_PTR(query_rot);
    }
    if (n_freqs > 0) {
        KMLL_REQUIRE_PTR(freqs);
        KMLL_REQUIRE_PTR(positions);
    }
    PrepareArgs a = {query, key, value, is_f32, (size_t)ld_query, (size_t)ld_key, (size_t)ld_value, freqs, n_freqs, positions, slots, tokens, heads, kv_heads, head_dim,
                     query_rot, k_codes, v_codes, k_scales, v_scales, pages, block, 1};
    if (tokens > 512) a.group = block;
    const dim3 grid((tokens + a.group - 1) / a.group, 2 * kv_heads + heads);
    const cudaError_t e = is_f32 ? launch(prepare_paged_kernel<float>, grid, dim3(kPrepareThreads), 0, as_stream(stream), true, a)
                                 : launch(prepare_paged_kernel<uint16_t>, grid, dim3(kPrepareThreads), 0, as_stream(stream), true, a);
    if (e != cudaSuccess) return fail(KMLL_ERR_CUDA, "prepare paged attention: %s", cudaGetErrorString(e));
    return check_launch("prepare paged attention");
}

extern "C" int kmll_paged_cache_rows(kmll_stream_t stream, const int8_t* k_codes, const float* k_scales, const int8_t* v_codes, const float* v_scales, int pages, int block,
                                     int kv_heads, int head_dim, const int32_t* slots, int count, float* k, float* v) {
    KMLL_REQUIRE(count >= 0, "paged cache rows: negative row count");
    KMLL_TRY_RC(check_paged_cache("paged cache rows", k_codes, k_scales, v_codes, v_scales, pages, block, kv_heads, head_dim));
    if (count == 0) return KMLL_OK;
    KMLL_REQUIRE_PTR(slots);
    KMLL_REQUIRE_PTR(k);
    KMLL_REQUIRE_PTR(v);
    const cudaError_t e = launch(paged_cache_rows_kernel, dim3(min(count, 8192)), dim3(256), 0, as_stream(stream), true, k_codes, k_scales, v_codes, v_scales, pages, block,
                                 kv_heads, head_dim, slots, count, k, v);
    if (e != cudaSuccess) return fail(KMLL_ERR_CUDA, "paged cache rows: %s", cudaGetErrorString(e));
    return check_launch("paged cache rows");
}
