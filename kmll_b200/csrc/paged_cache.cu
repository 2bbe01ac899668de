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
    size_t ldq, ldk, ldv;
    const float* freqs;
    int n_freqs;
    const int32_t *positions, *slots;
    int tokens, heads, kv_heads, head_dim;
    void* query_rot;
    int8_t *k_codes, *v_codes;
    float *k_scales, *v_scales;
    int pages, block;
    int group, groups;      // tokens whose runs a block of threads takes, and how many such blocks for a set of heads
    int head_sets;          // of kHeadSet kv heads
    int q_tokens;           // query rows' tokens of a block of threads
    int table_tokens;       // tokens whose angles fit into shared memory
};

template <typename T>
__device__ inline float load_as_f32(const T* p);
template <>
__device__ inline float load_as_f32<float>(const float* p) { return *p; }
template <>
__device__ inline float load_as_f32<uint16_t>(const uint16_t* p) { return bf16_bits_to_f32(*p); }
__device__ inline float2 load_pair(const float* p) { return *reinterpret_cast<const float2*>(p); }
__device__ inline float2 load_pair(const uint16_t* p) {
    const uint32_t u = *reinterpret_cast<const uint32_t*>(p);
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}
__device__ inline void store_one(float* p, float v) { *p = v; }
__device__ inline void store_one(uint16_t* p, float v) { *p = f32_to_bf16_bits(v); }
__device__ inline void store_pair(float* p, float x, float y) { *reinterpret_cast<float2*>(p) = make_float2(x, y); }
__device__ inline void store_pair(uint16_t* p, float x, float y) { *reinterpret_cast<uint32_t*>(p) = f32_to_bf16_bits(x) | ((uint32_t)f32_to_bf16_bits(y) << 16); }

// The nearest whole number to v * inv = v / scale, ties to even as the quotient itself has them: where the product is within its rounding
// error of a tie the quotient decides.
__device__ inline int code_of(double v, double scale, double inv) {
    if (inv == 0.0) return 0;  // (a page of zeros)
    const double t = v * inv, n = rint(t);
    const double c = fabs(fabs(t - n) - 0.5) < 1e-9 ? rint(v / scale) : n;
    return (int)fmin(fmax(c, -127.0), 127.0);
}
// A value that is not finite must not spoil its page: an infinity takes the largest code, NaN counts as 0.
__device__ inline double finite_size(double v) { return fabs(v) < 1e300 ? fabs(v) : 0.0; }

constexpr int kPrepareThreads = 256;
constexpr int kHeadSet = 4, kHeadThreads = kPrepareThreads / kHeadSet;  // kv heads of a block of threads; threads of one

// Blocks of threads along x: keys (groups of tokens x sets of heads), values (the same), query rows.  A run is a stretch of tokens with ascending
// slots in one page; the block whose tokens hold the first of a run takes all of it, so that a page's scale is known in one place.  A head has 64
// threads, a thread the same entries of every token; the first walk over the run finds the largest magnitude, the second (out of L1 / L2) codes.
// The angles of a token are computed once per block into shared memory, not for every head.  VEC: entries lie so that two load together.
template <typename T, int VEC>
__global__ void __launch_bounds__(kPrepareThreads) prepare_paged_kernel(const PrepareArgs a) {
    extern __shared__ __align__(16) double2 table[];  // [token][n_freqs] sine, cosine
    __shared__ int s_slots[2 * 128 + 1];
    __shared__ int s_run;
    __shared__ float s_top[kPrepareThreads / 32];
    const int tid = threadIdx.x, hd = a.head_dim, half = a.n_freqs, limit = a.pages * a.block;
    const int kv_blocks = a.groups * a.head_sets;
    pdl_wait();
    if ((int)blockIdx.x >= 2 * kv_blocks) {
        // ---- query rows: a warp has a row at a time
        const int t0 = ((int)blockIdx.x - 2 * kv_blocks) * a.q_tokens, n = min(a.q_tokens, a.tokens - t0), lane = tid & 31, warp = tid >> 5;
        for (int i = tid; i < n * half; i += kPrepareThreads) table[i] = sin_cos((double)a.positions[t0 + i / half] * (double)a.freqs[i % half]);
        __syncthreads();
        for (int t = 0; t < n; ++t) {
            const int slot = a.slots[t0 + t];
            if (slot < 0 || slot >= limit) continue;
            const double2* const turn = table + t * half;
            const T* const src = static_cast<const T*>(a.query) + (size_t)(t0 + t) * a.ldq;
            T* const dst = static_cast<T*>(a.query_rot) + (size_t)(t0 + t) * a.heads * hd;
#pragma unroll 2
            for (int h = warp; h < a.heads; h += kPrepareThreads / 32) {
                for (int d = lane * VEC; d < half; d += 32 * VEC) {
                    const T* const at = src + h * hd + d;
                    T* const to = dst + h * hd + d;
                    if constexpr (VEC == 2) {
                        const float2 u = load_pair(at), v = load_pair(at + half);
                        const double2 s0 = turn[d], s1 = turn[d + 1];
                        store_pair(to, (float)(u.x * s0.y - v.x * s0.x), (float)(u.y * s1.y - v.y * s1.x));
                        store_pair(to + half, (float)(u.x * s0.x + v.x * s0.y), (float)(u.y * s1.x + v.y * s1.y));
                    } else {
                        const double u = load_as_f32(at), v = load_as_f32(at + half);
                        const double2 s0 = turn[d];
                        store_one(to, (float)(u * s0.y - v * s0.x));
                        store_one(to + half, (float)(u * s0.x + v * s0.y));
                    }
                }
                for (int d = 2 * half + lane; d < hd; d += 32) dst[h * hd + d] = src[h * hd + d];
            }
        }
        return;
    }
    const bool keys = (int)blockIdx.x < kv_blocks;
    const int item = keys ? blockIdx.x : blockIdx.x - kv_blocks, set = item % a.head_sets, t0 = item / a.head_sets * a.group, t1 = min(a.tokens, t0 + a.group);
    const int sub = tid / kHeadThreads, lt = tid % kHeadThreads, h = set * kHeadSet + sub;
    const bool live = h < a.kv_heads;
    const T* const in = static_cast<const T*>(keys ? a.key : a.value) + (size_t)(live ? h : 0) * hd;
    const size_t ld = keys ? a.ldk : a.ldv;
    const int turned = keys ? half : 0;
    // slots of the tokens t0 - 1 .. (every run that begins here ends among them)
    for (int i = tid; i <= a.group + a.block; i += kPrepareThreads) {
        const int t = t0 - 1 + i;
        s_slots[i] = t >= 0 && t < a.tokens ? a.slots[t] : INT_MIN;
    }
    __syncthreads();
    for (int t = t0; t < t1; ++t) {
        const int* const slots = s_slots + (t - t0 + 1);
        const int slot = slots[0];
        if (slot < 0 || slot >= limit) continue;
        const int at = slot % a.block, page = slot / a.block;
        if (at != 0 && t > 0 && slots[-1] == slot - 1) continue;
        // ---- length of the run: up to the first token that does not follow
        if (tid == 0) s_run = min(a.block - at, a.tokens - t);
        __syncthreads();
        for (int i = tid; i < a.block - at; i += kPrepareThreads)
            if (slots[i] != slot + i) atomicMin(&s_run, i);
        __syncthreads();
        const int n = s_run;
        const bool kept = n <= a.table_tokens;  // the angles of the whole run stay in shared memory
        auto angles = [&](int i0, int i1) {
            __syncthreads();
            for (int i = tid; i < (i1 - i0) * turned; i += kPrepareThreads) table[i] = sin_cos((double)a.positions[t + i0 + i / turned] * (double)a.freqs[i % turned]);
            __syncthreads();
        };
        // calls f(token of the run, entry, value) for this thread's entries, 64-bit turned values
        auto walk = [&](bool again, auto f) {
            for (int i0 = 0; i0 < n; i0 += a.table_tokens) {
                const int i1 = min(n, i0 + a.table_tokens);
                if (turned > 0 && !(again && kept)) angles(i0, i1);
                if (!live) continue;
                for (int d = lt; d < turned; d += kHeadThreads) {
                    const T* src = in + (size_t)(t + i0) * ld + d;
                    const double2* turn = table + d;
#pragma unroll 8
                    for (int i = i0; i < i1; ++i, src += ld, turn += turned) {
                        const double p = load_as_f32(src), q = load_as_f32(src + turned);
                        const double2 sc = *turn;
                        f(i, d, p * sc.y - q * sc.x);
                        f(i, d + turned, p * sc.x + q * sc.y);
                    }
                }
                for (int d = 2 * turned + lt; d < hd; d += kHeadThreads) {
                    const T* src = in + (size_t)(t + i0) * ld + d;
#pragma unroll 8
                    for (int i = i0; i < i1; ++i, src += ld) f(i, d, (double)load_as_f32(src));
                }
            }
        };
        double largest = 0.0;
        walk(false, [&](int, int, double v) { largest = fmax(largest, finite_size(v)); });
        const float mine = warp_max((float)(largest / 127.0));
        if ((tid & 31) == 0) s_top[tid >> 5] = mine;
        float* const scale_at = (keys ? a.k_scales : a.v_scales) + (size_t)page * a.kv_heads + (live ? h : 0);
        const float before = at == 0 ? 0.0f : *scale_at;
        __syncthreads();  // (all have read the scale)
        const float scale = fmaxf(before, fmaxf(s_top[2 * sub], s_top[2 * sub + 1]));
        static_assert(kHeadThreads == 64, "two warps a head");
        const double s = scale, inv = scale > 0.0f ? 1.0 / s : 0.0;
        int8_t* const codes = (keys ? a.k_codes : a.v_codes) + ((size_t)page * a.kv_heads + (live ? h : 0)) * a.block * hd;
        auto place = [&](int token, int d) { return keys ? ((d >> 4) * a.block + token) * 16 + (d & 15) : ((token >> 4) * hd + d) * 16 + (token & 15); };
        if (live && lt == 0) *scale_at = scale;
        if (live && scale > before && at > 0)
            for (int d = lt; d < hd; d += kHeadThreads)
                for (int i = 0; i < at; ++i) {
                    int8_t* const c = codes + place(i, d);
                    *c = (int8_t)code_of((double)*c * (double)before, s, inv);
                }
        walk(true, [&](int i, int d, double v) { codes[place(at + i, d)] = (int8_t)code_of(v == v ? v : 0.0, s, inv); });
        __syncthreads();
    }
}

// Rows of the cache as f32; slots outside of it leave their row as it is.  A block of threads has 16 entries of the list: of keys a thread reads 16
// bytes (16 entries of a token), of values the 16 tokens of a column, again only where the list moves on to another group of 16.
__global__ void __launch_bounds__(256) paged_cache_rows_kernel(const int8_t* k_codes, const float* k_scales, const int8_t* v_codes, const float* v_scales, int pages, int block,
                                                               int kv_heads, int head_dim, const int32_t* slots, int count, float* k, float* v) {
    __shared__ int s_slots[16];
    const int tid = threadIdx.x, r0 = blockIdx.x * 16, n = min(16, count - r0), row_len = kv_heads * head_dim, units = head_dim / 16, limit = pages * block;
    const int block_log = 31 - __clz(block);
    pdl_wait();
    if (tid < 16) s_slots[tid] = tid < n ? slots[r0 + tid] : -1;
    __syncthreads();
    const bool aligned = (reinterpret_cast<uintptr_t>(k) & 15u) == 0;
    for (int i = tid; i < n * kv_heads * units; i += 256) {
        const int r = i / (kv_heads * units), hc = i - r * kv_heads * units, h = hc / units, c = hc - h * units, slot = s_slots[r];
        if (slot < 0 || slot >= limit) continue;
        const size_t ph = (size_t)(slot >> block_log) * kv_heads + h;
        const uint4 u = *reinterpret_cast<const uint4*>(k_codes + ph * block * head_dim + ((size_t)c * block + (slot & (block - 1))) * 16);
        const float s = k_scales[ph];
        float* const to = k + (size_t)(r0 + r) * row_len + h * head_dim + c * 16;
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const float4 y = make_float4((float)(int8_t)w[b] * s, (float)(int8_t)(w[b] >> 8) * s, (float)(int8_t)(w[b] >> 16) * s, (float)(int8_t)(w[b] >> 24) * s);
            if (aligned) {
                reinterpret_cast<float4*>(to)[b] = y;
            } else {
                to[4 * b] = y.x; to[4 * b + 1] = y.y; to[4 * b + 2] = y.z; to[4 * b + 3] = y.w;
            }
        }
    }
    for (int i = tid; i < row_len; i += 256) {
        const int h = i / head_dim, d = i - h * head_dim;
        uint4 u = make_uint4(0u, 0u, 0u, 0u);
        float s = 0.0f;
        int held = -1;
        for (int r = 0; r < n; ++r) {
            const int slot = s_slots[r];
            if (slot < 0 || slot >= limit) continue;
            if (slot >> 4 != held) {
                held = slot >> 4;
                const size_t ph = (size_t)(slot >> block_log) * kv_heads + h;
                u = *reinterpret_cast<const uint4*>(v_codes + ph * block * head_dim + ((size_t)((slot & (block - 1)) >> 4) * head_dim + d) * 16);
                s = v_scales[ph];
            }
            const uint32_t e = slot & 15, w = e < 4 ? u.x : e < 8 ? u.y : e < 12 ? u.z : u.w;
            v[(size_t)(r0 + r) * row_len + i] = (float)(int8_t)(w >> (8 * (e & 3))) * s;
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
    PrepareArgs a = {query, key, value, (size_t)ld_query, (size_t)ld_key, (size_t)ld_value, freqs, n_freqs, positions, slots, tokens, heads, kv_heads, head_dim,
                     query_rot, k_codes, v_codes, k_scales, v_scales, pages, block};
    // few tokens: each may begin a run; many: they come in pages, and one block of threads per page has no runs that begin elsewhere to step over
    a.group = tokens <= 512 ? 1 : block;
    a.groups = (tokens + a.group - 1) / a.group;
    a.head_sets = (kv_heads + kHeadSet - 1) / kHeadSet;
    a.q_tokens = tokens <= 512 ? 1 : 8;
    const int per_token = n_freqs * (int)sizeof(double2);
    a.table_tokens = per_token > 0 ? min(block, 96 * 1024 / per_token) : block;
    const size_t table_bytes = (size_t)per_token * (tokens <= 512 && a.table_tokens > tokens ? tokens : a.table_tokens);
    const long long blocks = 2ll * a.groups * a.head_sets + (heads > 0 ? (tokens + a.q_tokens - 1) / a.q_tokens : 0);
    KMLL_REQUIRE(blocks <= INT_MAX, "prepare paged attention: too many rows");
    const uintptr_t bits = reinterpret_cast<uintptr_t>(query) | reinterpret_cast<uintptr_t>(query_rot);
    const bool pairs = n_freqs % 2 == 0 && ld_query % 2 == 0 && bits % (is_f32 ? 8 : 4) == 0;
    auto go = [&](auto kern) {
        const cudaError_t e = allow_all_dynamic_smem(kern);
        return e != cudaSuccess ? e : launch(kern, dim3((unsigned)blocks), dim3(kPrepareThreads), table_bytes, as_stream(stream), true, a);
    };
    const cudaError_t e = is_f32 ? pairs ? go(prepare_paged_kernel<float, 2>) : go(prepare_paged_kernel<float, 1>)
                                 : pairs ? go(prepare_paged_kernel<uint16_t, 2>) : go(prepare_paged_kernel<uint16_t, 1>);
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
    const cudaError_t e = launch(paged_cache_rows_kernel, dim3((count + 15) / 16), dim3(256), 0, as_stream(stream), true, k_codes, k_scales, v_codes, v_scales, pages, block,
                                 kv_heads, head_dim, slots, count, k, v);
    if (e != cudaSuccess) return fail(KMLL_ERR_CUDA, "paged cache rows: %s", cudaGetErrorString(e));
    return check_launch("paged cache rows");
}
