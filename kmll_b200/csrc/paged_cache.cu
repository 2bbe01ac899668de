// The paged 8-bit cache of requests of unequal length: the pages of a step, rotation and storage of its rows, reading rows back.
//
// A page holds `block` tokens of every kv head, as int8 codes and one f32 scale for each (page, head): value = code * scale, scale = (largest
// magnitude written to the page so far) / 127, the rule of the RS-I8 weights.  Codes lie the way the products read them, in groups of 16
// bytes along the axis that is summed over: keys [page][head][dim / 16][token][16], values [page][head][token / 16][dim][16].  Both are
// operand rows of the 8-bit tensor-core instructions as they lie (a contraction runs along the bytes of a group), eight groups are 128
// bytes without bank conflicts, and a page of a head is one run of block * head_dim bytes.
#include <climits>
#include <type_traits>

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
// have read, so the outputs may be the inputs' own buffers.  Latency: one load, one scan, one dependent load (the page), one store: 64
// requests of a token 3.4 us, 200 requests with 8117 tokens 5.2 us (eight blocks for more than 1024 tokens).
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

// Pages of the requests that have ended go back on the stack, request after request, first page first; negative entries of the table are no pages.
__global__ void __launch_bounds__(kPlanThreads) paged_release_kernel(const int32_t* context, const int32_t* ended, int requests, int block, int32_t* table, int width,
                                                                     int32_t* free_blocks, int free_capacity, const int32_t* free_count, int32_t* context_out,
                                                                     int32_t* free_count_out, int32_t* status) {
    extern __shared__ int32_t plan_smem[];
    __shared__ longlong2 scratch[kPlanThreads / 32];
    int32_t* const s_entries = plan_smem;           // of the table, of a request that has ended
    int32_t* const s_pages = s_entries + requests;  // those that are pages
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
        s_entries[r] = ended[r] != 0 && c >= 0 && n <= width ? (int)n : 0;
    }
    __syncthreads();
    for (int r = tid >> 5; r < requests; r += kPlanThreads / 32) {
        int pages = 0;
        for (int i = tid & 31; i < s_entries[r]; i += 32) pages += table[(size_t)r * width + i] >= 0 ? 1 : 0;
        pages = __reduce_add_sync(0xffffffffu, pages);
        if ((tid & 31) == 0) s_pages[r] = pages;
    }
    __syncthreads();
    for (int i = 0; i < per && tid * per + i < requests; ++i) mine.x += s_pages[tid * per + i];
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
    for (int r = tid >> 5; r < requests; r += kPlanThreads / 32) {
        int at = s_at[r];
        for (int i0 = 0; i0 < s_entries[r]; i0 += 32) {
            const int i = i0 + (tid & 31);
            int32_t* const entry = table + (size_t)r * width + i;
            const int page = i < s_entries[r] ? *entry : -1;
            const uint32_t there = __ballot_sync(0xffffffffu, page >= 0);
            if (page >= 0) {
                free_blocks[at + __popc(there & ((1u << (tid & 31)) - 1u))] = page;
                *entry = -1;
            }
            at += __popc(there);
        }
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
    int head_sets;          // of HS kv heads
    int q_tokens;           // query rows' tokens of a block of threads
    int table_tokens;       // tokens whose angles fit into shared memory
};

template <typename T>
__device__ inline float load_as_f32(const T* p);
template <>
__device__ inline float load_as_f32<float>(const float* p) { return *p; }
template <>
__device__ inline float load_as_f32<uint16_t>(const uint16_t* p) { return bf16_bits_to_f32(*p); }
// V entries that lie together (4: aligned to all of them)
template <int V>
__device__ inline void load_some(const float* p, float (&x)[V]) {
    if constexpr (V == 4) {
        const float4 u = *reinterpret_cast<const float4*>(p);
        x[0] = u.x; x[1] = u.y; x[2] = u.z; x[3] = u.w;
    } else {
        x[0] = *p;
    }
}
template <int V>
__device__ inline void load_some(const uint16_t* p, float (&x)[V]) {
    if constexpr (V == 4) {
        const uint2 u = *reinterpret_cast<const uint2*>(p);
        x[0] = __uint_as_float(u.x << 16); x[1] = __uint_as_float(u.x & 0xffff0000u);
        x[2] = __uint_as_float(u.y << 16); x[3] = __uint_as_float(u.y & 0xffff0000u);
    } else {
        x[0] = bf16_bits_to_f32(*p);
    }
}
template <int V>
__device__ inline void store_some(float* p, const float (&x)[V]) {
    if constexpr (V == 4) *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
    else *p = x[0];
}
template <int V>
__device__ inline void store_some(uint16_t* p, const float (&x)[V]) {
    if constexpr (V == 4) {
        *reinterpret_cast<uint2*>(p) = make_uint2(bf16_pair_of(x[0], x[1]), bf16_pair_of(x[2], x[3]));
    } else {
        *p = bf16_of(x[0]);
    }
}

// The nearest whole number to v * inv = v / scale, ties to even as the quotient itself has them: where the product is within its rounding
// error of a tie the quotient decides.  Adding 1.5 * 2^52 rounds to a whole number and leaves it in the low word.
__device__ __noinline__ int code_of(double v, double scale, double inv) {
    constexpr double kWhole = 6755399441055744.0;
    double t = v * inv;
    if (!(fabs(t) < 200.0)) return t > 0.0 && inv > 0.0 ? 127 : t < 0.0 && inv > 0.0 ? -127 : 0;  // (infinities; NaN, and a page of zeros: inv is 0)
    if (fabs(fabs(t - ((t + kWhole) - kWhole)) - 0.5) < 1e-9) t = v / scale;
    return min(max(__double2loint(t + kWhole), -127), 127);
}
// The same in 32 bits where they tell: v is an f32 value (v * inv32 is off by 2e-5 of a code) or one that was turned in 32 bits (off by 4e-7 of the
// page's largest: 1e-4 of a code with it); -1000 where a tie may be near or v is at the ends.
__device__ inline int quick_code(float v, float inv32) {
    const float t = v * inv32, n = rintf(t);
    return fabsf(t) < 126.0f && fabsf(fabsf(t - n) - 0.5f) > 2.5e-4f ? (int)n : -1000;
}
__device__ inline int code_of(float v, double scale, double inv, float inv32) {
    const int c = quick_code(v, inv32);
    return c != -1000 ? c : code_of((double)v, scale, inv);
}
// Sine and cosine of an angle as sums of two floats each (48 bits): the first ones turn in 32 bits, all of them in 64.
struct Angle {
    float sin, cos, sin_rest, cos_rest;
    __device__ void set(double2 s) {
        sin = (float)s.x;
        cos = (float)s.y;
        sin_rest = (float)(s.x - (double)sin);
        cos_rest = (float)(s.y - (double)cos);
    }
    __device__ double first(float x, float y) const { return x * ((double)cos + cos_rest) - y * ((double)sin + sin_rest); }
    __device__ double second(float x, float y) const { return x * ((double)sin + sin_rest) + y * ((double)cos + cos_rest); }
};
// A value that is not finite must not spoil its page: an infinity takes the largest code, NaN counts as 0.
__device__ inline double finite_size(double v) { return fabs(v) < 1e300 ? fabs(v) : 0.0; }

constexpr int kPrepareThreads = 256;
constexpr int kPrepareShort = 4;  // tokens of a run that a warp takes

// Angles of `tokens` positions, [token][freq].  A thread has a frequency and kSteps tokens; where their positions follow one another it computes the first
// angle and turns on by one frequency at a time (in 64 bits: kSteps roundings).  It steps through its places without dividing.
__device__ inline void put_angle(double2* to, double2 s) { *to = s; }
__device__ inline void put_angle(Angle* to, double2 s) { to->set(s); }
template <int kSteps, typename A>
__device__ inline void fill_angles(A* table, const int32_t* positions, const float* freqs, int tokens, int n) {
    if (n == 0) return;
    int c = threadIdx.x / n, d = threadIdx.x - c * n;
    const int by_c = kPrepareThreads / n, by_d = kPrepareThreads - by_c * n;
    while (c * kSteps < tokens) {
        const int i0 = c * kSteps, m = min(kSteps, tokens - i0);
        const double f = freqs[d];
        const int first = positions[i0];
        bool follow = m > 1;
#pragma unroll
        for (int i = 1; i < kSteps; ++i) follow = follow && (i >= m || positions[i0 + i] == first + i);
        double2 s = sin_cos((double)first * f);
        put_angle(table + i0 * n + d, s);
        const double2 step = follow ? sin_cos(f) : make_double2(0.0, 1.0);
        for (int i = 1; i < m; ++i) {
            if (follow) s = make_double2(s.x * step.y + s.y * step.x, s.y * step.y - s.x * step.x);
            else s = sin_cos((double)positions[i0 + i] * f);
            put_angle(table + (i0 + i) * n + d, s);
        }
        c += by_c;
        d += by_d;
        if (d >= n) { d -= n; ++c; }
    }
}

// The tokens in front of place `at` of a page are coded again, four codes a word: whole words of a key; of a value's column those in front.
__device__ __noinline__ void code_again(int8_t* codes, bool keys, int at, float before, double s, double inv, int hd, int block, int lt, int threads) {
    if (keys) {
        for (int j = lt; j < at * (hd / 4); j += threads) {
            const int i = j / (hd / 4), d = (j - i * (hd / 4)) * 4;
            char4* const c = reinterpret_cast<char4*>(codes + ((d >> 4) * block + i) * 16 + (d & 15));
            const char4 x = *c;
            *c = make_char4((signed char)code_of(x.x * (double)before, s, inv), (signed char)code_of(x.y * (double)before, s, inv),
                            (signed char)code_of(x.z * (double)before, s, inv), (signed char)code_of(x.w * (double)before, s, inv));
        }
    } else {
        for (int j = lt; j < hd * ((at + 3) / 4); j += threads) {
            const int i = j / hd * 4, d = j % hd;
            signed char* const c = reinterpret_cast<signed char*>(codes + ((i >> 4) * hd + d) * 16 + (i & 15));
            char4 x = *reinterpret_cast<char4*>(c);
            x.x = (signed char)code_of(x.x * (double)before, s, inv);
            if (i + 1 < at) x.y = (signed char)code_of(x.y * (double)before, s, inv);
            if (i + 2 < at) x.z = (signed char)code_of(x.z * (double)before, s, inv);
            if (i + 3 < at) x.w = (signed char)code_of(x.w * (double)before, s, inv);
            *reinterpret_cast<char4*>(c) = x;
        }
    }
}

// A short run of one head by a warp: `in` is the run's first row, `codes` and `scale_at` the page's of that head.  The same numbers as the walks below make.
template <typename T>
__device__ inline void prepare_short(const T* in, size_t ld, bool keys, int turned, const float* freqs, const int32_t* positions, int n, int at, int hd, int block,
                                           int8_t* codes, float* scale_at) {
    const int lane = threadIdx.x & 31;
    const float before = at == 0 ? 0.0f : *scale_at;
    auto each = [&](auto f) {
        for (int i = 0; i < n; ++i, in += ld) {
            for (int d = lane; d < turned; d += 32) {
                Angle turn;
                turn.set(sin_cos((double)positions[i] * (double)freqs[d]));
                const float x = load_as_f32(in + d), y = load_as_f32(in + d + turned);
                f(i, d, turn.first(x, y));
                f(i, d + turned, turn.second(x, y));
            }
            for (int d = 2 * turned + lane; d < hd; d += 32) f(i, d, (double)load_as_f32(in + d));
        }
        in -= (size_t)n * ld;
    };
    double largest = 0.0;
    each([&](int, int, double v) { largest = fmax(largest, finite_size(v)); });
    const float scale = fmaxf(before, warp_max((float)(largest / 127.0)));
    const double s = scale, inv = scale > 0.0f ? 1.0 / s : 0.0;
    if (lane == 0) *scale_at = scale;  // (all have read it: warp_max is behind the load)
    if (scale > before && at > 0) code_again(codes, keys, at, before, s, inv, hd, block, lane, 32);
    __syncwarp();  // (a word that holds codes of both is written above first)
    each([&](int i, int d, double v) {
        const int j = at + i;
        codes[keys ? ((d >> 4) * block + j) * 16 + (d & 15) : ((j >> 4) * hd + d) * 16 + (j & 15)] = (int8_t)code_of(v, s, inv);
    });
}

// Blocks of threads along x: keys (groups of tokens x sets of heads), values (the same), query rows.  A run is a stretch of tokens with ascending
// slots in one page; the block whose tokens hold the first of a run takes all of it, so that a page's scale is known in one place.  A head has
// 256 / HS threads; the first walk over the run finds the largest magnitude, the second (out of L1 / L2) codes.  The angles of a token are computed
// once per block into shared memory, not for every head.  Keys are turned in 32 bits, and in 64 where that could make another code or another
// largest magnitude: their codes are those of the 64-bit values.  Codes leave as words: four entries of a key, the sixteen tokens of a value's column.
// Bound: loads and the arithmetic of codes and angles (2672 tokens of five prompts, 32 query heads over 8 of size 128, bf16: 38 us for 33 MB in and 27
// MB out); single tokens are latency (48 requests 5.4 us).
// V: entries that a thread loads together.
// HS: kv heads of a block of threads.
template <typename T, int V, int HS>
__global__ void __launch_bounds__(kPrepareThreads) prepare_paged_kernel(const PrepareArgs a) {
    extern __shared__ __align__(16) unsigned char prepare_smem[];  // [token][n_freqs] angles
    double2* const table = reinterpret_cast<double2*>(prepare_smem);
    Angle* const key_table = reinterpret_cast<Angle*>(prepare_smem);
    constexpr int kHeadThreads = kPrepareThreads / HS;
    __shared__ int s_slots[2 * 128 + 1];
    __shared__ int s_run;
    __shared__ uint32_t s_first[4], s_short[4];
    __shared__ float s_top[kPrepareThreads / 32];
    const int tid = threadIdx.x, hd = a.head_dim, half = a.n_freqs, limit = a.pages * a.block;
    const int kv_blocks = a.groups * a.head_sets;
    pdl_wait();
    if ((int)blockIdx.x >= 2 * kv_blocks) {
        // ---- query rows of q_tokens tokens: (head, V entries) over the threads, all tokens of a place in turn
        const int t0 = ((int)blockIdx.x - 2 * kv_blocks) * a.q_tokens, n = min(a.q_tokens, a.tokens - t0), Q = half / V, rest = (hd - 2 * half) / V;
        if (tid < n) s_slots[tid] = a.slots[t0 + tid];
        fill_angles<4>(table, a.positions + t0, a.freqs, n, half);
        __syncthreads();
        for (int i = tid; i < a.heads * (Q + rest); i += kPrepareThreads) {
            const int h = i / (Q + rest), d = (i - h * (Q + rest)) * V;
            const T* src = static_cast<const T*>(a.query) + (size_t)t0 * a.ldq + h * hd + d;
            T* dst = static_cast<T*>(a.query_rot) + ((size_t)t0 * a.heads + h) * hd + d;
#pragma unroll 4
            for (int t = 0; t < n; ++t, src += a.ldq, dst += (size_t)a.heads * hd) {
                if (s_slots[t] < 0 || s_slots[t] >= limit) continue;
                float u[V], v[V];
                if (d >= half) {  // (entries from 2 * n_freqs on)
                    load_some<V>(src + half, u);
                    store_some<V>(dst + half, u);
                    continue;
                }
                load_some<V>(src, u);
                load_some<V>(src + half, v);
                const double2* const turn = table + t * half + d;
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const double2 s = turn[e];
                    const double x = u[e], y = v[e];
                    u[e] = (float)(x * s.y - y * s.x);
                    v[e] = (float)(x * s.x + y * s.y);
                }
                store_some<V>(dst, u);
                store_some<V>(dst + half, v);
            }
        }
        return;
    }
    const bool keys = (int)blockIdx.x < kv_blocks;
    const int item = keys ? blockIdx.x : blockIdx.x - kv_blocks, set = item % a.head_sets, t0 = item / a.head_sets * a.group, t1 = min(a.tokens, t0 + a.group);
    const int sub = tid / kHeadThreads, lt = tid % kHeadThreads, h = set * HS + sub;
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
    const int block_log = 31 - __clz(a.block);
    if (tid < 128) {  // first tokens of runs, a bit each
        bool first = false, few = false;
        if (tid < t1 - t0) {
            const int slot = s_slots[tid + 1];
            first = slot >= 0 && slot < limit && ((slot & (a.block - 1)) == 0 || t0 + tid == 0 || s_slots[tid] != slot - 1);
            if constexpr (HS == 1) {
                const int n = min(a.block - (slot & (a.block - 1)), kPrepareShort + 1);
                few = first && n <= kPrepareShort;
                for (int i = 1; i < n; ++i) few = few || (first && s_slots[tid + 1 + i] != slot + i);
            }
        }
        const uint32_t bits = __ballot_sync(0xffffffffu, first && !few), few_bits = __ballot_sync(0xffffffffu, few);
        if ((tid & 31) == 0) {
            s_first[tid >> 5] = bits;
            s_short[tid >> 5] = few_bits;
        }
    }
    __syncthreads();
    if constexpr (HS == 1) {  // single tokens of many requests: a warp takes each
        int turn = 0;
        for (int word = 0; word < 4; ++word) {
            for (uint32_t bits = s_short[word]; bits != 0u; bits &= bits - 1u) {
                if (turn++ % (kPrepareThreads / 32) != tid >> 5) continue;
                const int t = t0 + word * 32 + __ffs(bits) - 1;
                const int* const slots = s_slots + (t - t0 + 1);
                const int slot = slots[0], at = slot & (a.block - 1), most = min(a.block - at, a.tokens - t);
                const size_t place = (size_t)(slot >> block_log) * a.kv_heads + h;
                int n = 1;
                while (n < most && slots[n] == slot + n) ++n;
                prepare_short(in + (size_t)t * ld, ld, keys, turned, a.freqs, a.positions + t, n, at, hd, a.block, (keys ? a.k_codes : a.v_codes) + place * a.block * hd,
                              (keys ? a.k_scales : a.v_scales) + place);
            }
        }
    }
    for (int word = 0; word < 4; ++word) {
        for (uint32_t bits = s_first[word]; bits != 0u; bits &= bits - 1u) {
            const int t = t0 + word * 32 + __ffs(bits) - 1;
            const int* const slots = s_slots + (t - t0 + 1);
            const int slot = slots[0], at = slot & (a.block - 1), page = slot >> block_log;
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
                fill_angles<16>(key_table, a.positions + t + i0, a.freqs, i1 - i0, turned);
                __syncthreads();
            };
            // calls f(token of the run, first entry, angles, the V pairs, the V turned pairs) for this thread's turned entries, and g(token, entry, V values) for the others
            auto walk = [&](bool again, auto f, auto g) {
                for (int i0 = 0; i0 < n && turned > 0; i0 += a.table_tokens) {
                    const int i1 = min(n, i0 + a.table_tokens), Q = turned / V;
                    if (!(again && kept)) angles(i0, i1);
                    if (!live) continue;
    #pragma unroll 2
                    for (int j = lt; j < (i1 - i0) * Q; j += kHeadThreads) {
                        const int i = j / Q, d = (j - i * Q) * V;
                        const T* const src = in + (size_t)(t + i0 + i) * ld + d;
                        float x[V], y[V], p[V], q[V];
                        load_some<V>(src, x);
                        load_some<V>(src + turned, y);
                        const Angle* const turn = key_table + i * turned + d;
    #pragma unroll
                        for (int e = 0; e < V; ++e) {
                            p[e] = fmaf(x[e], turn[e].cos, -(y[e] * turn[e].sin));
                            q[e] = fmaf(x[e], turn[e].sin, y[e] * turn[e].cos);
                        }
                        f(i0 + i, d, turn, x, y, p, q);
                    }
                }
                const int R = (hd - 2 * turned) / V;
                if (!live || R == 0) return;
    #pragma unroll 4
                for (int j = lt; j < n * R; j += kHeadThreads) {
                    const int i = j / R, d = 2 * turned + (j - i * R) * V;
                    float x[V];
                    load_some<V>(in + (size_t)(t + i) * ld + d, x);
                    g(i, d, x);
                }
            };
            using Some = const float (&)[V];
            // ---- the largest magnitude, in 32 bits; of the turned keys those that may be it once more in 64 (of few tokens all at once: a walk less)
            constexpr bool kAtOnce = HS > 1;
            double largest = 0.0;
            float largest32 = 0.0f;
            bool beyond = false;  // a pair whose 32-bit rotation overflows (its entries may be infinities themselves)
            walk(false, [&](int, int, const Angle* turn, Some x, Some y, Some p, Some q) {
    #pragma unroll
                for (int e = 0; e < V; ++e) {
                    if constexpr (kAtOnce) {
                        largest = fmax(largest, fmax(finite_size(turn[e].first(x[e], y[e])), finite_size(turn[e].second(x[e], y[e]))));
                        continue;
                    }
                    const float size = fmaxf(fabsf(p[e]), fabsf(q[e]));
                    beyond = beyond || !(fabsf(p[e]) < INFINITY) || !(fabsf(q[e]) < INFINITY);
                    if (size < INFINITY) largest32 = fmaxf(largest32, size);
                }
            }, [&](int, int, Some v) {
    #pragma unroll
                for (int e = 0; e < V; ++e) largest32 = fmaxf(largest32, fabsf(v[e]) < INFINITY ? fabsf(v[e]) : 0.0f);
            });
            if (kAtOnce || turned == 0) {
                largest = fmax(largest, (double)largest32);
            } else {
                const float own = largest32;
                const float mine = warp_max(own);
                if ((tid & 31) == 0) s_top[tid >> 5] = mine;
                const bool all = __syncthreads_or(beyond) != 0;
                float most = 0.0f;
    #pragma unroll
                for (int w = 0; w < kHeadThreads / 32; ++w) most = fmaxf(most, s_top[sub * (kHeadThreads / 32) + w]);
                const float near = all ? 0.0f : most * (1.0f - 0x1p-18f);
                // (few threads have such entries; one that has none of its own goes along where the angles are not all there)
                const bool mine_too = own >= near;
                if (!kept || __any_sync(0xffffffffu, mine_too)) walk(true, [&](int, int, const Angle* turn, Some x, Some y, Some p, Some q) {
                    if (!mine_too) return;
    #pragma unroll 1
                    for (int e = 0; e < V; ++e)
                        if (all || fmaxf(fabsf(p[e]), fabsf(q[e])) >= near) largest = fmax(largest, fmax(finite_size(turn[e].first(x[e], y[e])), finite_size(turn[e].second(x[e], y[e]))));
                }, [&](int, int, Some v) {
                    if (!mine_too) return;
    #pragma unroll
                    for (int e = 0; e < V; ++e) largest = fmax(largest, finite_size((double)v[e]));
                });
                __syncthreads();  // (s_top is written again)
            }
            const float mine = warp_max((float)(largest / 127.0));
            if ((tid & 31) == 0) s_top[tid >> 5] = mine;
            float* const scale_at = (keys ? a.k_scales : a.v_scales) + (size_t)page * a.kv_heads + (live ? h : 0);
            const float before = at == 0 || !live ? 0.0f : *scale_at;
            __syncthreads();  // (all have read the scale)
            float scale = before;
    #pragma unroll
            for (int w = 0; w < kHeadThreads / 32; ++w) scale = fmaxf(scale, s_top[sub * (kHeadThreads / 32) + w]);
            const double s = scale, inv = scale > 0.0f ? 1.0 / s : 0.0;
            const float inv32 = (float)inv;
            int8_t* const codes = (keys ? a.k_codes : a.v_codes) + ((size_t)page * a.kv_heads + (live ? h : 0)) * a.block * hd;
            if (live && lt == 0) *scale_at = scale;
            if (live && scale > before && at > 0) code_again(codes, keys, at, before, s, inv, hd, a.block, lt, kHeadThreads);
            __syncthreads();  // (a word that holds codes of both is written above first)
            if (keys) {
                auto put = [&](int i, int d, const int (&c)[V]) {
                    int8_t* const to = codes + ((d >> 4) * a.block + at + i) * 16 + (d & 15);
                    if constexpr (V == 4) *reinterpret_cast<char4*>(to) = make_char4((signed char)c[0], (signed char)c[1], (signed char)c[2], (signed char)c[3]);
                    else *to = (int8_t)c[0];
                };
                walk(true, [&](int i, int d, const Angle* turn, Some x, Some y, Some p, Some q) {
                    int c[2][V];
    #pragma unroll
                    for (int e = 0; e < V; ++e) {
                        c[0][e] = quick_code(p[e], inv32);
                        c[1][e] = quick_code(q[e], inv32);
                    }
    #pragma unroll
                    for (int e = 0; e < V; ++e) {
                        if (c[0][e] == -1000) c[0][e] = code_of(turn[e].first(x[e], y[e]), s, inv);
                        if (c[1][e] == -1000) c[1][e] = code_of(turn[e].second(x[e], y[e]), s, inv);
                    }
                    put(i, d, c[0]);
                    put(i, d + turned, c[1]);
                }, [&](int i, int d, Some v) {
                    int c[V];
    #pragma unroll
                    for (int e = 0; e < V; ++e) c[e] = code_of(v[e], s, inv, inv32);
                    put(i, d, c);
                });
            } else if (live) {
                // groups of 16 tokens of a column: one 16-byte store where the run has all of them
                const int g0 = at >> 4, g1 = (at + n - 1) >> 4;
                for (int j = lt; j < (g1 - g0 + 1) * hd; j += kHeadThreads) {
                    const int g = g0 + j / hd, d = j % hd, i0 = g * 16 - at;  // token of the run at the group's first place
                    int8_t* const to = codes + ((size_t)g * hd + d) * 16;
                    if (i0 >= 0 && i0 + 16 <= n) {
                        const T* src = in + (size_t)(t + i0) * ld + d;
                        float x[16];
    #pragma unroll
                        for (int e = 0; e < 16; ++e) x[e] = load_as_f32(src + (size_t)e * ld);
                        uint32_t w[4] = {0u, 0u, 0u, 0u};
    #pragma unroll
                        for (int e = 0; e < 16; ++e) w[e >> 2] |= (uint32_t)(code_of(x[e], s, inv, inv32) & 255) << (8 * (e & 3));
                        *reinterpret_cast<uint4*>(to) = make_uint4(w[0], w[1], w[2], w[3]);
                    } else {
                        for (int i = max(i0, 0); i < min(i0 + 16, n); ++i) to[i - i0] = (int8_t)code_of(load_as_f32(in + (size_t)(t + i) * ld + d), s, inv, inv32);
                    }
                }
            }
            __syncthreads();
        }
    }
}

// Rows of the cache as f32; slots outside of it leave their row as it is.  A block of threads has 16 entries of the list and one head: of keys a
// thread reads 16 bytes (16 entries of a token), of values the 16 tokens of a column, again only where the list moves on to another group of 16.
// Bound: the f32 rows it writes (2853 rows of 8 heads of 128: 10 us for 29 MB; 772 rows 4.4 us).
__global__ void __launch_bounds__(128) paged_cache_rows_kernel(const int8_t* k_codes, const float* k_scales, const int8_t* v_codes, const float* v_scales, int pages, int block,
                                                               int kv_heads, int head_dim, const int32_t* slots, int count, float* k, float* v) {
    __shared__ int s_slots[16];
    const int tid = threadIdx.x, r0 = blockIdx.x * 16, h = blockIdx.y, n = min(16, count - r0), row_len = kv_heads * head_dim, units = head_dim / 16, limit = pages * block;
    const int block_log = 31 - __clz(block);
    pdl_wait();
    if (tid < 16) s_slots[tid] = tid < n ? slots[r0 + tid] : -1;
    __syncthreads();
    const bool aligned = (reinterpret_cast<uintptr_t>(k) & 15u) == 0;
    for (int i = tid; i < 16 * units; i += 128) {
        const int r = i & 15, c = i >> 4, slot = s_slots[r];
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
    for (int d = tid; d < head_dim; d += 128) {
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
            v[(size_t)(r0 + r) * row_len + h * head_dim + d] = (float)(int8_t)(w >> (8 * (e & 3))) * s;
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
    cudaError_t e = allow_dynamic_smem(paged_plan_kernel, (3 * (size_t)requests + 2) * 4);
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
    cudaError_t e = allow_dynamic_smem(paged_release_kernel, 3 * (size_t)requests * 4);
    if (e == cudaSuccess)
        e = launch(paged_release_kernel, dim3(1), dim3(kPlanThreads), 3 * (size_t)requests * 4, as_stream(stream), true, context, ended, requests, block, block_table,
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
    KMLL_REQUIRE(heads == 0 || query_rot != query || ld_query == heads * head_dim || tokens <= 1, "prepare paged attention: rows that do not lie together cannot turn in place");
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
    // Few tokens: each may begin a run, 64 threads a head (64 requests of a token: 5.8 us, in groups of 16 8.4; a prompt of 64: 23 and 14).  More: a block takes
    // the runs of a group, short ones by warps.  Groups are short while blocks are few (600 tokens of as many requests: 21 us, in groups of a page of 64
    // 31) and pages from there on (2574 tokens of four prompts: 38 us, in groups of 16 43).
    constexpr int kFewTokens = 64, kSomeTokens = 1024;
    a.group = tokens <= kFewTokens ? 1 : tokens <= kSomeTokens ? min(block, 16) : block;
    a.groups = (tokens + a.group - 1) / a.group;
    const int head_set = tokens <= kFewTokens ? 4 : 1;  // (a page of tokens is work for 256 threads, single tokens are not)
    a.head_sets = (kv_heads + head_set - 1) / head_set;
    a.q_tokens = tokens <= 512 ? 1 : 8;
    const int per_token = n_freqs * (int)sizeof(double2);
    a.table_tokens = per_token > 0 ? min(block, 128 * 1024 / per_token) : block;
    const int key_tokens = min(tokens, a.table_tokens);
    static_assert(sizeof(Angle) == sizeof(double2), "either table");
    const size_t table_bytes = (size_t)per_token * max(key_tokens, a.q_tokens);
    const long long blocks = 2ll * a.groups * a.head_sets + (heads > 0 ? (tokens + a.q_tokens - 1) / a.q_tokens : 0);
    KMLL_REQUIRE(blocks <= INT_MAX, "prepare paged attention: too many rows");
    const uintptr_t bits = reinterpret_cast<uintptr_t>(query) | reinterpret_cast<uintptr_t>(query_rot) | reinterpret_cast<uintptr_t>(key) | reinterpret_cast<uintptr_t>(value);
    const bool fours = n_freqs % 4 == 0 && (ld_query | ld_key | ld_value) % 4 == 0 && bits % (is_f32 ? 16 : 8) == 0;
    auto go = [&](auto kern) {
        const cudaError_t e = allow_dynamic_smem(kern, table_bytes);
        return e != cudaSuccess ? e : launch(kern, dim3((unsigned)blocks), dim3(kPrepareThreads), table_bytes, as_stream(stream), true, a);
    };
    auto pick = [&](auto hs) {
        constexpr int HS = decltype(hs)::value;
        return is_f32 ? fours ? go(prepare_paged_kernel<float, 4, HS>) : go(prepare_paged_kernel<float, 1, HS>)
                      : fours ? go(prepare_paged_kernel<uint16_t, 4, HS>) : go(prepare_paged_kernel<uint16_t, 1, HS>);
    };
    const cudaError_t e = head_set == 4 ? pick(std::integral_constant<int, 4>()) : pick(std::integral_constant<int, 1>());
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
    const cudaError_t e = launch(paged_cache_rows_kernel, dim3((count + 15) / 16, kv_heads), dim3(128), 0, as_stream(stream), true, k_codes, k_scales, v_codes, v_scales, pages, block,
                                 kv_heads, head_dim, slots, count, k, v);
    if (e != cudaSuccess) return fail(KMLL_ERR_CUDA, "paged cache rows: %s", cudaGetErrorString(e));
    return check_launch("paged cache rows");
}
