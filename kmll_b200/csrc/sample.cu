// The next token of every row of logits: temperature, top-k, top-p and min-p, from one given random number per row.
//
// With the tokens in the order of their logits (the lower index first among equals) every filter keeps the first so many of them, so a set is told by
// its weight alone, and the choice itself is one more search of the same kind: the first token at which the weight so far reaches a
// target.  Nothing is sorted.  Weights exp((logit - largest) / temperature) are whole numbers of 2^-44: sums do not depend on an order, and
// what is lost is below 2^-45 of the largest weight per token.  One pass fills a histogram of the weights over 2048 bins of equal
// ratio; a search finds its bin there, collects the bin's tokens and ranks them (or splits the bin again while it holds too many).
// A cluster of blocks has one row: every block a share of the tokens, block 0 the sums.
#include <cooperative_groups.h>

#include <cfloat>

#include "internal.cuh"

namespace kmll {
namespace {
namespace cg = cooperative_groups;

constexpr int kSampleThreads = 1024;
constexpr int kBins = 2048;
constexpr int kList = 2048;          // tokens that are ranked at once
constexpr int kUnit = 44;            // weights are multiples of 2^-kUnit
constexpr double kBinsPerFactor2 = (double)kBins / (kUnit + 1.5);

struct SampleArgs {
    const void* logits;
    int f32, vocab;
    size_t ld;
    const double* u;
    const float* temperature;
    const int32_t* top_k;
    const float *top_p, *min_p;
    int32_t* tokens;
    float* logprobs;
};

struct SampleShared {
    uint32_t count[kBins], low[kBins], high[kBins];  // tokens; weight of the bin in two words
    uint32_t sub_count[kBins], sub_low[kBins], sub_high[kBins];
    unsigned long long before[kBins];                // block 0: weight in front of the bin
    uint32_t count_before[kBins];
    unsigned long long list[kList], sorted[kList];
    unsigned long long warp_sum[32];
    unsigned long long least_sum;                    // weight at or above the min-p border
    float top;
    // block 0: what a search has found
    int bin;
    uint32_t listed;
    unsigned long long base, low_key, high_key, found_key, found_sum;
};

// larger logits have larger keys; among equals the lower index has the larger one
__device__ inline unsigned long long token_key(float l, uint32_t index) {
    const uint32_t b = __float_as_uint(l + 0.0f);
    return ((unsigned long long)(b & 0x80000000u ? ~b : b | 0x80000000u) << 32) | (0xffffffffu - index);
}
__device__ inline float key_logit(unsigned long long key) {
    const uint32_t o = (uint32_t)(key >> 32);
    return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
__device__ inline uint32_t key_index(unsigned long long key) { return 0xffffffffu - (uint32_t)key; }

struct Weigher {
    double top, inv;  // largest logit, 1 / temperature
    __device__ double exponent(float l) const { return l == top ? 0.0 : ((double)l - top) * inv; }
    __device__ unsigned long long weight(double x) const { return (unsigned long long)rint(exp(x) * (double)(1ull << kUnit)); }
    __device__ int bin(double x) const { return (int)fmin(-x * (1.4426950408889634 * kBinsPerFactor2), (double)kBins); }  // kBins: weighs nothing
};
__device__ inline void add_weight(uint32_t* low, uint32_t* high, unsigned long long w) {
    const uint32_t lo = (uint32_t)w, old = atomicAdd(low, lo), more = (uint32_t)(w >> 32) + (old + lo < old ? 1u : 0u);
    if (more != 0u) atomicAdd(high, more);
}

template <typename T>
__device__ inline float logit_at(const T* row, int i);
template <>
__device__ inline float logit_at<float>(const float* row, int i) { return row[i]; }
template <>
__device__ inline float logit_at<uint16_t>(const uint16_t* row, int i) { return bf16_bits_to_f32(row[i]); }

// Sums in front of each of the kBins entries, from counts and two-word weights; all threads of block 0.
__device__ inline void scan_bins(SampleShared& s, const uint32_t* count, const uint32_t* low, const uint32_t* high) {
    static_assert(kBins == 2 * kSampleThreads, "two bins a thread");
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    unsigned long long w0 = ((unsigned long long)high[2 * tid] << 32) + low[2 * tid], w1 = ((unsigned long long)high[2 * tid + 1] << 32) + low[2 * tid + 1];
    uint32_t c0 = count[2 * tid], c1 = count[2 * tid + 1];
    unsigned long long w = w0 + w1;
    uint32_t c = c0 + c1;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long a = __shfl_up_sync(0xffffffffu, w, o);
        const uint32_t b = __shfl_up_sync(0xffffffffu, c, o);
        if (lane >= o) { w += a; c += b; }
    }
    __shared__ uint32_t warp_count[32];
    if (lane == 31) { s.warp_sum[warp] = w; warp_count[warp] = c; }
    __syncthreads();
    unsigned long long wb = 0;
    uint32_t cb = 0;
    for (int i = 0; i < warp; ++i) { wb += s.warp_sum[i]; cb += warp_count[i]; }
    s.before[2 * tid] = wb + w - w0 - w1;
    s.before[2 * tid + 1] = wb + w - w1;
    s.count_before[2 * tid] = cb + c - c0 - c1;
    s.count_before[2 * tid + 1] = cb + c - c1;
    __syncthreads();
}

// CL blocks per row.
template <typename T>
__global__ void __launch_bounds__(kSampleThreads, 1) sample_rows_kernel(const SampleArgs a) {
    extern __shared__ unsigned char sample_smem[];
    SampleShared& s = *reinterpret_cast<SampleShared*>(sample_smem);
    cg::cluster_group cluster = cg::this_cluster();
    const int blocks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int row = blockIdx.x / blocks;
    SampleShared& s0 = *cluster.map_shared_rank(&s, 0);
    pdl_wait();
    const T* const logits = static_cast<const T*>(a.logits) + (size_t)row * a.ld;
    const int share = (a.vocab + blocks - 1) / blocks, i0 = rank * share, i1 = min(a.vocab, i0 + share);
    // ---- the largest logit (NaN and -infinity are tokens that are never taken)
    float top = -INFINITY;
    for (int i = i0 + tid; i < i1; i += kSampleThreads) top = fmaxf(top, logit_at(logits, i));
    __shared__ float scratch[33];
    top = block_max(top, scratch);
    if (tid == 0) s.top = top;
    for (int i = tid; i < kBins; i += kSampleThreads) s.count[i] = s.low[i] = s.high[i] = 0u;
    if (tid == 0) s.least_sum = 0ull;
    cluster.sync();
    for (int b = 0; b < blocks; ++b) top = fmaxf(top, cluster.map_shared_rank(&s, b)->top);
    float temperature = a.temperature != nullptr ? a.temperature[row] : 1.0f;
    if (top == -INFINITY) {  // nothing to choose from
        if (rank == 0 && tid == 0) {
            a.tokens[row] = -1;
            if (a.logprobs != nullptr) a.logprobs[row] = -INFINITY;
        }
        cluster.sync();
        return;
    }
    const bool greedy = !(temperature > FLT_EPSILON);
    const Weigher weigh = {(double)top, greedy ? (double)INFINITY : 1.0 / (double)temperature};
    const float least_p = a.min_p != nullptr ? a.min_p[row] : 0.0f;
    const double least = least_p > 0.0f ? log((double)fminf(least_p, 1.0f)) : -INFINITY;
    // ---- weights into the bins
    unsigned long long least_sum = 0ull;
    for (int i = i0 + tid; i < i1; i += kSampleThreads) {
        const float l = logit_at(logits, i);
        if (!(l > -INFINITY)) continue;
        const double x = weigh.exponent(l);
        const int b = weigh.bin(x);
        if (b >= kBins) continue;
        const unsigned long long w = weigh.weight(x);
        atomicAdd(&s.count[b], 1u);
        add_weight(&s.low[b], &s.high[b], w);
        if (x >= least) least_sum += w;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) least_sum += __shfl_xor_sync(0xffffffffu, least_sum, o);
    if (lane == 0) atomicAdd(&s.least_sum, least_sum);
    cluster.sync();
    if (rank == 0) {
        for (int b = 1; b < blocks; ++b) {
            const SampleShared& o = *cluster.map_shared_rank(&s, b);
            for (int i = tid; i < kBins; i += kSampleThreads) {
                s.count[i] += o.count[i];
                const unsigned long long w = (((unsigned long long)s.high[i] << 32) | s.low[i]) + (((unsigned long long)o.high[i] << 32) + o.low[i]);
                s.low[i] = (uint32_t)w;
                s.high[i] = (uint32_t)(w >> 32);
            }
            if (tid == 0) s.least_sum += o.least_sum;
        }
        __syncthreads();
    }
    // ---- search: the first token, in order, at which the tokens (by_count) or the weight so far reach `target`
    auto search = [&](bool by_count, unsigned long long target) {
        if (rank == 0) {
            scan_bins(s, s.count, s.low, s.high);
            for (int b = tid; b < kBins; b += kSampleThreads) {
                const unsigned long long before = by_count ? s.count_before[b] : s.before[b];
                const unsigned long long after = before + (by_count ? s.count[b] : (((unsigned long long)s.high[b] << 32) | s.low[b]));
                if (before < target && after >= target) {
                    s.bin = b;
                    s.listed = s.count[b];
                    s.base = before;
                    s.found_sum = s.before[b];
                }
            }
            __syncthreads();
            // logits of the bin: the bin is monotone in the logit, so halving between keys finds both ends
            if (tid < 2) {
                const int b = s.bin;
                const uint32_t highest = (uint32_t)(token_key((float)weigh.top, 0) >> 32);
                uint32_t lo = 0x007fffffu, hi = highest;  // (below every finite logit; in bin 0)
                // tid 0: the lowest key with bin <= b; tid 1: the highest key with bin >= b
                while (hi - lo > 1) {
                    const uint32_t mid = lo + (hi - lo) / 2;
                    const float l = key_logit((unsigned long long)mid << 32);
                    const int at = weigh.bin(weigh.exponent(l));
                    if (tid == 0 ? at <= b : at < b) hi = mid;
                    else lo = mid;
                }
                if (tid == 0) s.low_key = (unsigned long long)hi << 32;
                else s.high_key = ((unsigned long long)(b == 0 ? highest : lo) << 32) | 0xffffffffull;
            }
        }
        cluster.sync();
        // split while there are too many to rank
        while (s0.listed > (uint32_t)kList) {
            const unsigned long long low_key = s0.low_key, high_key = s0.high_key;
            int shift = 0;
            while (((high_key - low_key) >> shift) >= (unsigned long long)kBins) ++shift;
            for (int i = tid; i < kBins; i += kSampleThreads) s.sub_count[i] = s.sub_low[i] = s.sub_high[i] = 0u;
            __syncthreads();
            for (int i = i0 + tid; i < i1; i += kSampleThreads) {
                const float l = logit_at(logits, i);
                if (!(l > -INFINITY)) continue;
                const unsigned long long key = token_key(l, (uint32_t)i);
                if (key < low_key || key > high_key) continue;
                const int b = (int)((high_key - key) >> shift);
                atomicAdd(&s.sub_count[b], 1u);
                add_weight(&s.sub_low[b], &s.sub_high[b], weigh.weight(weigh.exponent(l)));
            }
            cluster.sync();
            if (rank == 0) {
                for (int b = 1; b < blocks; ++b) {
                    const SampleShared& o = *cluster.map_shared_rank(&s, b);
                    for (int i = tid; i < kBins; i += kSampleThreads) {
                        s.sub_count[i] += o.sub_count[i];
                        const unsigned long long w = (((unsigned long long)s.sub_high[i] << 32) | s.sub_low[i]) + (((unsigned long long)o.sub_high[i] << 32) + o.sub_low[i]);
                        s.sub_low[i] = (uint32_t)w;
                        s.sub_high[i] = (uint32_t)(w >> 32);
                    }
                }
                __syncthreads();
                scan_bins(s, s.sub_count, s.sub_low, s.sub_high);
                const unsigned long long base = s.base, sum = s.found_sum;
                __syncthreads();
                for (int b = tid; b < kBins; b += kSampleThreads) {
                    const unsigned long long before = base + (by_count ? s.count_before[b] : s.before[b]);
                    const unsigned long long after = before + (by_count ? s.sub_count[b] : (((unsigned long long)s.sub_high[b] << 32) | s.sub_low[b]));
                    if (before < target && after >= target) {
                        s.listed = s.sub_count[b];
                        s.base = before;
                        s.found_sum = sum + s.before[b];
                        s.high_key = high_key - ((unsigned long long)b << shift);
                        const unsigned long long reach = ((unsigned long long)(b + 1) << shift) - 1;
                        s.low_key = reach > high_key - low_key ? low_key : high_key - reach;
                    }
                }
            }
            cluster.sync();
        }
        const uint32_t listed = s0.listed;
        const unsigned long long low_key = s0.low_key, high_key = s0.high_key;
        cluster.sync();
        if (rank == 0 && tid == 0) s.listed = 0u;
        cluster.sync();
        for (int i = i0 + tid; i < i1; i += kSampleThreads) {
            const float l = logit_at(logits, i);
            if (!(l > -INFINITY)) continue;
            const unsigned long long key = token_key(l, (uint32_t)i);
            if (key >= low_key && key <= high_key) {
                const uint32_t at = atomicAdd(&s0.listed, 1u);
                if (at < (uint32_t)kList) s0.list[at] = key;
            }
        }
        cluster.sync();
        if (rank == 0) {
            for (uint32_t i = tid; i < listed; i += kSampleThreads) {
                const unsigned long long key = s.list[i];
                uint32_t place = 0;
                for (uint32_t j = 0; j < listed; ++j) place += s.list[j] > key ? 1u : 0u;
                s.sorted[place] = key;
            }
            __syncthreads();
            if (warp == 0) {
                if (lane == 0) s.found_key = s.sorted[listed - 1];
                __syncwarp();
                unsigned long long sum = s.found_sum, reached = s.base;
                for (uint32_t j0 = 0; j0 < listed; j0 += 32) {
                    const uint32_t j = j0 + lane;
                    const unsigned long long key = j < listed ? s.sorted[j] : 0ull;
                    const unsigned long long w = j < listed ? weigh.weight(weigh.exponent(key_logit(key))) : 0ull;
                    unsigned long long ws = w;
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const unsigned long long v = __shfl_up_sync(0xffffffffu, ws, o);
                        if (lane >= o) ws += v;
                    }
                    const unsigned long long at = reached + (by_count ? (unsigned long long)(lane + 1) : ws);
                    const uint32_t hit = __ballot_sync(0xffffffffu, j < listed && at >= target);
                    if (hit != 0u) {
                        if (lane == __ffs(hit) - 1) {
                            s.found_key = key;
                            s.found_sum = sum + ws;
                        }
                        break;
                    }
                    const unsigned long long all = __shfl_sync(0xffffffffu, ws, 31);
                    sum += all;
                    reached += by_count ? 32ull : all;
                }
            }
            __syncthreads();
        }
        cluster.sync();
    };
    if (greedy) {  // the first of the largest
        search(true, 1ull);
        if (rank == 0 && tid == 0) {
            a.tokens[row] = (int32_t)key_index(s.found_key);
            if (a.logprobs != nullptr) a.logprobs[row] = 0.0f;
        }
        cluster.sync();
        return;
    }
    if (rank == 0) scan_bins(s, s.count, s.low, s.high);
    cluster.sync();
    const int k = a.top_k != nullptr ? a.top_k[row] : 0;
    const float top_p = a.top_p != nullptr ? a.top_p[row] : 1.0f;
    const unsigned long long whole = s0.before[kBins - 1] + (((unsigned long long)s0.high[kBins - 1] << 32) | s0.low[kBins - 1]);
    const unsigned long long tokens = s0.count_before[kBins - 1] + s0.count[kBins - 1], least_mass = s0.least_sum;
    cluster.sync();
    unsigned long long kept = whole;
    if (k > 0 && (unsigned long long)k < tokens) {
        search(true, (unsigned long long)k);
        kept = s0.found_sum;
        cluster.sync();
    }
    if (top_p < 1.0f) {
        const double want = ceil((double)fmaxf(top_p, 0.0f) * (double)kept);
        search(false, min(kept, max(1ull, (unsigned long long)want)));
        kept = s0.found_sum;
        cluster.sync();
    }
    kept = min(kept, least_mass);
    const double u = a.u[row], at = floor((u > 0.0 ? u : 0.0) * (double)kept);
    search(false, at >= (double)kept ? kept : (unsigned long long)at + 1ull);
    if (rank == 0 && tid == 0) {
        a.tokens[row] = (int32_t)key_index(s.found_key);
        if (a.logprobs != nullptr) a.logprobs[row] = (float)(weigh.exponent(key_logit(s.found_key)) - log((double)kept / (double)(1ull << kUnit)));
    }
    cluster.sync();
}

}  // namespace
}  // namespace kmll

using namespace kmll;

extern "C" int kmll_sample_rows(kmll_stream_t stream, const void* logits, int is_f32, int ld, int rows, int vocab, const double* u, const float* temperature,
                                const int32_t* top_k, const float* top_p, const float* min_p, int32_t* tokens, float* logprobs) {
    KMLL_REQUIRE(rows >= 0 && vocab > 0, "sample rows: %d rows of %d logits", rows, vocab);
    KMLL_REQUIRE(vocab <= 1 << 19, "sample rows: %d logits in a row, at most %d", vocab, 1 << 19);
    KMLL_REQUIRE(ld >= vocab, "sample rows: rows overlap");
    if (rows == 0) return KMLL_OK;
    KMLL_REQUIRE_PTR(logits);
    KMLL_REQUIRE_PTR(u);
    KMLL_REQUIRE_PTR(tokens);
    const SampleArgs a = {logits, is_f32, vocab, (size_t)ld, u, temperature, top_k, top_p, min_p, tokens, logprobs};
    const int cluster = rows <= 18 ? 8 : rows <= 37 ? 4 : rows <= 74 ? 2 : 1;
    auto go = [&](auto kern) {
        cudaError_t e = allow_all_dynamic_smem(kern);
        if (e != cudaSuccess) return e;
        return launch_cluster(kern, dim3((unsigned)rows * cluster), cluster, dim3(kSampleThreads), sizeof(SampleShared), as_stream(stream), true, a);
    };
    const cudaError_t e = is_f32 ? go(sample_rows_kernel<float>) : go(sample_rows_kernel<uint16_t>);
    if (e != cudaSuccess) return fail(KMLL_ERR_CUDA, "sample rows: %s", cudaGetErrorString(e));
    return check_launch("sample rows");
}
