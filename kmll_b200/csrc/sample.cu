// The next token of every row of logits: temperature, top-k, top-p and min-p, from one given random number per row.
//
// With the tokens in the order of their logits (the lower index first among equals) every filter keeps the first so many of them, so a set is told by
// its weight alone, and the choice itself is one more search of the same kind: the first token at which the weight so far reaches a
// target.  No row is sorted.  Weights exp((logit - largest) / temperature) are whole numbers of 2^-44: sums do not depend on an order, and
// what is lost is below 2^-45 of the largest weight per token.
//   1  the largest logit
//   2  a histogram over 4096 bins of equal ratio, the highest logits first: with top-k of the tokens (no weights are needed), otherwise of the weights
//   3  with top-k: the tokens of all bins up to the one in which the k-th lies are collected; one block ranks them by counting, sums their
//      weights, cuts and chooses at once.  Otherwise each border (top-p, then the choice; both at once where their bins hold few tokens) is a search: its
//      bin's tokens are collected and ranked; a bin of more than 1024 (flat rows, equal logits) is split until they are fewer.  A large k, or equals around the
//      k-th, is a search by count.
// A cluster of blocks has one row: every block a share of the tokens, block 0 the sums.
// Bound: latency of the steps for few rows; for many the weights of step 2 (64-bit exponentials and shared-memory atomics, one per token: half of the time
// of a row that has them) and instructions per token in the other passes, whose logits come out of L2.  Greedy, top-k 50, no filter, top-p 0.9 at
// temperature 0.8: a row of 32000 f32 logits 10, 12, 15 and 16 us; 16 of 151936 18, 19, 28 and 31; 64 of 152064 (39 MB, 6 us at the copy bandwidth)
// 25, 28, 43 and 47; flat rows with top-p, whose bins hold more than are ranked together, 86 (both borders one after another always: 51 and 84).
#include <cooperative_groups.h>

#include <atomic>
#include <cfloat>
#include <type_traits>

#include "internal.cuh"

namespace kmll {
namespace {
namespace cg = cooperative_groups;

constexpr int kSampleThreads = 1024;
constexpr int kBins = 4096, kSubBins = 1024;
constexpr int kList = 1024;          // tokens that are ranked at once
constexpr int kBoth = 700;           // tokens up to which two borders are ranked together: ranking costs their square, a search one pass over the row
constexpr int kUnit = 44;            // weights are multiples of 2^-kUnit
constexpr float kBinsPerFactor2 = (float)kBins / (kUnit + 1.5f);  // tokens behind the last bin weigh less than half a unit

struct SampleArgs {
    const void* logits;
    int vocab;
    size_t ld;
    const double* u;
    const float* temperature;
    const int32_t* top_k;
    const float *top_p, *min_p;
    int32_t* tokens;
    float* logprobs;
};

struct SampleBins {  // of a row, in its block 0: tokens and weight of a bin, and of all bins in front of it
    uint32_t *count, *count_before;
    unsigned long long *weight, *before;
};
struct SampleShared {
    uint32_t count[kBins], low[kBins], high[kBins];  // this block's: tokens; weight of the bin in two words
    // block 0, of the row
    uint32_t all_count[kBins], count_before[kBins];
    unsigned long long all_weight[kBins], before[kBins];
    uint32_t sub_count[kSubBins], sub_count_before[kSubBins];
    unsigned long long sub_weight[kSubBins], sub_before[kSubBins];
    unsigned long long list[kList], sorted[kList], sums[kList];
    double powers[256];                              // 2^(j / 256)
    unsigned long long warp_sum[32];
    uint32_t warp_count[32];
    unsigned long long least_sum;                    // weight at or above the min-p border
    unsigned long long key_range[2];                 // of a bin's tokens in this block
    float scratch[33], tops[8];                      // largest logit of every block of the cluster
    int bin, overflow, choice[2], many, both;        // many: more tokens than can be listed, by their weight; both: few enough for two borders
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

constexpr float kPlace0 = 8388608.0f;  // 2^23: adding it rounds to a whole number, and leaves it in the low bits
struct Weigher {
    float top, per_bin;  // largest logit; bins per unit of logit
    double inv, steps;   // 1 / temperature; steps of 2^(1 / 256) per unit of logit
    const double* powers;
    __device__ double exponent(float l) const { return l == top ? 0.0 : ((double)l - (double)top) * inv; }
    // Of a token that has a bin: 2^(y / 256) = 2^(j / 256) * 2^n * e^(c r) with 256 n + j the nearest whole number to y, c = ln 2 / 256: Taylor's series in
    // |c r| <= c / 2, whose first term left out is below 2^-54.  Adding 1.5 * 2^52 (2^52) rounds to a whole number and leaves it in the low bits:
    // conversions run at an eighth of the rate.
    __device__ unsigned long long weight(float l) const {
        constexpr double kC = 0.693147180559945309 / 256.0, kWhole = 6755399441055744.0;
        const double y = l == top ? 0.0 : ((double)l - (double)top) * steps, m = y + kWhole, r = y - (m - kWhole);
        const int i = __double2loint(m);
        double p = kC * kC * kC * kC / 24.0;
        p = fma(p, r, kC * kC * kC / 6.0);
        p = fma(p, r, kC * kC / 2.0);
        p = fma(p, r, kC);
        p = fma(p, r, 1.0);
        const double e = p * powers[i & 255];
        const double w = __hiloint2double(__double2hiint(e) + (kUnit + (i >> 8)) * (1 << 20), __double2loint(e));
        return (unsigned long long)__double_as_longlong(w + 4503599627370496.0) & 0xfffffffffffffull;
    }
    // kPlace0 + its bin, monotone in the logit; beyond the last bin (and for -infinity), or NaN (of NaN): weighs nothing
    __device__ float place(float l) const { return (l == top ? 0.0f : (top - l) * per_bin) + kPlace0; }
};
__device__ inline bool has_bin(float place) { return place <= kPlace0 + (float)(kBins - 1); }
__device__ inline int bin_at(float place) { return (int)(__float_as_uint(place) - 0x4b000000u); }
__device__ inline void add_weight(uint32_t* low, uint32_t* high, unsigned long long w) {
    const uint32_t lo = (uint32_t)w, old = atomicAdd(low, lo), more = (uint32_t)(w >> 32) + (old + lo < old ? 1u : 0u);
    if (more != 0u) atomicAdd(high, more);
}

// Calls f(index of the first, logits) for the 16-byte pieces of the block's share of a row; what is not the row's is -infinity.
template <typename T, typename F>
__device__ inline void each_logit(const T* row, int vocab, int rank, int blocks, F f) {
    constexpr int N = 16 / (int)sizeof(T);
    const int shift = (int)((reinterpret_cast<uintptr_t>(row) & 15u) / sizeof(T)), pieces = (vocab + shift + N - 1) / N, share = (pieces + blocks - 1) / blocks;
    const int end = min(pieces, (rank + 1) * share);
#pragma unroll 1
    for (int c = rank * share + (int)threadIdx.x; c < end; c += kSampleThreads) {
        const int i0 = c * N - shift;
        float x[N];
        if (i0 >= 0 && i0 + N <= vocab) {
            const uint4 u = __ldg(reinterpret_cast<const uint4*>(row + i0));
            const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int e = 0; e < N; ++e) x[e] = __uint_as_float(sizeof(T) == 4 ? w[e & 3] : e & 1 ? w[e >> 1 & 3] & 0xffff0000u : w[e >> 1 & 3] << 16);
        } else {
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const int i = i0 + e;
                x[e] = i < 0 || i >= vocab ? -INFINITY : sizeof(T) == 4 ? reinterpret_cast<const float*>(row)[i] : __uint_as_float((uint32_t)reinterpret_cast<const uint16_t*>(row)[i] << 16);
            }
        }
        f(i0, x);
    }
}

// Sums in front of each entry; all threads of block 0.
template <int N>
__device__ inline void scan_bins(SampleShared& s, const SampleBins& b) {
    constexpr int E = N / kSampleThreads;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    unsigned long long w = 0;
    uint32_t c = 0;
#pragma unroll
    for (int i = 0; i < E; ++i) { w += b.weight[E * tid + i]; c += b.count[E * tid + i]; }
    const unsigned long long own_w = w;
    const uint32_t own_c = c;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long x = __shfl_up_sync(0xffffffffu, w, o);
        const uint32_t y = __shfl_up_sync(0xffffffffu, c, o);
        if (lane >= o) { w += x; c += y; }
    }
    if (lane == 31) { s.warp_sum[warp] = w; s.warp_count[warp] = c; }
    __syncthreads();
    w -= own_w;
    c -= own_c;
    for (int i = 0; i < warp; ++i) { w += s.warp_sum[i]; c += s.warp_count[i]; }
#pragma unroll
    for (int i = 0; i < E; ++i) {
        b.before[E * tid + i] = w;
        b.count_before[E * tid + i] = c;
        w += b.weight[E * tid + i];
        c += b.count[E * tid + i];
    }
    __syncthreads();
}

// The listed tokens in order (s.sorted), with the weight up to and with each (s.sums, counted from `sum`); all threads of block 0.
__device__ inline void rank_list(SampleShared& s, const Weigher& weigh, uint32_t listed, unsigned long long sum) {
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    static_assert(kList == kSampleThreads, "a token a thread");
    if (tid < listed) {
        const unsigned long long key = s.list[tid];
        uint32_t place = 0;
#pragma unroll 8
        for (uint32_t j = 0; j < listed; ++j) place += s.list[j] > key ? 1u : 0u;
        s.sorted[place] = key;
    }
    __syncthreads();
    unsigned long long w = tid < listed ? weigh.weight(key_logit(s.sorted[tid])) : 0ull;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long v = __shfl_up_sync(0xffffffffu, w, o);
        if (lane >= o) w += v;
    }
    if (lane == 31) s.warp_sum[warp] = w;
    __syncthreads();
    for (uint32_t i = 0; i < warp; ++i) sum += s.warp_sum[i];
    s.sums[tid] = sum + w;
    __syncthreads();
}
// Number of the first ranked token at which the weight so far reaches `target` (the last one where none does); all threads of block 0 get it.
__device__ inline uint32_t reach(SampleShared& s, uint32_t listed, unsigned long long target) {
    if (threadIdx.x == 0) s.bin = (int)listed - 1;
    __syncthreads();
    const uint32_t i = threadIdx.x;
    if (i < listed && s.sums[i] >= target && (i == 0 || s.sums[i - 1] < target)) s.bin = (int)i;
    __syncthreads();
    const uint32_t at = (uint32_t)s.bin;
    __syncthreads();
    return at;
}

template <typename T>
__global__ void __launch_bounds__(kSampleThreads, 1) sample_rows_kernel(const SampleArgs a) {
    extern __shared__ __align__(16) unsigned char sample_smem[];
    SampleShared& s = *reinterpret_cast<SampleShared*>(sample_smem);
    cg::cluster_group cluster = cg::this_cluster();
    const int blocks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), tid = threadIdx.x, lane = tid & 31;
    const int row = blockIdx.x / blocks;
    SampleShared& s0 = *cluster.map_shared_rank(&s, 0);
    for (int i = tid; i < kBins; i += kSampleThreads) {
        s.count[i] = s.low[i] = s.high[i] = s.all_count[i] = 0u;
        s.all_weight[i] = 0ull;
    }
    const SampleBins bins = {s.all_count, s.count_before, s.all_weight, s.before}, subs = {s.sub_count, s.sub_count_before, s.sub_weight, s.sub_before};
    if (tid < 256) s.powers[tid] = exp2((double)tid / 256.0);
    if (tid == 0) {
        s.least_sum = 0ull;
        s.listed = 0u;
        s.overflow = 0;
    }
    asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");  // this block runs: the others may write to its shared memory
    pdl_wait();
    const T* const logits = static_cast<const T*>(a.logits) + (size_t)row * a.ld;
    auto each = [&](auto f) {
        each_logit(logits, a.vocab, rank, blocks, [&](int i0, const auto& x) {
#pragma unroll
            for (int e = 0; e < (int)(sizeof(x) / 4); ++e) f(i0 + e, x[e]);
        });
    };
    const float temperature = a.temperature != nullptr ? a.temperature[row] : 1.0f, least_p = a.min_p != nullptr ? a.min_p[row] : 0.0f;
    const float top_p = a.top_p != nullptr ? a.top_p[row] : 1.0f;
    const int k = a.top_k != nullptr ? a.top_k[row] : 0;
    const double u = a.u[row];
    // ---- the largest logit (NaN and -infinity are tokens that are never taken)
    float top = -INFINITY;
    each([&](int, float l) { top = fmaxf(top, l); });
    top = block_max(top, s.scratch);
    asm volatile("barrier.cluster.wait;" ::: "memory");  // every block of the cluster has started
    if (tid < blocks) cluster.map_shared_rank(&s, tid)->tops[rank] = top;
    cluster.sync();
    for (int b = 0; b < blocks; ++b) top = fmaxf(top, s.tops[b]);
    top += 0.0f;  // (-0 is 0)
    if (top == -INFINITY) {  // nothing to choose from
        if (rank == 0 && tid == 0) {
            a.tokens[row] = -1;
            if (a.logprobs != nullptr) a.logprobs[row] = -INFINITY;
        }
        cluster.sync();
        return;
    }
    const bool greedy = !(temperature > FLT_EPSILON);
    const Weigher weigh = {top, greedy ? INFINITY : kBinsPerFactor2 * 1.442695041f / temperature, greedy ? (double)INFINITY : 1.0 / (double)temperature,
                           greedy ? (double)INFINITY : 256.0 / 0.693147180559945309 / (double)temperature, s.powers};
    const double least = least_p > 0.0f ? log((double)fminf(least_p, 1.0f)) : -INFINITY;
    const bool k_on = k > 0 && k < a.vocab, by_k = greedy || (k_on && k <= kList), large_k = !greedy && k_on && k > kList;
    const int want_k = greedy ? 1 : k;
    // the smallest logit that min-p leaves: next to where the logarithm says, by the comparison that defines it
    float least_logit = -INFINITY;
    if (least > -INFINITY && !greedy) {
        least_logit = (float)((double)top + least * (double)temperature);
        for (int i = 0; i < 4 && weigh.exponent(least_logit) >= least; ++i) least_logit = nextafterf(least_logit, -INFINITY);
        for (int i = 0; i < 8 && !(weigh.exponent(least_logit) >= least); ++i) least_logit = nextafterf(least_logit, INFINITY);
    }

    // this block's bins into those of the row, and back to zero
    auto merge = [&](uint32_t* counts, unsigned long long* weights, int n) {
        __syncthreads();
        for (int i = tid; i < n; i += kSampleThreads) {
            const uint32_t c = s.count[i];
            const unsigned long long w = ((unsigned long long)s.high[i] << 32) | s.low[i];
            if (c != 0u) atomicAdd(&counts[i], c);
            if (w != 0ull) atomicAdd(&weights[i], w);
            s.count[i] = s.low[i] = s.high[i] = 0u;
        }
        cluster.sync();
    };
    // tokens that `take` names into the list of block 0 (which is empty); few pieces have any
    auto collect = [&](auto take) {
        each_logit(logits, a.vocab, rank, blocks, [&](int i0, const auto& x) {
            bool any = false;
#pragma unroll
            for (int e = 0; e < (int)(sizeof(x) / 4); ++e) any |= take(i0 + e, x[e]);
            if (!any) return;
#pragma unroll
            for (int e = 0; e < (int)(sizeof(x) / 4); ++e) {
                if (!take(i0 + e, x[e])) continue;
                const uint32_t at = atomicAdd(&s0.listed, 1u);
                if (at < (uint32_t)kList) s0.list[at] = token_key(x[e], (uint32_t)(i0 + e));
                else s0.overflow = 1;
            }
        });
        cluster.sync();
    };
    // weight at or above the min-p border, and weights into the bins
    auto weigh_all = [&](bool counts) {
        unsigned long long least_sum = 0ull;
        each([&](int, float l) {
            const float place = weigh.place(l);
            if (!has_bin(place)) return;
            const int b = bin_at(place);
            const unsigned long long w = weigh.weight(l);
            if (counts) atomicAdd(&s.count[b], 1u);
            add_weight(&s.low[b], &s.high[b], w);
            if (l >= least_logit) least_sum += w;
        });
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) least_sum += __shfl_xor_sync(0xffffffffu, least_sum, o);
        if (lane == 0 && least_sum != 0ull) atomicAdd(&s0.least_sum, least_sum);
        merge(s0.all_count, s0.all_weight, kBins);
    };
    auto target_of_u = [&](unsigned long long kept) {
        const double at = floor((u > 0.0 ? u : 0.0) * (double)kept);
        return at >= (double)kept ? kept : (unsigned long long)at + 1ull;
    };
    auto target_of_p = [&](unsigned long long whole) {
        const double want = ceil((double)fmaxf(top_p, 0.0f) * (double)whole);
        return min(whole, max(1ull, (unsigned long long)want));
    };
    auto answer = [&](unsigned long long key, unsigned long long kept) {
        if (tid == 0) {
            a.tokens[row] = (int32_t)key_index(key);
            if (a.logprobs != nullptr) a.logprobs[row] = greedy ? 0.0f : (float)(weigh.exponent(key_logit(key)) - log((double)kept / (double)(1ull << kUnit)));
        }
    };

    if (by_k) {
        each([&](int, float l) {
            const float place = weigh.place(l);
            if (has_bin(place)) atomicAdd(&s.count[bin_at(place)], 1u);
        });
        merge(s0.all_count, s0.all_weight, kBins);
        if (rank == 0) {
            scan_bins<kBins>(s, bins);
            const uint32_t tokens = s.count_before[kBins - 1] + s.all_count[kBins - 1], target = min((uint32_t)want_k, tokens);
            for (int b = tid; b < kBins; b += kSampleThreads)
                if (s.count_before[b] < target && s.count_before[b] + s.all_count[b] >= target) s.bin = b;
        }
        cluster.sync();
        const float last = kPlace0 + (float)s0.bin;
        collect([&](int, float l) { return weigh.place(l) <= last; });
        if (s0.overflow == 0) {
            if (rank == 0) {
                const uint32_t listed = s.listed, n = min(listed, (uint32_t)want_k);
                rank_list(s, weigh, listed, 0ull);
                unsigned long long kept = s.sums[n - 1];
                if (top_p < 1.0f) kept = s.sums[reach(s, n, target_of_p(kept))];
                if (least > -INFINITY) {
                    const int heavy = __syncthreads_count((uint32_t)tid < n && weigh.exponent(key_logit(s.sorted[tid])) >= least);
                    kept = min(kept, s.sums[heavy - 1]);
                }
                answer(s.sorted[reach(s, n, target_of_u(kept))], kept);
            }
            cluster.sync();
            return;
        }
        cluster.sync();
    }
    if (!greedy) weigh_all(large_k);
    // Tokens that weigh so much around bin b, within a hundredth: those of a bin differ by no more.
    auto tokens_of = [&](unsigned long long weight, int b) { return (float)weight * exp2f((float)b / kBinsPerFactor2 - (float)kUnit); };
    // The first token, in order, at which the tokens (by_count) or the weight so far reach `target` (block 0's): block 0 gets its key (found_key), and the
    // weight up to and with it (found_sum).  The bins' sums are there.
    auto search = [&](bool by_count, unsigned long long target) {
        if (rank == 0) {
            __syncthreads();  // (all have read what the search before found)
            for (int b = tid; b < kBins; b += kSampleThreads) {
                const unsigned long long before = by_count ? s.count_before[b] : s.before[b], after = before + (by_count ? s.all_count[b] : s.all_weight[b]);
                if (before < target && after >= target) {
                    s.bin = b;
                    s.base = before;
                    s.found_sum = s.before[b];
                    s.many = by_count ? s.all_count[b] > (uint32_t)kList : tokens_of(s.all_weight[b], b) > (float)kList;
                }
            }
            if (tid == 0) { s.listed = 0u; s.overflow = 0; }
        }
        if (tid == 0) { s.key_range[0] = ~0ull; s.key_range[1] = 0ull; }
        cluster.sync();
        const float bin = kPlace0 + (float)s0.bin;
        const bool many = s0.many != 0;
        if (!many) collect([&](int, float l) { return weigh.place(l) == bin; });
        if (many || s0.overflow != 0) {
            unsigned long long low_key = ~0ull, high_key = 0ull;
            each([&](int i, float l) {
                if (weigh.place(l) != bin) return;
                const unsigned long long key = token_key(l, (uint32_t)i);
                low_key = min(low_key, key);
                high_key = max(high_key, key);
            });
            if (high_key != 0ull) {
                atomicMin(&s.key_range[0], low_key);
                atomicMax(&s.key_range[1], high_key);
            }
            cluster.sync();
            low_key = ~0ull;
            high_key = 0ull;
            for (int b = 0; b < blocks; ++b) {
                const SampleShared& o = *cluster.map_shared_rank(&s, b);
                low_key = min(low_key, o.key_range[0]);
                high_key = max(high_key, o.key_range[1]);
            }
            // split: every round leaves one of kSubBins parts of the range, one key at the last
            bool more = true;
            while (more) {
                int shift = 0;
                while (((high_key - low_key) >> shift) >= (unsigned long long)kSubBins) ++shift;
                if (rank == 0)
                    for (int i = tid; i < kSubBins; i += kSampleThreads) { s.sub_count[i] = 0u; s.sub_weight[i] = 0ull; }
                cluster.sync();
                each([&](int i, float l) {
                    if (!(l > -INFINITY)) return;
                    const unsigned long long key = token_key(l, (uint32_t)i);
                    if (key < low_key || key > high_key) return;
                    const int b = (int)((high_key - key) >> shift);
                    atomicAdd(&s.count[b], 1u);
                    add_weight(&s.low[b], &s.high[b], weigh.weight(l));
                });
                merge(s0.sub_count, s0.sub_weight, kSubBins);
                if (rank == 0) {
                    scan_bins<kSubBins>(s, subs);
                    const unsigned long long base = s.base, sum = s.found_sum;
                    __syncthreads();
                    const unsigned long long before = base + (by_count ? s.sub_count_before[tid] : s.sub_before[tid]);
                    const unsigned long long after = before + (by_count ? s.sub_count[tid] : s.sub_weight[tid]);
                    if (before < target && after >= target) {
                        s.listed = s.sub_count[tid];
                        s.base = before;
                        s.found_sum = sum + s.sub_before[tid];
                        s.high_key = high_key - ((unsigned long long)tid << shift);
                        const unsigned long long far = ((unsigned long long)(tid + 1) << shift) - 1;
                        s.low_key = far > high_key - low_key ? low_key : high_key - far;
                    }
                }
                cluster.sync();
                more = s0.listed > (uint32_t)kList;
                low_key = s0.low_key;
                high_key = s0.high_key;
                cluster.sync();
            }
            if (rank == 0 && tid == 0) { s.listed = 0u; s.overflow = 0; }
            cluster.sync();
            collect([&](int i, float l) {
                const unsigned long long key = token_key(l, (uint32_t)i);
                return l > -INFINITY && key >= low_key && key <= high_key;
            });
        }
        if (rank == 0) {
            const uint32_t listed = s.listed;
            const unsigned long long base = s.base;
            rank_list(s, weigh, listed, s.found_sum);
            const uint32_t at = by_count ? min((uint32_t)(target - base), listed) - 1u : reach(s, listed, target);
            if (tid == 0) {
                s.found_key = s.sorted[at];
                s.found_sum = s.sums[at];
            }
            __syncthreads();
        }
    };
    if (rank == 0) scan_bins<kBins>(s, bins);
    if (greedy) {  // the first of the largest
        search(true, 1ull);
        if (rank == 0) answer(s.found_key, 1ull);
        cluster.sync();  // (block 0's shared memory stays while others read it)
        return;
    }
    unsigned long long kept = 0ull;  // (block 0's)
    if (rank == 0) kept = s.before[kBins - 1] + s.all_weight[kBins - 1];
    if (top_p < 1.0f && !k_on) {
        // Both borders at once: what top-p keeps ends within its bin, so the choice lies in one of few bins in front of it (one, as a rule).
        unsigned long long target = 0ull;
        if (rank == 0) {
            auto find = [&](unsigned long long t, int& to) {
                for (int b = tid; b < kBins; b += kSampleThreads)
                    if (s.before[b] < t && s.before[b] + s.all_weight[b] >= t) to = b;
            };
            target = target_of_p(kept);
            find(target, s.bin);
            if (tid == 0) { s.listed = 0u; s.overflow = 0; }
            __syncthreads();
            const unsigned long long before = s.before[s.bin];
            find(target_of_u(min(before + 1ull, s.least_sum)), s.choice[0]);
            find(target_of_u(min(before + s.all_weight[s.bin], s.least_sum)), s.choice[1]);
            __syncthreads();
            if (tid == 0) {
                const int c0 = s.choice[0], c1 = s.choice[1];
                const unsigned long long in_front = c1 < s.bin ? s.before[c1] + s.all_weight[c1] : before;  // up to the choice's last bin
                s.both = tokens_of(s.all_weight[s.bin], s.bin) + tokens_of(in_front - s.before[c0], c1) <= (float)kBoth;
            }
        }
        cluster.sync();
        if (s0.both != 0) {
            const float border = kPlace0 + (float)s0.bin, from = kPlace0 + (float)s0.choice[0], to = kPlace0 + (float)s0.choice[1];
            collect([&](int, float l) {
                const float place = weigh.place(l);
                return place == border || (place >= from && place <= to);
            });
            if (s0.overflow == 0) {
                if (rank == 0) {
                    const uint32_t listed = s.listed;
                    const unsigned long long before = s.before[s.bin], before_choice = s.before[s.choice[0]];
                    rank_list(s, weigh, listed, 0ull);
                    const uint32_t first = (uint32_t)__syncthreads_count((uint32_t)tid < listed && weigh.place(key_logit(s.sorted[tid])) < border);
                    const unsigned long long own = s.sums[tid], of_first = first > 0u ? s.sums[first - 1u] : 0ull;
                    __syncthreads();
                    s.sums[tid] = (uint32_t)tid < first ? before_choice + own : before + (own - of_first);
                    __syncthreads();
                    kept = min(s.sums[reach(s, listed, target)], s.least_sum);
                    answer(s.sorted[reach(s, listed, target_of_u(kept))], kept);
                }
                cluster.sync();
                return;
            }
            cluster.sync();
        }
    }
    if (k_on) {
        search(true, min((unsigned long long)k, (unsigned long long)s.count_before[kBins - 1] + s.all_count[kBins - 1]));
        kept = s.found_sum;
    }
    if (top_p < 1.0f) {
        search(false, target_of_p(kept));
        kept = s.found_sum;
    }
    if (rank == 0) kept = min(kept, s.least_sum);
    search(false, target_of_u(kept));
    if (rank == 0) answer(s.found_key, kept);
    cluster.sync();
}

// Clusters of `c` blocks that the current GPU runs at once: asked for once per kernel, GPU and size (an occupancy query, no allocation).
constexpr int kKnownDevices = 64;
template <auto kernel>
cudaError_t clusters_at_once(int device, int c, int& n) {
    static std::atomic<int> known[kKnownDevices][9];
    n = device < kKnownDevices ? known[device][c].load(std::memory_order_relaxed) : 0;
    if (n == 0) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(c * 16);
        cfg.blockDim = dim3(kSampleThreads);
        cfg.dynamicSmemBytes = sizeof(SampleShared);
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = c;
        attr[0].val.clusterDim.y = 1;
        attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        const cudaError_t e = cudaOccupancyMaxActiveClusters(&n, kernel, &cfg);
        if (e != cudaSuccess) return e;
        n = n < 1 ? 1 : n;
        if (device < kKnownDevices) known[device][c].store(n, std::memory_order_relaxed);
    }
    return cudaSuccess;
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
    KMLL_REQUIRE(reinterpret_cast<uintptr_t>(logits) % (is_f32 ? 4 : 2) == 0, "sample rows: logits are not aligned to their type");
    const SampleArgs a = {logits, vocab, (size_t)ld, u, temperature, top_k, top_p, min_p, tokens, logprobs};
    // The most blocks per row that still let all rows run at once: a row's steps are short, a second round of clusters costs as much as the first
    // (16 rows of 151936, greedy: clusters of 8, of which fewer than 16 fit, 29 us, of 4 19, of 2 29; 64 rows of 152064: of 4 41, of 2 30, of 1 51).
    auto go = [&](auto which) {
        constexpr auto kern = decltype(which)::value;
        int cluster = 1, device = 0, at_once = 0;
        cudaError_t e = allow_all_dynamic_smem(kern);
        if (e == cudaSuccess) e = cudaGetDevice(&device);
        for (int c = 8; c > 1 && cluster == 1 && e == cudaSuccess; c >>= 1) {
            if (rows > 148 / c) continue;
            e = clusters_at_once<kern>(device, c, at_once);
            if (rows <= at_once) cluster = c;
        }
        if (e != cudaSuccess) return e;
        return launch_cluster(kern, dim3((unsigned)rows * cluster), cluster, dim3(kSampleThreads), sizeof(SampleShared), as_stream(stream), true, a);
    };
    const cudaError_t e = is_f32 ? go(std::integral_constant<void (*)(SampleArgs), sample_rows_kernel<float>>()) : go(std::integral_constant<void (*)(SampleArgs), sample_rows_kernel<uint16_t>>());
    if (e != cudaSuccess) return fail(KMLL_ERR_CUDA, "sample rows: %s", cudaGetErrorString(e));
    return check_launch("sample rows");
}
