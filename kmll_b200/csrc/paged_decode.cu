// Attention of single tokens (and of a few rows) over the paged 8-bit cache: the codes go to the tensor cores as they lie.
//
//   S^T[key][row] = K[key] . q[row]: A = 16 keys x 32 codes by ldmatrix, B = q as a 24-bit integer below the largest
//   entry of its row, in bytes; mma.m16n8k32 s8 x u8 / s8 -> s32, one MMA per byte, exact; S = k_scale * q_scale * (D0 + 2^8 D1 + 2^16 D2)
//   O^T[dim][row] += V^T[dim][key] P^T[key][row]: A = 16 columns x 32 keys (values lie with the keys of a column together), B =
//   softmax weights times the page's value scale, as 24-bit (bf16 rows: 16-bit) fractions of the largest of them in the tile of 32 keys, in bytes
// Nothing is converted on the way from memory to the tensor cores, and both contractions are exact.  What is rounded:
//   q, to 2^-24 of its row's largest entry (of bf16 rows too: 16 bits below a strong channel leave the other entries fewer than the eight they have;
//   64 requests of 100 to 8000 tokens 75.5 us, with 16 bits 74.2);
//   the weights, to 2^-25 (bf16 rows 2^-17) of the largest of the tile.  Not of the row's largest: the sum of the weights has all of them, and what lies far below one
//   key that dominates a row is most of the result where that key's value is small.  For the same reason a tile with weights below 2^-14 (2^-10) of its
//   largest goes twice, the second time with 16 bits of what rounding left (64 requests of 8192, 32 query heads over 8 of size 128, f32: 183 us where scores
//   spread by 1, 201 where they spread by 3 and many tiles go twice; 185 without a second time).
// (f32 rows cost three MMAs where bf16 heads and remainders would cost two of twice the size, behind a conversion of every code.)
//
// A warp is a pipeline of its own over tiles of 32 keys (two stages of keys and values, cp.async in 16-byte groups), with its own running
// maximum and sum; four warps take the tiles of a stretch in turn and meet at its end.  The work of a call is one axis, requests x kv heads x
// tiles, cut into equal shares for the blocks, whatever the contexts; where a share ends within a head, the blocks that have parts of it leave
// maximum, sum and O in the workspace and the last to arrive joins them in the order of the blocks: results do not change from call to call.
// Bound: HBM (2 * head_dim bytes per key and kv head): 64 requests of 8192 tokens, 32 query heads over 8 of size 128, 184 us for 1074 MB, 5.8
// TB/s with f32 or bf16 rows (in a graph, one call behind the other); 64 of 100 to 8000 tokens 75 us for 369 MB, 10 us of which are fixed (share, queries, first
// tiles, join).  Few short requests are that latency alone: one of 2048 tokens 10.6 us.  Sixteen rows (16 query heads over one): 64 of 8192, 134 MB, 58 us.
#include <climits>
#include <type_traits>

#include "internal.cuh"
#include "mma_bf16.cuh"
#include "paged.cuh"

namespace kmll {
namespace {

constexpr int kPdWarps = 4;
constexpr int kPdThreads = kPdWarps * 32;
constexpr int kPdKeys = 32;      // keys of a tile
constexpr int kPdBlocks = 444;   // three blocks on each of 148 multiprocessors (sixteen rows: two)
constexpr int kPdStages = 2;
// What a stretch costs besides its tiles (queries, first copies, the warps' meeting), in tiles: so much longer is a head on the axis of work, or
// blocks whose share is many short requests would end last (64 requests of 100 to 8000 tokens, 32 / 8 heads of 128: 0 tiles 96 us,
// 4 80, 8 72, 20 72; one of 2048: 14.6, 11.0, 11.3, 11.8).
constexpr int kPdStretch = 8;
struct PdMeta {  // of a stage: the two groups of 16 keys may lie in two pages
    float k_scale[2], v_scale[2];
    int there[2], unused[2];
};

template <int HD>
struct PdShape {
    static constexpr int kTile = HD * kPdKeys;              // bytes of the keys or of the values of a tile
    static constexpr int kStage = 2 * kTile;
    static constexpr int kWarp = kPdStages * kStage;
    static constexpr int kOffMeta = kPdWarps * kWarp;
    static constexpr int kSmem = kOffMeta + kPdWarps * kPdStages * (int)sizeof(PdMeta);
};

__device__ inline void mma_s8u8(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.u8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ inline void mma_s8s8(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ inline void cp_async4_zfill_to(uint32_t smem_addr, const void* src, uint32_t bytes) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_addr), "l"(src), "r"(bytes) : "memory");
}
template <int N>
__device__ inline void cp_async_wait_group() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ inline void cp_async_commit_group() { asm volatile("cp.async.commit_group;" ::: "memory"); }

template <typename T>
__device__ inline void load4(const void* p, size_t i, float (&v)[4]);
template <>
__device__ inline void load4<float>(const void* p, size_t i, float (&v)[4]) {
    const float4 x = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
    v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
}
template <>
__device__ inline void load4<uint16_t>(const void* p, size_t i, float (&v)[4]) {
    const uint2 x = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + i);
    v[0] = __uint_as_float(x.x << 16); v[1] = __uint_as_float(x.x & 0xffff0000u);
    v[2] = __uint_as_float(x.y << 16); v[3] = __uint_as_float(x.y & 0xffff0000u);
}

struct PdWork {
    int* arrived;     // [requests * kv_heads] of kPagedCounters, zero between calls
    float* partials;  // [blocks][2]: (maximum, sum) of 8 * NC rows, then their O
};

// Tiles of a request that this kernel serves (one where its rows attend nothing: they are written as zeros).
__device__ inline int pd_tiles(const PagedRequest& q, int group, int limit) {
    if (q.rows == 0 || (long long)q.rows * group > limit) return 0;
    return max(1, (q.hi + kPdKeys - 1) / kPdKeys - q.lo / kPdKeys);
}
__device__ inline long long pd_length(int tiles) { return tiles > 0 ? tiles + kPdStretch : 0; }

// ---- the order of the prompt kernel's blocks (one block of this kernel, beside those that attend) ---------------------------------------------
// A unit of T key tiles costs about T + kPdFixed; 148 run at once.  Units are cut into parts of at most `cut` tiles where that evens out the
// end: of sixteen cuts the one with the smallest max(longest, all / 148 + half of the longest) is taken.  The longest parts start first.  More units
// than kPdUnits even out by themselves: they go in the order of the requests, the last rows of each first, whole.
constexpr int kPdFixed = 3, kPdCuts = 16, kPdUnits = 2048;
struct PdOrderShared {
    int request[kPdUnits];
    unsigned short unit[kPdUnits], tiles[kPdUnits];
    int bucket[64], cost_parts[kPdCuts], cost_split[kPdCuts], warp_sum[kPdWarps], most, all, cut, place;
};
__device__ inline void paged_order(const PagedArgs& a, const PagedOrder& o, int group, PdOrderShared& s) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid < 64) s.bucket[tid] = 0;
    if (tid == 0) s.most = s.all = s.place = 0;
    // ---- units, request after request
    int units = 0;
    for (int r0 = 0; r0 < a.requests; r0 += kPdThreads) {
        const int r = r0 + tid;
        int n = 0;
        if (r < a.requests) {
            const long long rows = (long long)PagedRequest::of(a, r).rows * group;
            n = rows > a.skip_rows ? (int)((rows + kPpUnit - 1) / kPpUnit) : 0;
        }
        int up = n;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, up, d);
            if (lane >= d) up += v;
        }
        __syncthreads();
        if (lane == 31) s.warp_sum[warp] = up;
        __syncthreads();
        int base = units + up - n;
        for (int w = 0; w < kPdWarps; ++w) {
            if (w < warp) base += s.warp_sum[w];
            units += s.warp_sum[w];
        }
        for (uint32_t bits = __ballot_sync(0xffffffffu, n > 0); bits != 0u; bits &= bits - 1u) {  // a warp fills in its requests one by one
            const int from = __ffs(bits) - 1, b = __shfl_sync(0xffffffffu, base, from), m = __shfl_sync(0xffffffffu, n, from), rr = __shfl_sync(0xffffffffu, r, from);
            for (int u = lane; u < m; u += 32) {
                const int last_first = m - 1 - u;
                if (b + u < o.capacity) o.list[1 + b + u] = make_int4(rr, last_first, 1 << 16, 0);
                if (b + u < kPdUnits) {
                    s.request[b + u] = rr;
                    s.unit[b + u] = (unsigned short)last_first;
                }
            }
        }
    }
    if (tid == 0) o.list[0] = make_int4(min(units, o.capacity), 0, 0, 0);
    if (units > kPdUnits) return;
    __syncthreads();
    // ---- their tiles
    int most = 0, all = 0;
    for (int i = tid; i < units; i += kPdThreads) {
        const PagedRequest q = PagedRequest::of(a, s.request[i]);
        const int tiles = min(65535, PagedUnit::of(a, q, group, s.unit[i]).tiles(q, group));
        s.tiles[i] = (unsigned short)tiles;
        most = max(most, tiles);
        all += tiles;
    }
    most = __reduce_max_sync(0xffffffffu, most);
    all = __reduce_add_sync(0xffffffffu, all);
    if (lane == 0) {
        atomicMax(&s.most, most);
        atomicAdd(&s.all, all);
    }
    __syncthreads();
    most = max(s.most, 1);
    auto cut_of = [&](int i) { return max(4, (most * (kPdCuts - i) + kPdCuts - 1) / kPdCuts); };  // i = 0: whole units
    for (int i = warp; i < kPdCuts; i += kPdWarps) {
        const int cut = cut_of(i);
        int parts = 0, split = 0;
        for (int j = lane; j < units; j += 32) {
            const int n = max(1, (s.tiles[j] + cut - 1) / cut);
            parts += n;
            split += n > 1 ? n : 0;
        }
        parts = __reduce_add_sync(0xffffffffu, parts);
        split = __reduce_add_sync(0xffffffffu, split);
        if (lane == 0) { s.cost_parts[i] = parts; s.cost_split[i] = split; }
    }
    __syncthreads();
    if (warp == 0) {
        unsigned long long mine = ~0ull;  // (cost, which): the smallest cost, of equal ones the longest parts
        if (lane < kPdCuts) {
            const int parts = s.cost_parts[lane], split = s.cost_split[lane];
            const float longest = (float)(min(cut_of(lane), most) + kPdFixed + (split > 0 ? kPdFixed : 0));
            const float cost = fmaxf(longest, ((float)s.all + (float)parts * kPdFixed) * (float)a.kv_heads / 148.0f + 0.5f * longest);
            if (lane == 0 || ((long long)split * a.kv_heads <= o.split_blocks && parts <= o.capacity)) mine = ((unsigned long long)__float_as_uint(cost) << 32) | lane;
        }
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) {
            const unsigned long long v = __shfl_xor_sync(0xffffffffu, mine, d);
            mine = v < mine ? v : mine;
        }
        if (lane == 0) s.cut = cut_of((int)(mine & 31u));
    }
    __syncthreads();
    const int cut = min(s.cut, most);
    auto parts_of = [&](int tiles) { return max(1, (tiles + cut - 1) / cut); };
    auto bucket_of = [&](int tiles, int parts) { return 63 - min(63, (tiles + parts - 1) / parts * 64 / (cut + 1)); };
    for (int i = tid; i < units; i += kPdThreads) atomicAdd(&s.bucket[bucket_of(s.tiles[i], parts_of(s.tiles[i]))], parts_of(s.tiles[i]));
    __syncthreads();
    if (warp == 0) {
        const int n0 = s.bucket[2 * lane], n1 = s.bucket[2 * lane + 1];
        int up = n0 + n1;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, up, d);
            if (lane >= d) up += v;
        }
        s.bucket[2 * lane] = up - n0 - n1;
        s.bucket[2 * lane + 1] = up - n1;
        if (lane == 31) o.list[0] = make_int4(min(up, o.capacity), 0, 0, 0);
    }
    __syncthreads();
    for (int i = tid; i < units; i += kPdThreads) {
        const int tiles = s.tiles[i], parts = parts_of(tiles), place = parts > 1 ? atomicAdd(&s.place, parts) : 0, at = atomicAdd(&s.bucket[bucket_of(tiles, parts)], parts);
        for (int p = 0; p < parts; ++p)
            if (at + p < o.capacity) o.list[1 + at + p] = make_int4(s.request[i], s.unit[i], parts << 16 | p, place);
    }
}

// NB: bytes of the weights; NC: columns of eight rows.
template <int HD, typename T, int NB, int NC>
__global__ void __launch_bounds__(kPdThreads, NC == 1 ? 3 : 2) paged_decode_kernel(const PagedArgs a, const PdWork work, const PagedOrder order) {
    using S = PdShape<HD>;
    constexpr int KS = HD / 32, DT = HD / 16, ROWS = 8 * NC, PITCH = HD + 4;
    // A tile's largest weight times its largest value scale becomes kWhole (rounding errors of the factors stay below 2^24, 2^16).  A tile that has a weight below
    // kNarrow, of which less than ten (six) bits would be left, takes the rest of all of them as well; below kNothing there is no rest.
    constexpr float kWhole = NB == 3 ? 16776960.0f : 65520.0f, kNarrow = NB == 3 ? 1024.0f : 64.0f, kNothing = 0x1p-16f;
    extern __shared__ __align__(128) unsigned char pd_smem[];
    __shared__ long long s_before[kPdWarps + 1];
    __shared__ long long s_start;
    __shared__ int s_request, s_last;
    __shared__ float s_run[3 * ROWS];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3, group = a.heads / a.kv_heads;
    pdl_wait();
    const int blocks = (int)gridDim.x - (order.list != nullptr ? 1 : 0);
    if ((int)blockIdx.x == blocks) {
        static_assert(sizeof(PdOrderShared) <= S::kSmem, "the order's tables fit into the block's shared memory");
        paged_order(a, order, group, *reinterpret_cast<PdOrderShared*>(pd_smem));
        return;
    }
    // ---- the share of this block
    const int per = (a.requests + kPdThreads - 1) / kPdThreads;
    long long mine = 0;
    for (int i = 0; i < per; ++i) {
        const int r = tid * per + i;
        if (r < a.requests) mine += pd_length(pd_tiles(PagedRequest::of(a, r), group, ROWS));
    }
    long long before = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long v = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += v;
    }
    if (lane == 31) s_before[warp] = before;
    __syncthreads();
    before -= mine;
    long long total = 0;
    for (int w = 0; w < kPdWarps; ++w) {
        if (w == warp) before += total;
        total += s_before[w];
    }
    total *= a.kv_heads;
    before *= a.kv_heads;
    mine *= a.kv_heads;
    const long long share = max((long long)kPdWarps, (total + blocks - 1) / blocks);
    const long long w0 = (long long)blockIdx.x * share, w1 = min(total, w0 + share);
    if (w0 >= w1) return;
    if (w0 >= before && w0 < before + mine) {
        long long at = before;
        for (int i = 0; i < per; ++i) {
            const int r = tid * per + i;
            if (r >= a.requests) break;
            const long long n = pd_length(pd_tiles(PagedRequest::of(a, r), group, ROWS)) * a.kv_heads;
            if (w0 < at + n) {
                s_request = r;
                s_start = at;
                break;
            }
            at += n;
        }
    }
    __syncthreads();
    int r = s_request;
    long long start = s_start;  // of the request on the axis
    unsigned char* const ring = pd_smem + warp * S::kWarp;
    PdMeta* const meta = reinterpret_cast<PdMeta*>(pd_smem + S::kOffMeta) + warp * kPdStages;
    const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring), meta_at = (uint32_t)__cvta_generic_to_shared(meta);
    const int half = lane >> 4;  // group of 16 keys whose copies this lane makes
    // place of a key among the 16 of its group: the keys of the MMA's rows 0-7 and 8-15 are such that the weights come out of the
    // transpose with four keys in a row in one lane, which is how the values have them
    const int key16 = lane & 15, place16 = 8 * ((key16 >> 1) & 1) + 2 * (key16 >> 2) + (key16 & 1);

    for (long long w = w0; w < w1;) {
        const PagedRequest rq = PagedRequest::of(a, r);
        const int tiles = pd_tiles(rq, group, ROWS), length = (int)pd_length(tiles);
        if (tiles == 0 || w >= start + (long long)length * a.kv_heads) {
            start += (long long)length * a.kv_heads;
            ++r;
            continue;
        }
        const int h = (int)((w - start) / length), ua = (int)((w - start) - (long long)h * length);
        const int ub = (int)min((long long)length, ua + (w1 - w)), ta = max(0, ua - kPdStretch), tb = max(0, ub - kPdStretch);
        if (ta == tb) {
            w += ub - ua;
            continue;
        }
        const int key0 = rq.lo / kPdKeys * kPdKeys;  // of tile 0
        const int32_t* const table = a.table + (size_t)r * a.width;
        const int mine_n = tb - ta > warp ? (tb - ta - warp + kPdWarps - 1) / kPdWarps : 0;
        auto page_of = [&](int i) {  // of this lane's group of 16 keys in the warp's i-th tile; -1: nothing there, or nothing attended (the page may be another request's by now)
            const int key = key0 + (ta + warp + i * kPdWarps) * kPdKeys + half * 16;
            if (i >= mine_n || key >= rq.hi || key + 16 <= rq.lo) return -1;
            const int p = table[key / a.block];
            return p >= 0 && p < a.pages ? p : -1;
        };
        auto in_page = [&](int i) { return (key0 + (ta + warp + i * kPdWarps) * kPdKeys + half * 16) % a.block; };
        auto copy_keys = [&](int i, int page) {
            if (i < mine_n) {
                const int st = i % kPdStages, at = in_page(i);
                const size_t ph = (size_t)max(page, 0) * a.kv_heads + h;
                const uint32_t bytes = page >= 0 ? 16u : 0u;
                const int8_t* const src = a.k_codes + ph * a.block * HD + (at + key16) * 16;
                const uint32_t dst = ring_at + st * S::kStage + (half * 16 + place16) * 16;
#pragma unroll
                for (int c = 0; c < HD / 16; ++c) cp_async16_zfill_to(dst + c * (kPdKeys * 16), src + (size_t)c * a.block * 16, bytes);
                if (key16 == 0) {
                    const uint32_t m = meta_at + st * (uint32_t)sizeof(PdMeta) + half * 4;
                    cp_async4_zfill_to(m, a.k_scales + ph, page >= 0 ? 4u : 0u);
                    cp_async4_zfill_to(m + 8, a.v_scales + ph, page >= 0 ? 4u : 0u);
                    meta[st].there[half] = page >= 0;
                }
            }
            cp_async_commit_group();
        };
        auto copy_values = [&](int i, int page) {
            if (i < mine_n) {
                const int st = i % kPdStages, at = in_page(i);
                const size_t ph = (size_t)max(page, 0) * a.kv_heads + h;
                const uint32_t bytes = page >= 0 ? 16u : 0u;
                const int8_t* const src = a.v_codes + ph * a.block * HD + ((size_t)(at >> 4) * HD + key16) * 16;
                const uint32_t dst = ring_at + st * S::kStage + S::kTile + (half * HD + key16) * 16;
#pragma unroll
                for (int d = 0; d < HD / 16; ++d) cp_async16_zfill_to(dst + d * 256, src + d * 256, bytes);
            }
            cp_async_commit_group();
        };
        auto entry_of = [&](int i) {  // the same, not yet looked at
            const int key = key0 + (ta + warp + i * kPdWarps) * kPdKeys + half * 16;
            return i >= mine_n || key >= rq.hi || key + 16 <= rq.lo ? -1 : table[key / a.block];
        };
        int pages[kPdStages];
#pragma unroll
        for (int i = 0; i < kPdStages; ++i) pages[i] = entry_of(i);
        // (queries are on their way before the table's entries are needed)
        const int n_rows = rq.rows * group;
        float q[NC][KS][2][4];
#pragma unroll
        for (int nc = 0; nc < NC; ++nc) {
            const int row = nc * 8 + g;
            const size_t at = ((size_t)(rq.first + (row < n_rows ? row / group : 0)) * a.heads + (size_t)h * group + (row < n_rows ? row % group : 0)) * HD;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                for (int e = 0; e < 2; ++e) load4<T>(a.query, at + ks * 32 + e * 16 + t * 4, q[nc][ks][e]);
        }
#pragma unroll
        for (int i = 0; i < kPdStages; ++i) {
            const int page = pages[i] >= 0 && pages[i] < a.pages ? pages[i] : -1;
            copy_keys(i, page);
            copy_values(i, page);
        }
        int next_page = page_of(kPdStages);

        // ---- q of eight rows a column: bytes of round(q * 2^sh), the largest entry of a row between 2^22 and 2^23
        uint32_t qb[NC][3][KS][2];
        float q_unit[NC][2];   // of this lane's two score columns: 2^-sh * scale
        int last[NC][2], first_key[NC][2];
#pragma unroll
        for (int nc = 0; nc < NC; ++nc) {
            const int row = nc * 8 + g;
            const bool live = row < n_rows;
            float top = 0.0f;
            bool finite = true;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        top = fmaxf(top, fabsf(q[nc][ks][e][i]));
                        finite = finite && fabsf(q[nc][ks][e][i]) < INFINITY;
                    }
                }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const int bits = finite ? 1 : 0;
            finite = (bits & __shfl_xor_sync(0xffffffffu, bits, 1)) != 0;
            finite = ((finite ? 1 : 0) & __shfl_xor_sync(0xffffffffu, finite ? 1 : 0, 2)) != 0;
            int e2 = 0;
            if (top > 0.0f && top < INFINITY) frexpf(top, &e2);  // top in [2^(e2 - 1), 2^e2)
            const int sh = max(-120, min(120, 23 - e2));
            const float up = ldexpf(1.0f, sh);
            const int most = (1 << 23) - 1;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    uint32_t x[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[i] = live ? (uint32_t)max(-most, min(most, __float2int_rn(q[nc][ks][e][i] * up))) : 0u;
#pragma unroll
                    for (int b = 0; b < 3; ++b) {
                        const uint32_t pick = (uint32_t)(b | ((b + 4) << 4));
                        qb[nc][b][ks][e] = __byte_perm(__byte_perm(x[0], x[1], pick), __byte_perm(x[2], x[3], pick), 0x5410);
                    }
                }
            // (a row with an infinity or NaN has no scores)
            const float unit = finite ? ldexpf(a.scale2, -sh) : __int_as_float(0x7fffffff);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                q_unit[nc][e] = __shfl_sync(0xffffffffu, unit, 8 * t + 4 * e);
                const int col = nc * 8 + 2 * t + e;
                last[nc][e] = col < n_rows ? min(rq.pos0 + col / group, rq.hi - 1) : -1;
                first_key[nc][e] = window_start(rq.pos0 + col / group, a.window);
            }
        }
        const int sure_end = min(rq.pos0 + 1, rq.hi), sure_from = window_start(rq.pos0 + rq.rows - 1, a.window);  // keys that every row attends

        float m[NC][2], l[NC][2], acc[NC][DT][4];
#pragma unroll
        for (int nc = 0; nc < NC; ++nc) {
            m[nc][0] = m[nc][1] = -INFINITY;
            l[nc][0] = l[nc][1] = 0.0f;
#pragma unroll
            for (int d = 0; d < DT; ++d) acc[nc][d][0] = acc[nc][d][1] = acc[nc][d][2] = acc[nc][d][3] = 0.0f;
        }
        for (int i = 0; i < mine_n; ++i) {
            const int st = i % kPdStages;
            const unsigned char* const keys = ring + st * S::kStage;
            const unsigned char* const vals = keys + S::kTile;
            cp_async_wait_group<2 * kPdStages - 1>();
            __syncwarp();
            const PdMeta mt = meta[st];
            // ---- scores of 2 x 16 keys
            float s[NC][2][4];
#pragma unroll
            for (int half16 = 0; half16 < 2; ++half16) {
                int d[NC][3][4];
#pragma unroll
                for (int nc = 0; nc < NC; ++nc)
#pragma unroll
                    for (int b = 0; b < 3; ++b) d[nc][b][0] = d[nc][b][1] = d[nc][b][2] = d[nc][b][3] = 0;
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    uint32_t f[4];
                    ldmatrix_x4(f, keys + ((2 * ks + (lane >> 4)) * kPdKeys + half16 * 16 + (lane & 15)) * 16);
#pragma unroll
                    for (int nc = 0; nc < NC; ++nc) {
#pragma unroll
                        for (int b = 0; b < 2; ++b) mma_s8u8(d[nc][b], f, qb[nc][b][ks][0], qb[nc][b][ks][1]);
                        mma_s8s8(d[nc][2], f, qb[nc][2][ks][0], qb[nc][2][ks][1]);
                    }
                }
#pragma unroll
                for (int nc = 0; nc < NC; ++nc)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float v = fmaf((float)d[nc][2][e], 65536.0f, (float)(d[nc][0][e] + (d[nc][1][e] << 8)));
                        s[nc][half16][e] = v * (mt.k_scale[half16] * q_unit[nc][e & 1]);
                    }
            }
            // (the places of the keys are free again)
            __syncwarp();
            const int page_next = next_page;
            // The scales of a stage come with its keys, but its value scales are read above: both are in registers now.
            copy_keys(i + kPdStages, page_next);
            next_page = page_of(i + kPdStages + 1);
            const int tile_key = key0 + (ta + warp + i * kPdWarps) * kPdKeys;
            if (tile_key + kPdKeys > sure_end || tile_key < sure_from || !(mt.there[0] && mt.there[1])) {
#pragma unroll
                for (int nc = 0; nc < NC; ++nc)
#pragma unroll
                    for (int half16 = 0; half16 < 2; ++half16)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int key = tile_key + half16 * 16 + 4 * (g >> 1) + (g & 1) + 2 * (e >> 1);
                            if (key > last[nc][e & 1] || key < first_key[nc][e & 1] || !mt.there[half16]) s[nc][half16][e] = -INFINITY;
                        }
            }
            // ---- running maximum and sum of this lane's two columns; weights times value scale, the tile's largest weight times its largest scale as kWhole
            const float vmax = fmaxf(mt.v_scale[0], mt.v_scale[1]);
            const float whole[2] = {vmax > 0.0f ? kWhole * __fdividef(mt.v_scale[0], vmax) : 0.0f, vmax > 0.0f ? kWhole * __fdividef(mt.v_scale[1], vmax) : 0.0f};
            float v_unit[NC][2];
            bool wide = false;
#pragma unroll
            for (int nc = 0; nc < NC; ++nc) {
                float turn[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float own = fmaxf(fmaxf(s[nc][0][e], s[nc][0][e + 2]), fmaxf(s[nc][1][e], s[nc][1][e + 2]));
#pragma unroll
                    for (int o = 4; o < 32; o <<= 1) own = fmaxf(own, __shfl_xor_sync(0xffffffffu, own, o));
                    const float top = fmaxf(own, m[nc][e]);
                    const float base = top == -INFINITY ? 0.0f : top, own_base = own == -INFINITY ? 0.0f : own;
                    const float down = ex2_approx(own - base);  // (weights below are 2^(score - own): `down` times as much of the row's)
                    turn[e] = ex2_approx(m[nc][e] - base);
                    m[nc][e] = top;
                    v_unit[nc][e] = down * (vmax * (1.0f / kWhole));
                    float sum = 0.0f;
#pragma unroll
                    for (int half16 = 0; half16 < 2; ++half16)
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            float& x = s[nc][half16][e + 2 * k];
                            x = ex2_approx(x - own_base);
                            sum += x;
                            x *= whole[half16];
                            wide = wide || __float_as_uint(x) - __float_as_uint(kNothing) < __float_as_uint(kNarrow) - __float_as_uint(kNothing);
                        }
                    l[nc][e] = fmaf(l[nc][e], turn[e], sum * down);
                }
                if (__any_sync(0xffffffffu, turn[0] != 1.0f || turn[1] != 1.0f)) {
#pragma unroll
                    for (int d = 0; d < DT; ++d)
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc[nc][d][e] *= turn[e & 1];
                }
            }
            // O += V^T times whole numbers, in bytes (of the rest the second one has the sign)
            auto take = [&](auto rest, auto whole_of, float unit) {
                constexpr bool kRest = decltype(rest)::value;
                constexpr int B = kRest ? 2 : NB;
                uint32_t pb[NC][B][2];
#pragma unroll
                for (int nc = 0; nc < NC; ++nc)
#pragma unroll
                    for (int half16 = 0; half16 < 2; ++half16) {
                        uint32_t x[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) x[e] = whole_of(s[nc][half16][e]);
                        const uint32_t r0 = movmatrix_trans(__byte_perm(x[0], x[1], 0x5410)), r1 = movmatrix_trans(__byte_perm(x[2], x[3], 0x5410));
                        pb[nc][0][half16] = __byte_perm(r0, r1, 0x6420);
                        pb[nc][1][half16] = __byte_perm(r0, r1, 0x7531);
                        if constexpr (B == 3) {
                            const uint32_t r2 = movmatrix_trans(__byte_perm(x[0], x[1], 0x7632)), r3 = movmatrix_trans(__byte_perm(x[2], x[3], 0x7632));
                            pb[nc][2][half16] = __byte_perm(r2, r3, 0x6420);
                        }
                    }
                cp_async_wait_group<2 * kPdStages - 1>();
                __syncwarp();
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) {
                    uint32_t f[4];
                    ldmatrix_x4(f, vals + ((lane >> 4) * HD + dt * 16 + (lane & 15)) * 16);
#pragma unroll
                    for (int nc = 0; nc < NC; ++nc) {
                        int d[B][4];
#pragma unroll
                        for (int b = 0; b < B; ++b) {
                            d[b][0] = d[b][1] = d[b][2] = d[b][3] = 0;
                            if (kRest && b == B - 1) mma_s8s8(d[b], f, pb[nc][b][0], pb[nc][b][1]);
                            else mma_s8u8(d[b], f, pb[nc][b][0], pb[nc][b][1]);
                        }
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            float v = (float)(d[0][e] + (d[1][e] << 8));
                            if (B == 3) v = fmaf((float)d[B - 1][e], 65536.0f, v);
                            acc[nc][dt][e] = fmaf(v, v_unit[nc][e & 1] * unit, acc[nc][dt][e]);
                        }
                    }
                }
            };
            if (__any_sync(0xffffffffu, wide))  // what rounding leaves, in 16 bits more
                take(std::true_type(), [](float x) { return (uint32_t)min(__float2int_rn((x - rintf(x)) * 65536.0f), 32767); }, 1.0f / 65536.0f);
            take(std::false_type(), [](float x) { return __float2uint_rn(x); }, 1.0f);
            __syncwarp();
            copy_values(i + kPdStages, page_next);
        }
        cp_async_wait_group<0>();
        __syncthreads();
        // ---- the four warps' shares of the stretch
        float* const stage = reinterpret_cast<float*>(ring);        // [ROWS][PITCH], then maximum and sum of each row
        static_assert(ROWS * (PITCH + 2) * 4 <= S::kWarp, "the sums of a warp fit over its ring");
#pragma unroll
        for (int nc = 0; nc < NC; ++nc)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float sum = l[nc][e];
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                const int row = nc * 8 + 2 * t + e;
                if (g == 0) {
                    stage[ROWS * PITCH + 2 * row] = m[nc][e];
                    stage[ROWS * PITCH + 2 * row + 1] = sum;
                }
#pragma unroll
                for (int d = 0; d < DT; ++d) {
                    stage[row * PITCH + d * 16 + g] = acc[nc][d][e];
                    stage[row * PITCH + d * 16 + g + 8] = acc[nc][d][e + 2];
                }
            }
        __syncthreads();
        const bool whole = ta == 0 && tb == tiles;
        // (a block has at most one head that it goes on with, and one that it begins and leaves)
        float* const part = work.partials + ((size_t)blockIdx.x * 2 + (ta > 0 ? 0 : 1)) * ROWS * (HD + 2);
        for (int i = tid; i < n_rows * (HD / 4); i += kPdThreads) {
            const int row = i / (HD / 4), c = i % (HD / 4) * 4;
            float mw[kPdWarps], top = -INFINITY, sum = 0.0f;
            float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int k = 0; k < kPdWarps; ++k) {
                mw[k] = reinterpret_cast<const float*>(pd_smem + k * S::kWarp)[ROWS * PITCH + 2 * row];
                top = fmaxf(top, mw[k]);
            }
            const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll
            for (int k = 0; k < kPdWarps; ++k) {
                const float* const from = reinterpret_cast<const float*>(pd_smem + k * S::kWarp);
                const float f = ex2_approx(mw[k] - base);
                const float4 x = *reinterpret_cast<const float4*>(from + row * PITCH + c);
                sum = fmaf(from[ROWS * PITCH + 2 * row + 1], f, sum);
                y.x = fmaf(x.x, f, y.x); y.y = fmaf(x.y, f, y.y); y.z = fmaf(x.z, f, y.z); y.w = fmaf(x.w, f, y.w);
            }
            if (whole) {
                const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;  // (a row that attends nothing is zero)
                T* const to = static_cast<T*>(a.out) + ((size_t)(rq.first + row / group) * a.heads + (size_t)h * group + row % group) * HD + c;
                store_row(to, y.x * inv);
                store_row(to + 1, y.y * inv);
                store_row(to + 2, y.z * inv);
                store_row(to + 3, y.w * inv);
            } else {
                if (c == 0) reinterpret_cast<float2*>(part)[row] = make_float2(top, sum);
                *reinterpret_cast<float4*>(part + 2 * ROWS + row * HD + c) = y;
            }
        }
        if (!whole) {
            __threadfence();
            __syncthreads();
            // blocks that have tiles of this head
            const long long seq0 = start + (long long)h * length;
            const int c0 = (int)((seq0 + kPdStretch) / share), n = (int)((seq0 + length - 1) / share) - c0 + 1;
            if (tid == 0) s_last = atomicAdd(work.arrived + (size_t)r * a.kv_heads + h, 1) == n - 1;
            __syncthreads();
            if (s_last) {
                __threadfence();
                if (tid == 0) work.arrived[(size_t)r * a.kv_heads + h] = 0;
                auto part_of = [&](int k) { return work.partials + ((size_t)(c0 + k) * 2 + (k == 0 ? 1 : 0)) * ROWS * (HD + 2); };
                // [part][row]: maxima, sums, then 2^(maximum - largest) / sum; as many parts as fit over the ring at once
                constexpr int kHeld = kPdWarps * S::kWarp / (ROWS * 8);
                float* const tops = reinterpret_cast<float*>(pd_smem);
                float* const sums = tops + kHeld * ROWS;
                float4 y[(ROWS * (HD / 4) + kPdThreads - 1) / kPdThreads];
#pragma unroll
                for (float4& v : y) v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                float* const run = reinterpret_cast<float*>(s_run);  // running maximum and sum of a row, and what the parts before are worth now
                if (tid < ROWS) { run[tid] = -INFINITY; run[ROWS + tid] = 0.0f; }
                for (int k0 = 0; k0 < n; k0 += kHeld) {
                    const int held = min(kHeld, n - k0);
                    __syncthreads();
                    for (int i = tid; i < held * ROWS; i += kPdThreads) {
                        const float2 st = __ldcg(reinterpret_cast<const float2*>(part_of(k0 + i / ROWS)) + i % ROWS);
                        tops[i] = st.x;
                        sums[i] = st.y;
                    }
                    __syncthreads();
                    for (int row = warp; row < n_rows; row += kPdWarps) {
                        float top = run[row], sum = 0.0f;
                        const float before_top = top;
                        for (int k = lane; k < held; k += 32) top = fmaxf(top, tops[k * ROWS + row]);
                        top = warp_max(top);
                        const float base = top == -INFINITY ? 0.0f : top;
                        for (int k = lane; k < held; k += 32) {
                            const float f = ex2_approx(tops[k * ROWS + row] - base);
                            tops[k * ROWS + row] = f;
                            sum = fmaf(sums[k * ROWS + row], f, sum);
                        }
                        sum = warp_sum(sum);
                        if (lane == 0) {
                            const float turn = ex2_approx(before_top - base);
                            run[row] = top;
                            run[ROWS + row] = fmaf(run[ROWS + row], turn, sum);
                            run[2 * ROWS + row] = turn;
                        }
                    }
                    __syncthreads();
#pragma unroll
                    for (int j = 0; j < (int)(sizeof(y) / sizeof(y[0])); ++j) {
                        const int i = tid + j * kPdThreads, row = i / (HD / 4), c = i % (HD / 4) * 4;
                        if (i >= n_rows * (HD / 4)) break;
                        const float turn = run[2 * ROWS + row];
                        y[j].x *= turn; y[j].y *= turn; y[j].z *= turn; y[j].w *= turn;
#pragma unroll 8
                        for (int k = 0; k < held; ++k) {
                            const float4 x = __ldcg(reinterpret_cast<const float4*>(part_of(k0 + k) + 2 * ROWS + row * HD + c));
                            const float f = tops[k * ROWS + row];
                            y[j].x = fmaf(x.x, f, y[j].x); y[j].y = fmaf(x.y, f, y[j].y); y[j].z = fmaf(x.z, f, y[j].z); y[j].w = fmaf(x.w, f, y[j].w);
                        }
                    }
                }
#pragma unroll
                for (int j = 0; j < (int)(sizeof(y) / sizeof(y[0])); ++j) {
                    const int i = tid + j * kPdThreads, row = i / (HD / 4), c = i % (HD / 4) * 4;
                    if (i >= n_rows * (HD / 4)) break;
                    const float sum = run[ROWS + row], inv = sum == 0.0f ? 0.0f : 1.0f / sum;
                    T* const to = static_cast<T*>(a.out) + ((size_t)(rq.first + row / group) * a.heads + (size_t)h * group + row % group) * HD + c;
                    store_row(to, y[j].x * inv);
                    store_row(to + 1, y[j].y * inv);
                    store_row(to + 2, y[j].z * inv);
                    store_row(to + 3, y[j].w * inv);
                }
            }
        }
        __syncthreads();  // (the ring is free again)
        w += ub - ua;
    }
}

}  // namespace

bool paged_decode_serves(int head_dim) { return head_dim == 64 || head_dim == 128; }

size_t paged_decode_scratch_bytes(int head_dim, int max_rows) { return (size_t)kPdBlocks * 2 * (max_rows <= 8 ? 8 : 16) * (head_dim + 2) * 4; }

int paged_decode_launch(cudaStream_t stream, const PagedArgs& a, bool f32, int max_rows, int max_context, int* arrived, void* scratch, const PagedOrder& order) {
    const PdWork work = {arrived, static_cast<float*>(scratch)};
    // no more blocks than there can be shares of one tile a warp
    const long long most = (long long)a.requests * a.kv_heads * (max_context / kPdKeys + 2 + kPdStretch), blocks = (most + kPdWarps - 1) / kPdWarps;
    const int at_once = max_rows <= 8 ? kPdBlocks : kPdBlocks / 3 * 2;
    const dim3 grid((unsigned)(blocks < at_once ? blocks : at_once) + (order.list != nullptr ? 1 : 0));
    auto go = [&](auto kern, int smem) {
        const cudaError_t e = allow_all_dynamic_smem(kern);
        return e != cudaSuccess ? e : launch(kern, grid, dim3(kPdThreads), (size_t)smem, stream, true, a, work, order);
    };
    auto pick = [&](auto hd) {
        constexpr int HD = decltype(hd)::value;
        if (max_rows <= 8) return f32 ? go(paged_decode_kernel<HD, float, 3, 1>, PdShape<HD>::kSmem) : go(paged_decode_kernel<HD, uint16_t, 2, 1>, PdShape<HD>::kSmem);
        return f32 ? go(paged_decode_kernel<HD, float, 3, 2>, PdShape<HD>::kSmem) : go(paged_decode_kernel<HD, uint16_t, 2, 2>, PdShape<HD>::kSmem);
    };
    const cudaError_t e = a.head_dim == 128 ? pick(std::integral_constant<int, 128>()) : pick(std::integral_constant<int, 64>());
    if (e != cudaSuccess) return fail(KMLL_ERR_CUDA, "paged attention: %s", cudaGetErrorString(e));
    return KMLL_OK;
}

}  // namespace kmll
