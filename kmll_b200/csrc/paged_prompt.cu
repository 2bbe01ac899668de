// Attention of portions of prompts over the paged 8-bit cache on tcgen05: one block = up to 256 rows of a request and kv head.
//
// A row is a (token, query head) pair: all query heads of a kv head are in the same block, so codes are turned into operands once for all of
// them, and short portions still fill the 128 rows of an MMA.  Codes are exact in binary16, which is what both contractions run on:
//   S = Q K^T    Q as x * 2^sh = x0 + x1, two binary16 planes (f32 rows: 2^-22 of the row's largest entry) or one (bf16 rows: exact down to 2^-24 of
//                it); times k_scale of the key's page and 2^-sh
//   O += P V     the value scale of a key's page goes into the exponent, P = 2^(s + log2 v_scale - m + 7): no multiplication, and the sum of the
//                weights takes 1 / v_scale once per group of 16 keys.  P is two planes (f32 rows, 2^-22) or one (bf16 rows: 2^-11, and the weights of
//                many keys are rounded either way, where the result is rounded to 2^-9).  A maximum is one of s + log2 v_scale; with the 2^7 and
//                the 2^8 by which it may lag, P reaches 2^15 and ends at 2^-25, so that O loses what is 2^-32 of the row's largest weight times value scale;
//                the sum of the weights has all of them.
// Two streams of work share the keys that are brought in: two tiles of 128 rows, or (where there are 128 rows at most) the even and the odd
// key tiles of one, each with a maximum, a sum and an O of its own, merged at the end.  Roles of the 28 warps:
//   warps 0-7, 8-15  softmax of a stream, two threads per row with 64 keys of a tile each: scores by tcgen05.ld, their maximum (both threads'), then
//                    the weights, which go back in the place of the scores
//   warps 16-23      fetch the codes of a tile of 128 keys into registers while the tile before is at work, and write them as binary16 operands
//                    (128-byte swizzle, both K-major: values lie with the keys of a column together)
//   warp 24          issues S = Q K^T and O += P V
// O is rescaled only when a row's maximum has grown by more than 2^8.  The accumulators cut what does not fit into 24 bits, so an O of many tiles
// comes out short, by 2.4e-7 a tile where every tile adds two planes: of f32 rows it leaves tensor memory every six tiles and is summed in f32,
// rounded, in the workspace (relative error of a prompt of 2048: 1.4e-6 without, 8.9e-7 so; of 8192 5.4e-6 and 1.1e-6; every four tiles 6.6e-7
// and 8.0e-7; 32 query heads over 8, 2048 tokens: 73, 85 and 88 us).  Where in the workspace is a block's for as long as it runs: a bit that it claims.  bf16 results are rounded to 2^-9 in any case.
// Which rows a block takes, and which part of their keys, stands in a list that a block of the kernel for few rows has made (paged_decode.cu):
// parts leave maximum, sum and O in the workspace, and the last to arrive joins them in order.
// Every wait is bounded; a time-out raises the status word, and the block frees its tensor memory and returns (no copies are under way: the
// fetches are loads).
// Bound: the softmax between the two MMAs of a tile (one thread a row took 3400 cycles a tile, all of it latency), beside the MMAs of f32 rows' two
// planes.  32 query heads over 8, head size 128, random codes: 2048 tokens 61 us (bf16), 85 us (f32), 8192
// tokens 583 us (bf16, 0.94 PFLOP/s of the causal half) and 914 us (f32); 512 tokens behind 32256 328 us (bf16, 0.83).
#include <climits>
#include <type_traits>

#include "internal.cuh"
#include "mma_bf16.cuh"
#include "paged.cuh"
#include "tcgen05.cuh"

namespace kmll {

__device__ int g_paged_prompt_status = 0;

namespace {

constexpr int kPpRows = 128, kPpGroups = kPpKeys / 16;
constexpr int kPpConvert = 16, kPpIssue = 24;  // first warps of the roles behind the softmax
constexpr int kPpThreads = 28 * 32;
// Registers a thread: 72 at the launch (896 threads), then by warpgroup: 4 * 128 * 88 + 2 * 128 * 64 + 128 * 24 = 896 * 72.
constexpr int kPpRegsLaunch = 72;
constexpr int kPpBox = 128 * 128;      // 128 rows of 64 binary16 entries
constexpr uint32_t kPpTmemO = 256;     // scores at 0 and 128, the streams' O behind them

struct PpScales {  // of a tile, per group of 16 keys
    float k[kPpGroups], log_v[kPpGroups], inv_v[kPpGroups];
    uint32_t there, unused[7];
};

// NP: planes of Q and of P
template <int HD, int NP>
struct PpShape {
    static constexpr int kQPlane = kPpRows * HD * 2, kQTile = NP * kQPlane, kK = kPpKeys * HD * 2, kVBox = HD * 128, kV = 2 * kVBox;
    static constexpr int kOffK = 2 * kQTile, kStages = kOffK + 2 * (kK + kV) <= 216 * 1024 ? 2 : 1;
    static constexpr int kOffV = kOffK + kStages * kK, kOffScales = kOffV + kStages * kV;
    static constexpr int kOffStat = kOffScales + 4 * (int)sizeof(PpScales), kOffTop = kOffStat + 4 * kPpRows * 16;
    static constexpr int kOffUnit = kOffTop + 2 * 4 * kPpRows * 4;
    static constexpr int kOffBars = kOffUnit + 2 * kPpRows * 8;
    static constexpr int kSmemBytes = kOffBars + 256 + 1024;
    static constexpr int kStagePitch = HD / 2 + 4;  // rows of O on their way out, over the operands
    static_assert(kSmemBytes <= 227 * 1024 && 16 * 32 * kStagePitch * 4 <= kOffScales, "shape");
};

// two codes as binary16: 0x6400 + b is 1024 + b
__device__ inline uint32_t pp_halves(uint32_t biased, uint32_t pick) {
    uint32_t d;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(__byte_perm(biased, 0x64646464u, pick)), "r"(0x64806480u));
    return d;
}
// sixteen codes -> the 16-byte pieces c8, c8 + 1 of a 128-byte row
__device__ inline void pp_put(unsigned char* row, int c8, int swizzle, uint4 u) {
    uint4 a, b;
    u.x ^= 0x80808080u; u.y ^= 0x80808080u; u.z ^= 0x80808080u; u.w ^= 0x80808080u;
    a.x = pp_halves(u.x, 0x4140); a.y = pp_halves(u.x, 0x4342); a.z = pp_halves(u.y, 0x4140); a.w = pp_halves(u.y, 0x4342);
    b.x = pp_halves(u.z, 0x4140); b.y = pp_halves(u.z, 0x4342); b.z = pp_halves(u.w, 0x4140); b.w = pp_halves(u.w, 0x4342);
    *reinterpret_cast<uint4*>(row + ((c8 ^ swizzle) << 4)) = a;
    *reinterpret_cast<uint4*>(row + (((c8 + 1) ^ swizzle) << 4)) = b;
}
// (x0, x1) -> binary16 pair, and the pair of the remainders
__device__ inline uint32_t pp_round(float x0, float x1) {
    uint32_t d;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(x1), "f"(x0));
    return d;
}
__device__ inline uint32_t pp_rest(float x0, float x1, uint32_t hi) {
    const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&hi));
    return pp_round(x0 - y.x, x1 - y.y);
}

template <int E>
__device__ inline void load_entries(const float* p, float (&x)[E]) {
    if constexpr (E == 4) {
        const float4 u = *reinterpret_cast<const float4*>(p);
        x[0] = u.x; x[1] = u.y; x[2] = u.z; x[3] = u.w;
    } else {
        const float2 u = *reinterpret_cast<const float2*>(p);
        x[0] = u.x; x[1] = u.y;
    }
}
template <int E>
__device__ inline void load_entries(const uint16_t* p, float (&x)[E]) {
#pragma unroll
    for (int k = 0; k < E / 2; ++k) {
        const uint32_t u = reinterpret_cast<const uint32_t*>(p)[k];
        x[2 * k] = __uint_as_float(u << 16);
        x[2 * k + 1] = __uint_as_float(u & 0xffff0000u);
    }
}

// pairs of f32 in one instruction
__device__ inline uint64_t pp_pair(float x, float y) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(x), "f"(y));
    return d;
}
__device__ inline float2 pp_unpair(uint64_t d) {
    float2 v;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(v.x), "=f"(v.y) : "l"(d));
    return v;
}
__device__ inline uint64_t pp_fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ inline uint64_t pp_add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

struct PpWork {
    const int4* list;
    int* arrived;      // [kPpSplitBlocks]: parts' places * kv heads; zero between calls
    uint32_t* taken;   // [kPpSums / 32]: places of sums that a block holds, a bit each; zero between calls
    float* partials;   // [parts' places * kv heads]: (maximum, sum) of 256 rows, then their O
    float* sums;       // [place][2][HD / 4][128 rows][4]: O of earlier tiles, of one block at a time
};
template <int HD>
__host__ __device__ constexpr size_t pp_partial_floats() { return (size_t)kPpUnit * (HD + 2); }
constexpr int kPpDrain = 6;
// A weight is at most 2^(kPpLag + kPpRoom), half of what binary16 holds.
constexpr float kPpLag = 8.0f, kPpRoom = 7.0f;

template <int HD, typename T>
__global__ void __launch_bounds__(kPpThreads, 1) paged_prompt_kernel(const PagedArgs a, const PpWork work) {
    constexpr int NP = sizeof(T) == 4 ? 2 : 1;
    using S = PpShape<HD, NP>;
    constexpr int kStages = S::kStages;
    extern __shared__ unsigned char pp_smem_raw[];
    __shared__ int s_place;  // this block's place for sums, -1: none
    unsigned char* const smem = pp_smem_raw + ((1024u - (smem_u32(pp_smem_raw) & 1023u)) & 1023u);
    uint64_t* const s_full = reinterpret_cast<uint64_t*>(smem + S::kOffBars);  // [2] the scores of a stream's tile are there
    uint64_t* const p_ready = s_full + 2;    // [2] its weights are there (and O is rescaled)
    uint64_t* const pv_done = p_ready + 2;   // [2] its O has taken the tile
    uint64_t* const k_full = pv_done + 2;    // [kStages]
    uint64_t* const v_full = k_full + 2;     // [kStages]
    uint64_t* const k_free = v_full + 2;     // [kStages] the scores that need the stage are done
    uint64_t* const v_free = k_free + 2;     // [kStages]
    uint64_t* const sc_full = v_free + 2;    // [4] the scales of a tile are there
    uint64_t* const pair = sc_full + 4;      // [8] both threads of a row have left their maxima
    uint64_t* const q_full = pair + 8;       // the queries are there
    uint64_t* const place_full = q_full + 1; // the block's place for sums is known
    uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(place_full + 1);
    int* const s_last = reinterpret_cast<int*>(tmem_slot + 1);  // all other parts of the unit have arrived
    PpScales* const scales = reinterpret_cast<PpScales*>(smem + S::kOffScales);
    float* const units = reinterpret_cast<float*>(smem + S::kOffUnit);
    int* const row_of = reinterpret_cast<int*>(units + 2 * kPpRows);  // rows of the block among the step's (token, head) rows
    const int tid = threadIdx.x, lane = tid & 31, warp = uniform_warp_index(), group = a.heads / a.kv_heads, h = blockIdx.x;
    const int block_log = 31 - __clz(a.block), in_block = a.block - 1;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int entries = work.list[0].x;
    const int4 entry = work.list[1 + blockIdx.y];  // (the list has room for one per block)
    if ((int)blockIdx.y >= entries) return;
    if (tid == 0) {
        for (int b = 0; b < 2; ++b) {
            mbar_init(&s_full[b], 1);
            mbar_init(&p_ready[b], 8);
            mbar_init(&pv_done[b], 1);
            mbar_init(&k_full[b], 8);
            mbar_init(&v_full[b], 8);
            mbar_init(&k_free[b], 1);
            mbar_init(&v_free[b], 1);
        }
        for (int b = 0; b < 4; ++b) mbar_init(&sc_full[b], 1);
        for (int b = 0; b < 8; ++b) mbar_init(&pair[b], 2);
        mbar_init(q_full, kPpConvert);
        mbar_init(place_full, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (tid == 0) s_place = -1;
    if (warp == kPpIssue) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tcgen05_fence_before();
    __syncthreads();  // (columns first, then the dependents: tcgen05.cuh)
    tcgen05_fence_after();
    pdl_launch_dependents();
    constexpr bool drains = NP == 2;
    bool ok = true;
    {
        const PagedRequest rq = PagedRequest::of(a, entry.x);
        const PagedUnit un = PagedUnit::of(a, rq, group, entry.y);
        const int parts = entry.z >> 16, part = entry.z & 0xffff;
        const int row0 = un.row0, live = un.live;
        const bool two = live > kPpRows;  // two tiles of rows; else two shares of the keys
        auto own_pos = [&](int r) { return rq.pos0 + (row0 + r) / group; };  // (a context longer than its table row is cut at the table's end)
        // this part's tiles, counted from its first one
        const int all_tiles = un.tiles(rq, group), size = (all_tiles + parts - 1) / parts, from_tile = min(all_tiles, part * size);
        const int tiles = min(size, all_tiles - from_tile), first = un.first + from_tile * kPpKeys;
        const int tiles0 = two ? min(tiles, max(0, un.tiles_to(rq, group, kPpRows - 1) - from_tile)) : tiles;  // of the first stream where the streams are tiles of rows
        const bool keeps_sums = drains && (two ? tiles : (tiles + 1) / 2) > kPpDrain;  // a stream's O leaves tensor memory before its end
        const uint32_t base = smem_u32(smem);

        if (warp >= kPpConvert && warp < kPpIssue) {
            asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
            // ---- codes to operands
            const int tt = tid - 32 * kPpConvert & 127, side = tid - 32 * kPpConvert >> 7;  // the key; of the values the group of 16 keys tt / 16, columns tt % 16, + 16, ..; half of either
            const int32_t* const table = a.table + (size_t)entry.x * a.width;
            constexpr int U = HD / 32;  // 16-byte groups of half a key; columns of a group of values per thread
            uint4 kc[U], vc[U];
            // Lanes 0-7 (and again): page of group lane & 7 of tile j, -1: nothing there.  (An entry asked for a tile earlier costs registers that the loop lacks: a
            // prompt of 2048, 32 query heads over 8, f32 88 us, so 84.)
            auto page_of = [&](int j) {
                const int key = first + j * kPpKeys + (lane & 7) * 16, p = j < tiles && key < rq.hi ? table[key >> block_log] : -1;
                return p >= 0 && p < a.pages ? p : -1;
            };
            // (volatile loads: they stay where they are written, a tile ahead of their use; where nothing is there any codes do, no row sees them)
            // One page per thread and tile: more shuffles between the loads would share their scoreboards and wait for them.
            auto fetch_keys = [&](int j, int p) {
                const uint4* const src = reinterpret_cast<const uint4*>(a.k_codes + ((size_t)max(p, 0) * a.kv_heads + h) * a.block * HD) + ((first + j * kPpKeys + tt) & in_block) + (size_t)side * U * a.block;
#pragma unroll
                for (int c = 0; c < U; ++c) kc[c] = ld_stream_u4(src + (size_t)c * a.block);
            };
            auto fetch_values = [&](int j, int p) {
                const uint4* const src = reinterpret_cast<const uint4*>(a.v_codes + ((size_t)max(p, 0) * a.kv_heads + h) * a.block * HD) +
                                         (size_t)(((first + j * kPpKeys + (tt & ~15)) & in_block) >> 4) * HD + side * (HD / 2) + (tt & 15);
#pragma unroll
                for (int c = 0; c < U; ++c) vc[c] = ld_stream_u4(src + c * 16);
            };
            int page = page_of(0);
            float ks = 0.0f, vs = 0.0f;  // lanes 0-7 of the first warp: scales of the tile in kc
            auto fetch_scales = [&](int p) {
                if (warp == kPpConvert && lane < 8) {
                    ks = p >= 0 ? a.k_scales[(size_t)p * a.kv_heads + h] : 0.0f;
                    vs = p >= 0 ? a.v_scales[(size_t)p * a.kv_heads + h] : 0.0f;
                }
            };
            if (tiles > 0) {
                fetch_scales(page);
                const int p = __shfl_sync(0xffffffffu, page, tt >> 4);
                fetch_keys(0, p);
                fetch_values(0, p);
            }
            for (int j = 0; j < tiles; ++j) {
                const int st = j % kStages, before = j - kStages;  // the use of the stage before
                ok = before < 0 || warp_wait(&k_free[st], (uint32_t)(before / kStages) & 1u);
                if (!ok) break;
                if (warp == kPpConvert) {
                    // (every softmax warp has read the scales of tile j - 4: it wrote the weights of that tile before the scores of tile j - 2 began)
                    PpScales& sc = scales[j & 3];
                    if (lane < 8) {
                        sc.k[lane] = ks;
                        // (a page of zeros or of next to nothing: its weights still count in the sum, and do not push others out of binary16)
                        const float v = fmaxf(vs, 0x1p-80f);
                        sc.log_v[lane] = page >= 0 ? log2f(v) : 0.0f;
                        sc.inv_v[lane] = page >= 0 ? 1.0f / v : 0.0f;
                    }
                    const uint32_t there = __ballot_sync(0xffffffffu, page >= 0) & 0xffu;
                    if (lane == 0) sc.there = there;
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sc_full[j & 3]);
                }
                unsigned char* const krow = smem + S::kOffK + st * S::kK + tt * 128;
#pragma unroll
                for (int c = 0; c < U; ++c) pp_put(krow + ((side * U + c) >> 2) * kPpBox, ((side * U + c) & 3) * 2, tt & 7, kc[c]);
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&k_full[st]);
                const int next = page_of(j + 1), p_next = __shfl_sync(0xffffffffu, next, tt >> 4);
                if (j + 1 < tiles) {
                    fetch_scales(next);
                    fetch_keys(j + 1, p_next);
                }
                ok = before < 0 || warp_wait(&v_free[st], (uint32_t)(before / kStages) & 1u);
                if (!ok) break;
                unsigned char* const vrow = smem + S::kOffV + st * S::kV + (tt >> 6) * S::kVBox + (side * (HD / 2) + (tt & 15)) * 128;
#pragma unroll
                for (int c = 0; c < U; ++c) pp_put(vrow + c * 2048, ((tt >> 4) & 3) * 2, tt & 7, vc[c]);
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&v_full[st]);
                if (j + 1 < tiles) fetch_values(j + 1, p_next);
                page = next;
            }
        } else if (warp >= kPpIssue) {  // (a warpgroup changes its registers with one instruction)
            asm volatile("setmaxnreg.dec.sync.aligned.u32 24;");
            if (warp == kPpIssue + 1 && keeps_sums) {
                // a place for sums: the first free bit of a word from the block's number on (there are more places than blocks that run at once)
                const uint32_t number = blockIdx.y * gridDim.x + blockIdx.x;
                uint32_t word = number / 32 % (kPpSums / 32), bit = number % 32;
                int place = -1;
                for (int i = 0; i < 4 * kPpSums && place < 0 && lane == 0; ++i) {
                    const uint32_t held = atomicOr(&work.taken[word], 1u << bit), free = __funnelshift_r(~held, ~held, bit);
                    if ((free & 1u) != 0u) place = (int)(word * 32 + bit);
                    else if (free != 0u) bit = (bit + __ffs(free) - 1) & 31u;
                    else word = word + 1 == kPpSums / 32 ? 0 : word + 1;
                }
                if (lane == 0) {
                    __threadfence();  // (what the block before did there is done)
                    s_place = place;
                    mbar_arrive(place_full);
                }
            }
            if (warp == kPpIssue) {
                constexpr uint32_t idesc_s = gemm_idesc_f16(128, kPpKeys), idesc_o = gemm_idesc_f16(128, HD);
                const uint64_t dq = gemm_smem_desc(base), dk = gemm_smem_desc(base + S::kOffK), dv = gemm_smem_desc(base + S::kOffV);
                const uint32_t lead = elect_lead();
                // scores of tile j for stream s; `last`: nobody else needs the keys
                auto scores = [&](int j, int s, bool last) {
                    const int st = j % kStages;
                    if (!warp_wait(&k_full[st], (uint32_t)(j / kStages) & 1u)) return false;
                    tcgen05_fence_after();
                    const uint64_t dkj = dk + (uint64_t)(st * (S::kK >> 4)), dqs = dq + (uint64_t)(two ? s * (S::kQTile >> 4) : 0);
                    uint32_t acc = 0u;
#pragma unroll
                    for (int p = NP - 1; p >= 0; --p)  // the small products first
#pragma unroll
                        for (int ks = 0; ks < HD / 16; ++ks) {
                            const int at = (ks >> 2) * kPpBox + (ks & 3) * 32;
                            lead_mma_f16(lead, (uint32_t)s * 128u, dqs + (uint64_t)((p * S::kQPlane + at) >> 4), dkj + (uint64_t)(at >> 4), idesc_s, acc);
                            acc = 1u;
                        }
                    lead_commit(lead, &s_full[s]);
                    if (last) lead_commit(lead, &k_free[st]);
                    return true;
                };
                // O of stream s takes its n-th tile, tile j
                auto values = [&](int j, int s, int n, bool last) {
                    const int st = j % kStages;
                    if (!(warp_wait(&v_full[st], (uint32_t)(j / kStages) & 1u) && warp_wait(&p_ready[s], (uint32_t)n & 1u))) return false;
                    tcgen05_fence_after();
                    const uint64_t dvj = dv + (uint64_t)(st * (S::kV >> 4));
                    uint32_t acc = (drains ? n % kPpDrain : n) > 0 ? 1u : 0u;
#pragma unroll
                    for (int p = NP - 1; p >= 0; --p)
#pragma unroll
                        for (int ks = 0; ks < kPpKeys / 16; ++ks) {  // weights of 32 keys: 16 columns of the first plane, 16 of the second
                            lead_mma_f16_ts(lead, kPpTmemO + (uint32_t)s * 128u, (uint32_t)(s * 128 + (ks >> 1) * 32 + p * 16 + (ks & 1) * 8),
                                            dvj + (uint64_t)(((ks >> 2) * S::kVBox + (ks & 3) * 32) >> 4), idesc_o, acc);
                            acc = 1u;
                        }
                    lead_commit(lead, &pv_done[s]);
                    if (last) lead_commit(lead, &v_free[st]);
                    return true;
                };
                ok = warp_wait(q_full, 0u);
                tcgen05_fence_after();
                if (!ok) {
                } else if (two) {
                    // (the second stream has every tile, the first the tiles up to its own rows' positions)
                    if (tiles > 0) ok = (tiles0 < 1 || scores(0, 0, false)) && scores(0, 1, true);
                    for (int j = 0; j < tiles && ok; ++j) {
                        if (j < tiles0) ok = values(j, 0, j, false);
                        if (ok && j + 1 < tiles0) ok = scores(j + 1, 0, false);
                        if (ok) ok = values(j, 1, j, true);
                        if (ok && j + 1 < tiles) ok = scores(j + 1, 1, true);
                    }
                } else {
                    if (tiles > 0) ok = scores(0, 0, true) && (kStages < 2 || tiles < 2 || scores(1, 1, true));
                    for (int j = 0; j < tiles && ok; ++j) {
                        if (kStages < 2 && j + 1 < tiles) ok = scores(j + 1, (j + 1) & 1, true);
                        if (ok) ok = values(j, j & 1, j >> 1, true);
                        if (ok && kStages >= 2 && j + 2 < tiles) ok = scores(j + 2, j & 1, true);
                    }
                }
            }
        } else if (warp < kPpConvert) {
            asm volatile("setmaxnreg.inc.sync.aligned.u32 88;");
            // ---- Q first: a warp has a row at a time, HD / 32 entries a lane; its largest entry gives the power of two
            constexpr int E = HD / 32, kBatch = 8;
            for (int r0 = warp; r0 < (two ? 2 : 1) * kPpRows; r0 += kPpConvert * kBatch) {
                float x[kBatch][E];
#pragma unroll
                for (int i = 0; i < kBatch; ++i) {
                    const int r = r0 + i * kPpConvert;
#pragma unroll
                    for (int k = 0; k < E; ++k) x[i][k] = 0.0f;
                    const int token = (row0 + r) / group, place = (rq.first + token) * a.heads + h * group + (row0 + r - token * group);
                    if (lane == 0) row_of[r] = place;
                    if (r < live) load_entries<E>(static_cast<const T*>(a.query) + (size_t)place * HD + lane * E, x[i]);
                }
#pragma unroll
                for (int i = 0; i < kBatch; ++i) {
                    const int r = r0 + i * kPpConvert;
                    float top = 0.0f;
                    bool finite = true;
#pragma unroll
                    for (int k = 0; k < E; ++k) {
                        top = fmaxf(top, fabsf(x[i][k]));
                        finite = finite && fabsf(x[i][k]) < INFINITY;
                    }
                    // the power of two that brings the largest entry between 2^10 and 2^11 (its exponent field is 264 less the entry's)
                    const uint32_t most = __reduce_max_sync(0xffffffffu, __float_as_uint(top));
                    const float up = __uint_as_float((uint32_t)min(254, max(1, 264 - (int)(most >> 23))) << 23);
                    finite = __all_sync(0xffffffffu, finite) != 0;
                    if (lane == 0) units[r] = finite ? up : __int_as_float(0x7fffffff);
                    unsigned char* const at = smem + (r >> 7) * S::kQTile + (lane * E >> 6) * kPpBox + (r & 127) * 128 + ((((lane * E >> 3) & 7) ^ (r & 7)) << 4) + (lane * E & 7) * 2;
                    uint32_t hi[E / 2], lo[E / 2];
#pragma unroll
                    for (int k = 0; k < E / 2; ++k) {
                        hi[k] = pp_round(x[i][2 * k] * up, x[i][2 * k + 1] * up);
                        lo[k] = pp_rest(x[i][2 * k] * up, x[i][2 * k + 1] * up, hi[k]);
                    }
                    if constexpr (E == 4) {
                        *reinterpret_cast<uint2*>(at) = make_uint2(hi[0], hi[1]);
                        if (NP == 2) *reinterpret_cast<uint2*>(at + S::kQPlane) = make_uint2(lo[0], lo[1]);
                    } else {
                        *reinterpret_cast<uint32_t*>(at) = hi[0];
                        if (NP == 2) *reinterpret_cast<uint32_t*>(at + S::kQPlane) = lo[0];
                    }
                }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(q_full);
            asm volatile("bar.sync 1, 512;" ::: "memory");  // (units and places of rows are there)
            int place = -1;
            if (keeps_sums) {
                ok = warp_wait(place_full, 0u);
                place = s_place;
                ok = ok && place >= 0;  // (none: the workspace was not zero)
            }
            // ---- softmax: the stream's tiles j = j0, j0 + step, ..
            const int stream = warp >> 3, half = (warp >> 2) & 1, r = (warp & 3) * 32 + lane, in_unit = two ? stream * kPpRows + r : r;
            uint64_t* const pair_bar = pair + stream * 4 + (warp & 3);  // of the two warps that have the same rows
            float* const tops = reinterpret_cast<float*>(smem + S::kOffTop) + stream * 2 * kPpRows + r;  // [tile parity][stream][half][row]
            const int step = two ? 1 : 2, end = two && stream == 0 ? tiles0 : tiles;
            const int own = own_pos(in_unit), pos = min(own, rq.hi - 1), lo = window_start(own, a.window);
            const int row_a = two ? stream * kPpRows : 0, row_b = min(live, row_a + kPpRows) - 1, first_pos = own_pos(row_a), last_own = max(own_pos(max(row_b, row_a)), 0);
            const float unit = a.scale2 / units[in_unit];  // (a row with an infinity or NaN has no scores)
            const uint32_t rows = (uint32_t)((warp & 3) * 32) << 16;
            const uint32_t ts = rows + (uint32_t)stream * 128u, to = rows + kPpTmemO + (uint32_t)stream * 128u;
            float m_ref = -INFINITY, l = 0.0f;
            // O of the tiles so far leaves tensor memory: half of the columns each, relative to the maximum at that time
            float drained_ref = -INFINITY;
            // (four columns of 128 rows lie together, so that a warp writes whole runs)
            auto sums_of = [&](int s, int column) { return reinterpret_cast<float4*>(work.sums) + ((size_t)place * 2 + s) * (HD / 4) * kPpRows + (size_t)(column / 4) * kPpRows + r; };
            int n = 0;  // tiles of this stream so far
            auto drain = [&]() {
                const float turn = drained_ref == -INFINITY ? 0.0f : ex2_approx(drained_ref - m_ref);
                float4* const run = sums_of(stream, half * (HD / 2));
#pragma unroll 1
                for (int i = 0; i < HD / 32; ++i) {
                    float4 x[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) x[k] = n > kPpDrain ? run[(i * 4 + k) * kPpRows] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    uint32_t o[16];
                    tmem_load_x16(to + half * (HD / 2) + i * 16, o);
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        float4 v = make_float4(__uint_as_float(o[4 * k]), __uint_as_float(o[4 * k + 1]), __uint_as_float(o[4 * k + 2]), __uint_as_float(o[4 * k + 3]));
                        v.x = fmaf(x[k].x, turn, v.x); v.y = fmaf(x[k].y, turn, v.y); v.z = fmaf(x[k].z, turn, v.z); v.w = fmaf(x[k].w, turn, v.w);
                        run[(i * 4 + k) * kPpRows] = v;
                    }
                }
                drained_ref = m_ref;
            };
            for (int j = two ? 0 : stream; j < end && ok; j += step, ++n) {
                const int t0 = first + j * kPpKeys;
                ok = warp_wait(&sc_full[j & 3], (uint32_t)(j >> 2) & 1u) && warp_wait(&s_full[stream], (uint32_t)n & 1u);
                if (!ok) break;
                tcgen05_fence_after();
                const PpScales& sc = scales[j & 3];
                const uint32_t there_bits = sc.there;
                const bool masked = t0 + kPpKeys - 1 > first_pos || (a.window > 0 && t0 < last_own - a.window + 1) || there_bits != 0xffu;
                // keys of chunk c that the row attends, a bit each
                auto seen_of = [&](int c) {
                    const int k0 = t0 + c * 32, from = max(lo - k0, 0), to_key = min(pos - k0, 31);
                    const uint32_t pair = there_bits >> (2 * c);
                    const uint32_t there = (pair & 1u ? 0xffffu : 0u) | (pair & 2u ? 0xffff0000u : 0u);
                    return from <= to_key ? (0xffffffffu << from) & (0xffffffffu >> (31 - to_key)) & there : 0u;
                };
                // the largest s + log2 v_scale of 32 scores
                auto largest = [&](auto is_masked, int c, uint32_t (&d)[32]) {
                    const uint32_t seen = is_masked.value ? seen_of(c) : 0u;
                    if (is_masked.value) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) d[i] = (seen & (1u << i)) != 0u ? d[i] : 0xff800000u;
                    }
                    float top = -INFINITY;
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
                        for (int i = 0; i < 16; i += 4) {
                            mx[0] = fmaxf(fmaxf(mx[0], __uint_as_float(d[16 * k + i])), __uint_as_float(d[16 * k + i + 1]));
                            mx[1] = fmaxf(fmaxf(mx[1], __uint_as_float(d[16 * k + i + 2])), __uint_as_float(d[16 * k + i + 3]));
                        }
                        const float x = fmaxf(mx[0], mx[1]);
                        if (x > -INFINITY) top = fmaxf(top, fmaf(x, sc.k[2 * c + k] * unit, sc.log_v[2 * c + k]));
                    }
                    return top;
                };
                auto weights = [&](auto is_masked, int c, const uint32_t (&d)[32], float m) {
                    const uint32_t seen = is_masked.value ? seen_of(c) : 0u;
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const float f = sc.k[2 * c + k] * unit, off = sc.log_v[2 * c + k] - m;
                        const uint64_t ff = pp_pair(f, f), oo = pp_pair(off, off);
                        uint64_t sum = 0ull;
                        uint32_t hi[8];
                        [[maybe_unused]] uint32_t rest[NP == 2 ? 8 : 1];
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const int at = 8 * k + i;
                            const float2 e = pp_unpair(pp_fma2(pp_pair(__uint_as_float(d[2 * at]), __uint_as_float(d[2 * at + 1])), ff, oo));
                            float p0 = ex2_approx(e.x), p1 = ex2_approx(e.y);
                            if (is_masked.value) {  // (a scale of 0 makes 0 * -infinity of what is masked)
                                p0 = (seen & (1u << (2 * at))) != 0u ? p0 : 0.0f;
                                p1 = (seen & (2u << (2 * at))) != 0u ? p1 : 0.0f;
                            }
                            const uint64_t pp = pp_pair(p0, p1);
                            sum = pp_add2(sum, pp);
                            hi[i] = pp_round(p0, p1);
                            if constexpr (NP == 2) {
                                const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&hi[i]));
                                const float2 x = pp_unpair(pp_fma2(pp_pair(y.x, y.y), pp_pair(-1.0f, -1.0f), pp));
                                rest[i] = pp_round(x.x, x.y);
                            }
                        }
                        const float2 both = pp_unpair(sum);
                        l = fmaf(both.x + both.y, sc.inv_v[2 * c + k], l);
                        tmem_store_x8(ts + c * 32 + k * 8, hi);
                        if constexpr (NP == 2) tmem_store_x8(ts + c * 32 + 16 + k * 8, rest);
                    }
                };
                auto tile = [&](auto is_masked) {
                    const bool fresh = n == 0 || (drains && n % kPpDrain == 0);  // O begins anew with this tile
                    if (fresh && n > 0) {
                        ok = warp_wait(&pv_done[stream], (uint32_t)(n - 1) & 1u);
                        if (!ok) return;
                        tcgen05_fence_after();
                        drain();
                    }
                    uint32_t d[32];
                    tmem_load_x32(ts + half * 64, d);
                    float top = largest(is_masked, 2 * half, d);
                    tmem_load_x32(ts + half * 64 + 32, d);
                    top = fmaxf(top, largest(is_masked, 2 * half + 1, d));
                    // (two buffers: a thread writes the next value of this one behind a barrier that its partner reaches after it has read)
                    float* const at = tops + (n & 1) * 4 * kPpRows;
                    at[half * kPpRows] = top;
                    __syncwarp();
                    if (lane == 0) mbar_arrive(pair_bar);
                    ok = warp_wait(pair_bar, (uint32_t)n & 1u);
                    if (!ok) return;
                    top = fmaxf(top, at[(half ^ 1) * kPpRows]);
                    const bool grow = top > m_ref + kPpLag;  // (a row with nothing attended so far has -inf)
                    if (__any_sync(0xffffffffu, grow)) {
                        const float corr = grow ? ex2_approx(m_ref - top) : 1.0f;
                        if (grow) m_ref = top;
                        l *= corr;
                        if (!fresh) {  // half of the columns of O each
                            ok = warp_wait(&pv_done[stream], (uint32_t)(n - 1) & 1u);
                            if (!ok) return;
                            tcgen05_fence_after();
#pragma unroll 1
                            for (int i = half * (HD / 32); i < (half + 1) * (HD / 32); ++i) {
                                uint32_t o[16];
                                tmem_load_x16(to + i * 16, o);
#pragma unroll
                                for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * corr);
                                tmem_store_x16(to + i * 16, o);
                            }
                        }
                    }
                    const float m = (m_ref == -INFINITY ? 0.0f : m_ref) - kPpRoom;
                    weights(is_masked, 2 * half + 1, d, m);
                    tmem_load_x32(ts + half * 64, d);
                    weights(is_masked, 2 * half, d, m);
                };
                if (masked) tile(std::true_type());
                else tile(std::false_type());
                if (!ok) break;
                tmem_store_wait();
                tcgen05_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_ready[stream]);
            }
            if (ok && n > 0) ok = warp_wait(&pv_done[stream], (uint32_t)(n - 1) & 1u);
            if (drains && n > kPpDrain) __threadfence();
            // ---- the sum of both threads of a row; where the streams are shares of the keys, maximum and sum over both
            float4* const stat = reinterpret_cast<float4*>(smem + S::kOffStat);  // [stream][half][row]
            stat[(stream * 2 + half) * kPpRows + r] = make_float4(m_ref, l, drains && n > kPpDrain ? ex2_approx(drained_ref == -INFINITY ? -INFINITY : drained_ref - m_ref) : 0.0f, 0.0f);
            tcgen05_fence_before();
            asm volatile("bar.sync 1, 512;" ::: "memory");
            tcgen05_fence_after();
            const float m0 = stat[r].x, m1 = stat[2 * kPpRows + r].x, l0 = stat[r].y + stat[kPpRows + r].y, l1 = stat[2 * kPpRows + r].y + stat[3 * kPpRows + r].y;
            const float m = fmaxf(m0, m1), mm = m == -INFINITY ? 0.0f : m;
            const float w0 = ex2_approx(m0 - mm), w1 = ex2_approx(m1 - mm), sum = two ? (stream == 0 ? l0 : l1) : l0 * w0 + l1 * w1, inv = sum == 0.0f ? 0.0f : 1.0f / sum;
            const float whole = parts > 1 ? 1.0f : inv, f0 = two ? whole : w0 * whole, f1 = w1 * whole;
            const bool any0 = two ? n > 0 : tiles > 0, any1 = !two && tiles > 1;
            // what left tensor memory earlier, relative to the maximum of its stream
            const bool sums0 = drains && (two ? n : (tiles + 1) / 2) > kPpDrain, sums1 = drains && !two && tiles / 2 > kPpDrain;
            const float g0 = f0 * stat[(two ? stream * 2 : 0) * kPpRows + r].z, g1 = f1 * stat[2 * kPpRows + r].z;
            float* const partial = work.partials + (size_t)((entry.w + part) * a.kv_heads + h) * pp_partial_floats<HD>();
            if (parts > 1 && half == 0 && (two || stream == 0)) reinterpret_cast<float2*>(partial)[two ? in_unit : r] = make_float2(two ? m_ref : m, sum);
            // half of the columns each: of the stream's rows, or (one tile of rows) a quarter for each of the four warps
            const int columns = two ? HD / 2 : HD / 4, from = two ? half * columns : (stream * 2 + half) * columns;
            // the last MMAs are done and nobody loads: the rows leave over the operands' shared memory, so that a warp writes whole runs
            float* const stage = reinterpret_cast<float*>(smem) + warp * 32 * S::kStagePitch;
#pragma unroll 1
            for (int c = 0; c < columns; c += 16) {
                uint32_t d[16], e[16];
                const uint32_t col = rows + kPpTmemO + (uint32_t)((two ? stream * 128 : 0) + from + c);
                if (any0) tmem_load_x16(col, d);
                if (any1) tmem_load_x16(col + 128u, e);
#pragma unroll
                for (int i = 0; i < 16; i += 4) {
                    float y[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        y[k] = any0 ? __uint_as_float(d[i + k]) * f0 : 0.0f;
                        if (any1) y[k] = fmaf(__uint_as_float(e[i + k]), f1, y[k]);
                    }
                    if (sums0) {
                        const float4 x = __ldcg(sums_of(two ? stream : 0, from + c + i));
                        y[0] = fmaf(x.x, g0, y[0]); y[1] = fmaf(x.y, g0, y[1]); y[2] = fmaf(x.z, g0, y[2]); y[3] = fmaf(x.w, g0, y[3]);
                    }
                    if (sums1) {
                        const float4 x = __ldcg(sums_of(1, from + c + i));
                        y[0] = fmaf(x.x, g1, y[0]); y[1] = fmaf(x.y, g1, y[1]); y[2] = fmaf(x.z, g1, y[2]); y[3] = fmaf(x.w, g1, y[3]);
                    }
                    *reinterpret_cast<float4*>(stage + lane * S::kStagePitch + c + i) = make_float4(y[0], y[1], y[2], y[3]);
                }
            }
            __syncwarp();
            const int quads_log = (HD == 128 ? 5 : 4) - (two ? 1 : 2);  // groups of four columns
#pragma unroll 4
            for (int i = lane; i < 32 << quads_log; i += 32) {
                const int rr = i >> quads_log, c4 = i & ((1 << quads_log) - 1), row = (two ? stream * kPpRows : 0) + (warp & 3) * 32 + rr;
                if (!ok || row >= live) continue;
                const float4 y = *reinterpret_cast<const float4*>(stage + rr * S::kStagePitch + c4 * 4);
                if (parts > 1) {
                    *reinterpret_cast<float4*>(partial + 2 * kPpUnit + row * HD + from + c4 * 4) = y;
                    continue;
                }
                T* const out = static_cast<T*>(a.out) + (size_t)row_of[row] * HD + from + c4 * 4;
                if constexpr (sizeof(T) == 4) {
                    *reinterpret_cast<float4*>(out) = y;
                } else {
                    *reinterpret_cast<uint2*>(out) = make_uint2(bf16_pair_of(y.x, y.y), bf16_pair_of(y.z, y.w));
                }
            }
            if (parts > 1) {
                __threadfence();
                asm volatile("bar.sync 1, 512;" ::: "memory");
                int* const arrived = work.arrived + entry.w * a.kv_heads + h;
                if (tid == 0) *s_last = atomicAdd(arrived, 1) == parts - 1;
                asm volatile("bar.sync 1, 512;" ::: "memory");
                if (*s_last != 0) {
                    __threadfence();
                    if (tid == 0) *arrived = 0;
                    const float* const p0 = work.partials + (size_t)(entry.w * a.kv_heads + h) * pp_partial_floats<HD>();
                    const size_t pitch = (size_t)a.kv_heads * pp_partial_floats<HD>();
                    // 2^(maximum - largest) / sum of every part of a row, over the operands
                    float* const factor = reinterpret_cast<float*>(smem);
                    if (tid < live) {
                        float top = -INFINITY, all = 0.0f;
                        for (int k = 0; k < parts; ++k) top = fmaxf(top, __ldcg(p0 + k * pitch + 2 * tid));
                        const float base_top = top == -INFINITY ? 0.0f : top;
                        for (int k = 0; k < parts; ++k) {
                            const float2 st = __ldcg(reinterpret_cast<const float2*>(p0 + k * pitch) + tid);
                            all = fmaf(st.y, ex2_approx(st.x - base_top), all);
                        }
                        const float over = all == 0.0f ? 0.0f : 1.0f / all;
                        for (int k = 0; k < parts; ++k) factor[k * kPpUnit + tid] = ex2_approx(__ldcg(p0 + k * pitch + 2 * tid) - base_top) * over;
                    }
                    asm volatile("bar.sync 1, 512;" ::: "memory");
#pragma unroll 4
                    for (int i = tid; i < live * (HD / 4); i += 512) {
                        const int row = i / (HD / 4), c = i % (HD / 4) * 4;
                        const float* const x0 = p0 + 2 * kPpUnit + row * HD + c;
                        float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                        for (int k = 0; k < parts; ++k) {
                            const float4 x = __ldcg(reinterpret_cast<const float4*>(x0 + k * pitch));
                            const float f = factor[k * kPpUnit + row];
                            y.x = fmaf(x.x, f, y.x); y.y = fmaf(x.y, f, y.y); y.z = fmaf(x.z, f, y.z); y.w = fmaf(x.w, f, y.w);
                        }
                        T* const out = static_cast<T*>(a.out) + (size_t)row_of[row] * HD + c;
                        if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(out) = y;
                        else *reinterpret_cast<uint2*>(out) = make_uint2(bf16_pair_of(y.x, y.y), bf16_pair_of(y.z, y.w));
                    }
                }
            }
        }
    }
    if (!ok) atomicCAS(&g_paged_prompt_status, 0, 1);
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    if (drains && tid == 0 && s_place >= 0) {  // (all have written and read their sums)
        __threadfence();
        atomicAnd(&work.taken[s_place / 32], ~(1u << s_place % 32));
    }
    if (warp == kPpIssue) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(*tmem_slot), "r"(512u) : "memory");
}

}  // namespace

namespace {
long long pp_units(int heads, int kv_heads, int requests, int tokens) {  // each request ends in a unit of its own
    return ((long long)tokens * (heads / kv_heads) + kPpUnit - 1) / kPpUnit + requests;
}
int pp_capacity(int heads, int kv_heads, int requests, int tokens) {
    const long long n = pp_units(heads, kv_heads, requests, tokens) + kPpSplitBlocks / kv_heads;
    return (int)(n < 65535 ? n : 65535);
}
size_t pp_list_bytes(int capacity) { return ((size_t)(1 + capacity) * sizeof(int4) + 255) / 256 * 256; }
size_t pp_partial_bytes(int head_dim) { return kPpSplitBlocks * sizeof(float) * (size_t)kPpUnit * (head_dim + 2); }
}  // namespace

bool paged_prompt_serves(const PagedArgs& a) {
    return (a.head_dim == 64 || a.head_dim == 128) && ((reinterpret_cast<uintptr_t>(a.query) | reinterpret_cast<uintptr_t>(a.out)) & 15u) == 0;
}

bool paged_prompt_fits(const PagedArgs& a) {
    return pp_units(a.heads, a.kv_heads, a.requests, a.tokens) <= 65535 && (long long)a.tokens * a.heads <= INT_MAX;
}
size_t paged_prompt_scratch_bytes(int heads, int kv_heads, int head_dim, int requests, int tokens) {
    return pp_list_bytes(pp_capacity(heads, kv_heads, requests, tokens)) + pp_partial_bytes(head_dim) +
           kPpSums * sizeof(float) * (size_t)kPpUnit * head_dim;
}

PagedOrder paged_prompt_order(const PagedArgs& a, void* scratch) {
    return PagedOrder{static_cast<int4*>(scratch), pp_capacity(a.heads, a.kv_heads, a.requests, a.tokens), kPpSplitBlocks};
}

int paged_prompt_launch(cudaStream_t stream, const PagedArgs& a, bool f32, int* arrived, void* scratch) {
    const int capacity = pp_capacity(a.heads, a.kv_heads, a.requests, a.tokens);
    unsigned char* const at = static_cast<unsigned char*>(scratch) + pp_list_bytes(capacity);
    const PpWork work = {static_cast<const int4*>(scratch), arrived, reinterpret_cast<uint32_t*>(arrived + kPpSplitBlocks), reinterpret_cast<float*>(at), reinterpret_cast<float*>(at + pp_partial_bytes(a.head_dim))};
    auto go = [&](auto kern, int smem) {
        cudaFuncAttributes fa;
        cudaError_t e = cudaFuncGetAttributes(&fa, kern);
        if (e == cudaSuccess && fa.numRegs < kPpRegsLaunch) e = cudaErrorInvalidDeviceFunction;  // (the warpgroups would wait for registers that the block does not have)
        if (e == cudaSuccess) e = allow_all_dynamic_smem(kern);
        return e != cudaSuccess ? e : launch(kern, dim3(a.kv_heads, (unsigned)capacity), dim3(kPpThreads), (size_t)smem, stream, true, a, work);
    };
    cudaError_t e;
    if (a.head_dim == 128) e = f32 ? go(paged_prompt_kernel<128, float>, PpShape<128, 2>::kSmemBytes) : go(paged_prompt_kernel<128, uint16_t>, PpShape<128, 1>::kSmemBytes);
    else e = f32 ? go(paged_prompt_kernel<64, float>, PpShape<64, 2>::kSmemBytes) : go(paged_prompt_kernel<64, uint16_t>, PpShape<64, 1>::kSmemBytes);
    if (e != cudaSuccess) return fail(KMLL_ERR_CUDA, "paged attention: %s", cudaGetErrorString(e));
    return KMLL_OK;
}

int paged_prompt_status(int* status_out) {
    const cudaError_t e = cudaMemcpyFromSymbol(status_out, g_paged_prompt_status, sizeof(int));
    if (e != cudaSuccess) return fail(KMLL_ERR_CUDA, "device_status: %s", cudaGetErrorString(e));
    return KMLL_OK;
}

}  // namespace kmll
