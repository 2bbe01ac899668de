// Attention of portions of prompts over the paged 8-bit cache on tcgen05: one block = 128 rows of a request and kv head.
//
// A row is a (token, query head) pair: all query heads of a kv head are in the same block, so codes are turned into operands once for all of
// them, and short portions still fill the 128 rows.  Codes are exact in binary16, which is what both contractions run on:
//   S = Q K^T    Q as x * 2^sh = x0 + x1, two binary16 planes (f32 rows: 2^-22 of the row's largest entry) or one (bf16 rows: exact down to 2^-24 of
//                it); times k_scale of the key's page and 2^-sh
//   O += P V     the value scale of a key's page goes into the exponent, P = 2^(s + log2 v_scale - m): no multiplication, and the sum of the
//                weights takes 1 / v_scale once per group of 16 keys.  P is two planes (f32 rows) or one (bf16 rows: 2^-12, below the rounding of
//                the result).  A maximum is one of s + log2 v_scale; page scales of a head may differ by 2^100.
// Roles of the 13 warps:
//   warps 0-3, 4-7  softmax of the even and of the odd key tiles (128 keys), a thread per row: scores by tcgen05.ld, once for the maximum, once
//                   for the weights, which go back in the place of the scores they came from.  Two independent streams (maximum, sum, O), merged at the end
//   warps 8-11      fetch the codes of a tile into registers while the tile before is at work, and write them as binary16 operands (128-byte
//                   swizzle, both K-major: values lie with the keys of a column together)
//   warp 12         issues S = Q K^T and O += P V
// O is rescaled only when a row's maximum has grown by more than 2^8.  Every wait is bounded; a time-out raises the status word, and the block frees
// its tensor memory and returns (no copies are under way: the fetches are loads).
#include <climits>
#include <type_traits>

#include "internal.cuh"
#include "mma_bf16.cuh"
#include "paged.cuh"
#include "tcgen05.cuh"

namespace kmll {

__device__ int g_paged_prompt_status = 0;

namespace {

constexpr int kPpRows = 128, kPpKeys = 128, kPpGroups = kPpKeys / 16;
constexpr int kPpThreads = 13 * 32;
constexpr int kPpBox = 128 * 128;      // 128 rows of 64 binary16 entries
constexpr uint32_t kPpTmemO = 256;     // scores at 0 and 128, the streams' O behind them

struct PpScales {  // of a tile, per group of 16 keys
    float k[kPpGroups], log_v[kPpGroups], inv_v[kPpGroups];
    uint32_t there, unused[7];
};

// NP: planes of Q and of P
template <int HD, int NP>
struct PpShape {
    static constexpr int kQPlane = kPpRows * HD * 2, kK = kPpKeys * HD * 2, kVBox = HD * 128, kV = 2 * kVBox;
    static constexpr int kOffK = NP * kQPlane, kOffV = kOffK + 2 * kK, kOffScales = kOffV + 2 * kV;
    static constexpr int kOffStat = kOffScales + 4 * (int)sizeof(PpScales), kOffUnit = kOffStat + 2 * kPpRows * 8;
    static constexpr int kOffBars = kOffUnit + kPpRows * 8;
    static constexpr int kSmemBytes = kOffBars + 256 + 1024;
    static constexpr int kStagePitch = HD / 2 + 4;
    static_assert(kSmemBytes <= 227 * 1024 && 8 * 32 * kStagePitch * 4 <= kOffScales, "shape");
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

template <int HD, typename T>
__global__ void __launch_bounds__(kPpThreads, 1) paged_prompt_kernel(const PagedArgs a) {
    constexpr int NP = sizeof(T) == 4 ? 2 : 1;
    using S = PpShape<HD, NP>;
    extern __shared__ unsigned char pp_smem_raw[];
    unsigned char* const smem = pp_smem_raw + ((1024u - (smem_u32(pp_smem_raw) & 1023u)) & 1023u);
    uint64_t* const s_full = reinterpret_cast<uint64_t*>(smem + S::kOffBars);  // [2] the scores of a tile are there
    uint64_t* const p_ready = s_full + 2;    // [2] its weights are there (and O is rescaled)
    uint64_t* const pv_done = p_ready + 2;   // [2] O has taken the tile
    uint64_t* const k_full = pv_done + 2;    // [2]
    uint64_t* const v_full = k_full + 2;     // [2]
    uint64_t* const sc_full = v_full + 2;    // [4] the scales of a tile are there
    uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(sc_full + 4);
    int* const s_unit = reinterpret_cast<int*>(tmem_slot + 1);  // request, tile of 128 rows
    PpScales* const scales = reinterpret_cast<PpScales*>(smem + S::kOffScales);
    float* const units = reinterpret_cast<float*>(smem + S::kOffUnit);
    int* const row_of = reinterpret_cast<int*>(units + kPpRows);  // rows of the block among the step's (token, head) rows
    const int tid = threadIdx.x, lane = tid & 31, warp = uniform_warp_index(), group = a.heads / a.kv_heads, h = blockIdx.y, block_log = 31 - __clz(a.block), in_block = a.block - 1;
    if (tid == 0) {
        for (int b = 0; b < 2; ++b) {
            mbar_init(&s_full[b], 1);
            mbar_init(&p_ready[b], 4);
            mbar_init(&pv_done[b], 1);
            mbar_init(&k_full[b], 4);
            mbar_init(&v_full[b], 4);
        }
        for (int b = 0; b < 4; ++b) mbar_init(&sc_full[b], 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        s_unit[0] = -1;
    }
    if (warp == 12) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tcgen05_fence_before();
    __syncthreads();  // (columns first, then the dependents: tcgen05.cuh)
    tcgen05_fence_after();
    pdl_wait();
    // ---- the block's request and rows: tiles of 128 rows, request after request, the last rows of a request (which see most) first
    if (warp == 0) {
        int before = 0;
        for (int r0 = 0; r0 < a.requests; r0 += 32) {
            const int r = r0 + lane;
            int n = 0;
            if (r < a.requests) {
                const long long rows = (long long)PagedRequest::of(a, r).rows * group;
                n = rows > a.skip_rows ? (int)((rows + kPpRows - 1) / kPpRows) : 0;
            }
            int up = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, up, o);
                if (lane >= o) up += v;
            }
            const int at = (int)blockIdx.x - before - (up - n);
            if (n > 0 && at >= 0 && at < n) {
                s_unit[0] = r;
                s_unit[1] = n - 1 - at;
            }
            before += __shfl_sync(0xffffffffu, up, 31);
            if ((int)blockIdx.x < before) break;
        }
    }
    __syncthreads();
    const int request = s_unit[0];
    bool ok = true;
    if (request >= 0) {
        const PagedRequest rq = PagedRequest::of(a, request);
        const int row0 = s_unit[1] * kPpRows, live = min(kPpRows, rq.rows * group - row0);
        const int first_pos = rq.pos0 + row0 / group, last_pos = min(rq.pos0 + (row0 + live - 1) / group, rq.hi - 1);
        const int last_own = rq.pos0 + (row0 + live - 1) / group;  // (a context longer than its table row is cut at the table's end)
        const int low = a.window > 0 ? max(0, first_pos - a.window + 1) : 0, first = low & ~15;
        const int tiles = last_pos >= low ? (last_pos - first) / kPpKeys + 1 : 0;
        // ---- Q: a warp has a row at a time, HD / 32 entries a lane; its largest entry gives the power of two
        constexpr int E = HD / 32, kWarps = kPpThreads / 32, kOwn = (kPpRows + kWarps - 1) / kWarps;
        float x[kOwn][E];
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
            const int r = warp + i * kWarps;
#pragma unroll
            for (int k = 0; k < E; ++k) x[i][k] = 0.0f;
            if (r >= kPpRows) continue;
            const int token = (row0 + r) / group, place = (rq.first + token) * a.heads + h * group + (row0 + r - token * group);
            if (lane == 0) row_of[r] = place;
            if (r < live) load_entries<E>(static_cast<const T*>(a.query) + (size_t)place * HD + lane * E, x[i]);
        }
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
            const int r = warp + i * kWarps;
            if (r >= kPpRows) continue;
            float top = 0.0f;
            bool finite = true;
#pragma unroll
            for (int k = 0; k < E; ++k) {
                top = fmaxf(top, fabsf(x[i][k]));
                finite = finite && fabsf(x[i][k]) < INFINITY;
            }
            top = warp_max(top);
            int e2 = 0;
            if (top > 0.0f && top < INFINITY) frexpf(top, &e2);
            const float up = ldexpf(1.0f, max(-120, min(120, 11 - e2)));  // the largest entry between 2^10 and 2^11
            if (lane == 0) units[r] = up;
            if (!__all_sync(0xffffffffu, finite) && lane == 0) units[r] = __int_as_float(0x7fffffff);
            unsigned char* const at = smem + (lane * E >> 6) * kPpBox + r * 128 + ((((lane * E >> 3) & 7) ^ (r & 7)) << 4) + (lane * E & 7) * 2;
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
        fence_proxy_async_smem();
        __syncthreads();
        const uint32_t base = smem_u32(smem);

        if (warp >= 8 && warp < 12) {
            // ---- codes to operands
            const int tt = tid - 256;  // 0 .. 127: the key; of the values the group of 16 keys tt / 16, columns tt % 16, + 16, ..
            const int32_t* const table = a.table + (size_t)request * a.width;
            constexpr int U = HD / 16;  // 16-byte groups of a key; columns of a group of values per thread
            uint4 kc[U], vc[U];
            auto entry_of = [&](int j) {  // lanes 0-7 (and again): table entry of group lane & 7 of tile j; looked at a tile later, when it has come
                const int key = first + j * kPpKeys + (lane & 7) * 16;
                int p = -1;
                if (j < tiles && key < rq.hi) p = table[key >> block_log];
                return p;
            };
            auto page_of = [&](int entry) { return entry >= 0 && entry < a.pages ? entry : -1; };  // -1: nothing there
            // (volatile loads: they stay where they are written, a tile ahead of their use; where nothing is there any codes do, no row sees them)
            // One page per thread and tile: more shuffles between the loads would share their scoreboards and wait for them.
            auto fetch_keys = [&](int j, int p) {
                const uint4* const src = reinterpret_cast<const uint4*>(a.k_codes + ((size_t)max(p, 0) * a.kv_heads + h) * a.block * HD) + ((first + j * kPpKeys + tt) & in_block);
#pragma unroll
                for (int c = 0; c < U; ++c) kc[c] = ld_stream_u4(src + (size_t)c * a.block);
            };
            auto fetch_values = [&](int j, int p) {
                const uint4* const src = reinterpret_cast<const uint4*>(a.v_codes + ((size_t)max(p, 0) * a.kv_heads + h) * a.block * HD) +
                                         (size_t)(((first + j * kPpKeys + (tt & ~15)) & in_block) >> 4) * HD + (tt & 15);
#pragma unroll
                for (int c = 0; c < U; ++c) vc[c] = ld_stream_u4(src + c * 16);
            };
            int page = page_of(entry_of(0)), entry = entry_of(1);
            float ks = 0.0f, vs = 0.0f;  // lanes 0-7 of warp 8: scales of the tile in kc
            auto fetch_scales = [&](int p) {
                if (warp == 8 && lane < 8) {
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
                const int st = j & 1, before = j - 2;
                ok = before < 0 || warp_wait(&s_full[st], (uint32_t)(before >> 1) & 1u);
                if (!ok) break;
                if (warp == 8) {
                    PpScales& sc = scales[j & 3];
                    if (lane < 8) {
                        sc.k[lane] = ks;
                        sc.log_v[lane] = vs > 0.0f ? log2f(vs) : page >= 0 ? -40.0f : 0.0f;
                        sc.inv_v[lane] = vs > 0.0f ? 1.0f / vs : page >= 0 ? 0x1p40f : 0.0f;
                    }
                    const uint32_t there = __ballot_sync(0xffffffffu, page >= 0) & 0xffu;
                    if (lane == 0) sc.there = there;
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sc_full[j & 3]);
                }
                unsigned char* const krow = smem + S::kOffK + st * S::kK + tt * 128;
#pragma unroll
                for (int c = 0; c < U; ++c) pp_put(krow + (c >> 2) * kPpBox, (c & 3) * 2, tt & 7, kc[c]);
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&k_full[st]);
                const int next = page_of(entry), p_next = __shfl_sync(0xffffffffu, next, tt >> 4);
                if (j + 1 < tiles) {
                    fetch_scales(next);
                    fetch_keys(j + 1, p_next);
                }
                ok = before < 0 || warp_wait(&pv_done[st], (uint32_t)(before >> 1) & 1u);
                if (!ok) break;
                unsigned char* const vrow = smem + S::kOffV + st * S::kV + (tt >> 6) * S::kVBox + (tt & 15) * 128;
#pragma unroll
                for (int c = 0; c < U; ++c) pp_put(vrow + c * 2048, ((tt >> 4) & 3) * 2, tt & 7, vc[c]);
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&v_full[st]);
                if (j + 1 < tiles) fetch_values(j + 1, p_next);
                page = next;
                entry = entry_of(j + 2);
            }
        } else if (warp == 12) {
            constexpr uint32_t idesc_s = gemm_idesc_f16(128, kPpKeys), idesc_o = gemm_idesc_f16(128, HD);
            const uint64_t dq = gemm_smem_desc(base), dk = gemm_smem_desc(base + S::kOffK), dv = gemm_smem_desc(base + S::kOffV);
            const uint32_t lead = elect_lead();
            auto scores = [&](int j) {
                const int st = j & 1;
                if (!warp_wait(&k_full[st], (uint32_t)(j >> 1) & 1u)) return false;
                tcgen05_fence_after();
                const uint64_t dkj = dk + (uint64_t)(st * (S::kK >> 4));
                uint32_t acc = 0u;
#pragma unroll
                for (int p = NP - 1; p >= 0; --p)  // the small products first
#pragma unroll
                    for (int ks = 0; ks < HD / 16; ++ks) {
                        const int at = (ks >> 2) * kPpBox + (ks & 3) * 32;
                        lead_mma_f16(lead, (uint32_t)st * 128u, dq + (uint64_t)((p * S::kQPlane + at) >> 4), dkj + (uint64_t)(at >> 4), idesc_s, acc);
                        acc = 1u;
                    }
                lead_commit(lead, &s_full[st]);
                return true;
            };
            if (tiles > 0) ok = scores(0) && (tiles < 2 || scores(1));
            for (int j = 0; j < tiles && ok; ++j) {
                const int st = j & 1;
                ok = warp_wait(&v_full[st], (uint32_t)(j >> 1) & 1u) && warp_wait(&p_ready[st], (uint32_t)(j >> 1) & 1u);
                if (!ok) break;
                tcgen05_fence_after();
                const uint64_t dvj = dv + (uint64_t)(st * (S::kV >> 4));
                uint32_t acc = j >= 2 ? 1u : 0u;
#pragma unroll
                for (int p = NP - 1; p >= 0; --p)
#pragma unroll
                    for (int ks = 0; ks < kPpKeys / 16; ++ks) {  // weights of 32 keys: 16 columns of the first plane, 16 of the second
                        lead_mma_f16_ts(lead, kPpTmemO + (uint32_t)st * 128u, (uint32_t)(st * 128 + (ks >> 1) * 32 + p * 16 + (ks & 1) * 8),
                                        dvj + (uint64_t)(((ks >> 2) * S::kVBox + (ks & 3) * 32) >> 4), idesc_o, acc);
                        acc = 1u;
                    }
                lead_commit(lead, &pv_done[st]);
                if (j + 2 < tiles) ok = scores(j + 2);
            }
        } else {
            // ---- softmax of the tiles j = stream, stream + 2, ..
            const int stream = warp >> 2, r = (warp & 3) * 32 + lane, own = rq.pos0 + (row0 + r) / group;
            const int pos = min(own, rq.hi - 1), lo = a.window > 0 ? own - a.window + 1 : 0;
            const float unit = a.scale2 / units[r];  // (a row with an infinity or NaN has no scores)
            const uint32_t rows = (uint32_t)((warp & 3) * 32) << 16;
            const uint32_t ts = rows + (uint32_t)stream * 128u, to = rows + kPpTmemO + (uint32_t)stream * 128u;
            float m_ref = -INFINITY, l = 0.0f;
            int n = 0;  // tiles of this stream so far
            for (int j = stream; j < tiles; j += 2, ++n) {
                const int t0 = first + j * kPpKeys;
                ok = warp_wait(&sc_full[j & 3], (uint32_t)(j >> 2) & 1u) && warp_wait(&s_full[stream], (uint32_t)n & 1u);
                if (!ok) break;
                tcgen05_fence_after();
                const PpScales& sc = scales[j & 3];
                const bool masked = t0 + kPpKeys - 1 > first_pos || t0 < low || (a.window > 0 && t0 < last_own - a.window + 1) || sc.there != 0xffu;
                // keys of chunk c that the row attends, a bit each
                auto seen_of = [&](int c) {
                    const int k0 = t0 + c * 32, from = max(lo - k0, 0), to = min(pos - k0, 31);
                    const uint32_t pair = sc.there >> (2 * c);
                    const uint32_t there = (pair & 1u ? 0xffffu : 0u) | (pair & 2u ? 0xffff0000u : 0u);
                    return from <= to ? (0xffffffffu << from) & (0xffffffffu >> (31 - to)) & there : 0u;
                };
                float top = -INFINITY;
                auto largest = [&](auto is_masked) {
#pragma unroll 1
                    for (int c = 0; c < kPpKeys / 32; ++c) {
                        uint32_t d[32];
                        tmem_load_x32(ts + c * 32, d);
                        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                        const uint32_t seen = is_masked.value ? seen_of(c) : 0u;
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            mx[(i >> 4) * 2 + (i & 1)] = fmaxf(mx[(i >> 4) * 2 + (i & 1)], is_masked.value && (seen & (1u << i)) == 0u ? -INFINITY : __uint_as_float(d[i]));
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            const float x = fmaxf(mx[2 * k], mx[2 * k + 1]);
                            if (x > -INFINITY) top = fmaxf(top, fmaf(x, sc.k[2 * c + k] * unit, sc.log_v[2 * c + k]));
                        }
                    }
                };
                if (masked) largest(std::true_type());
                else largest(std::false_type());
                const bool grow = top > m_ref + 8.0f;  // (a row with nothing attended so far has -inf)
                if (__any_sync(0xffffffffu, grow)) {
                    const float corr = grow ? ex2_approx(m_ref - top) : 1.0f;
                    if (grow) m_ref = top;
                    l *= corr;
                    if (n > 0) {
                        ok = warp_wait(&pv_done[stream], (uint32_t)(n - 1) & 1u);
                        if (!ok) break;
                        tcgen05_fence_after();
#pragma unroll
                        for (int c = 0; c < HD / 32; ++c) {
                            uint32_t d[32];
                            tmem_load_x32(to + c * 32, d);
#pragma unroll
                            for (int i = 0; i < 32; ++i) d[i] = __float_as_uint(__uint_as_float(d[i]) * corr);
                            tmem_store_x32(to + c * 32, d);
                        }
                    }
                }
                const float m = m_ref == -INFINITY ? 0.0f : m_ref;
                auto weights = [&](auto is_masked) {
#pragma unroll 1
                    for (int c = 0; c < kPpKeys / 32; ++c) {
                        uint32_t d[32], planes[NP * 16];
                        tmem_load_x32(ts + c * 32, d);
                        const uint32_t seen = is_masked.value ? seen_of(c) : 0u;
                        float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                        const float f[2] = {sc.k[2 * c] * unit, sc.k[2 * c + 1] * unit}, off[2] = {sc.log_v[2 * c] - m, sc.log_v[2 * c + 1] - m};
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const int k = i >> 3;
                            float p0 = ex2_approx(fmaf(__uint_as_float(d[2 * i]), f[k], off[k])), p1 = ex2_approx(fmaf(__uint_as_float(d[2 * i + 1]), f[k], off[k]));
                            if (is_masked.value) {
                                p0 = (seen & (1u << (2 * i))) != 0u ? p0 : 0.0f;
                                p1 = (seen & (2u << (2 * i))) != 0u ? p1 : 0.0f;
                            }
                            sum[2 * k] += p0;
                            sum[2 * k + 1] += p1;
                            planes[i] = pp_round(p0, p1);
                            if constexpr (NP == 2) planes[16 + i] = pp_rest(p0, p1, planes[i]);
                        }
                        l = fmaf(sum[0] + sum[1], sc.inv_v[2 * c], l);
                        l = fmaf(sum[2] + sum[3], sc.inv_v[2 * c + 1], l);
                        if constexpr (NP == 2) tmem_store_x32(ts + c * 32, planes);
                        else tmem_store_x16(ts + c * 32, planes);
                    }
                };
                if (masked) weights(std::true_type());
                else weights(std::false_type());
                tmem_store_wait();
                tcgen05_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_ready[stream]);
            }
            if (ok && n > 0) ok = warp_wait(&pv_done[stream], (uint32_t)(n - 1) & 1u);
            // ---- both streams of a row, then half of its columns per stream's warps
            float2* const stat = reinterpret_cast<float2*>(smem + S::kOffStat);
            stat[stream * kPpRows + r] = make_float2(m_ref, l);
            tcgen05_fence_before();
            asm volatile("bar.sync 1, 256;" ::: "memory");
            tcgen05_fence_after();
            const float2 st0 = stat[r], st1 = stat[kPpRows + r];
            const float m = fmaxf(st0.x, st1.x), mm = m == -INFINITY ? 0.0f : m;
            const float w0 = ex2_approx(st0.x - mm), w1 = ex2_approx(st1.x - mm), sum = st0.y * w0 + st1.y * w1, inv = sum == 0.0f ? 0.0f : 1.0f / sum;
            const float f0 = w0 * inv, f1 = w1 * inv;
            // the last MMAs are done and nobody loads: the rows leave over the operands' shared memory, so that a warp writes whole runs
            float* const stage = reinterpret_cast<float*>(smem) + warp * 32 * S::kStagePitch;
#pragma unroll
            for (int c = 0; c < HD / 64; ++c) {
                uint32_t d[32], e[32];
                const uint32_t col = rows + kPpTmemO + (uint32_t)(stream * (HD / 2) + c * 32);
                if (tiles > 0) tmem_load_x32(col, d);
                if (tiles > 1) tmem_load_x32(col + 128u, e);
#pragma unroll
                for (int i = 0; i < 32; i += 4) {
                    float y[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        y[k] = tiles > 0 ? __uint_as_float(d[i + k]) * f0 : 0.0f;
                        if (tiles > 1) y[k] = fmaf(__uint_as_float(e[i + k]), f1, y[k]);
                    }
                    *reinterpret_cast<float4*>(stage + lane * S::kStagePitch + c * 32 + i) = make_float4(y[0], y[1], y[2], y[3]);
                }
            }
            __syncwarp();
            for (int i = lane; i < 32 * (HD / 8); i += 32) {
                const int rr = i / (HD / 8), c4 = i - rr * (HD / 8), row = (warp & 3) * 32 + rr;
                if (!ok || row >= live) continue;
                T* const out = static_cast<T*>(a.out) + (size_t)row_of[row] * HD + stream * (HD / 2) + c4 * 4;
                const float4 y = *reinterpret_cast<const float4*>(stage + rr * S::kStagePitch + c4 * 4);
                if constexpr (sizeof(T) == 4) {
                    *reinterpret_cast<float4*>(out) = y;
                } else {
                    *reinterpret_cast<uint2*>(out) = make_uint2(f32_to_bf16_bits(y.x) | ((uint32_t)f32_to_bf16_bits(y.y) << 16),
                                                                f32_to_bf16_bits(y.z) | ((uint32_t)f32_to_bf16_bits(y.w) << 16));
                }
            }
        }
    }
    if (!ok) atomicCAS(&g_paged_prompt_status, 0, 1);
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    if (warp == 12) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(*tmem_slot), "r"(512u) : "memory");
}

}  // namespace

bool paged_prompt_serves(const PagedArgs& a) {
    return (a.head_dim == 64 || a.head_dim == 128) && ((reinterpret_cast<uintptr_t>(a.query) | reinterpret_cast<uintptr_t>(a.out)) & 15u) == 0;
}

int paged_prompt_launch(cudaStream_t stream, const PagedArgs& a, bool f32) {
    const int group = a.heads / a.kv_heads;
    const long long tiles = ((long long)a.tokens * group + kPpRows - 1) / kPpRows + a.requests;  // each request ends in a tile of its own
    KMLL_REQUIRE(tiles <= INT_MAX && (long long)a.tokens * a.heads <= INT_MAX, "paged attention: too many rows");
    auto go = [&](auto kern, int smem) {
        const cudaError_t e = allow_all_dynamic_smem(kern);
        return e != cudaSuccess ? e : launch(kern, dim3((unsigned)tiles, a.kv_heads), dim3(kPpThreads), (size_t)smem, stream, true, a);
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
