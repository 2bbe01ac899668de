// What the files of the paged 8-bit cache share.
#pragma once

#include "common.cuh"

namespace kmll {

int check_paged_cache(const char* who, const void* k_codes, const void* k_scales, const void* v_codes, const void* v_scales, int pages, int block, int kv_heads, int head_dim);

// A kernel whose dynamic shared memory varies with the call, and is small as a rule, is opted in when a call needs it (never back: graphs keep what their nodes need).
constexpr size_t kSmemWithoutOptIn = 46 * 1024;
template <typename K>
inline cudaError_t allow_dynamic_smem(K kernel, size_t bytes) { return bytes > kSmemWithoutOptIn ? allow_all_dynamic_smem(kernel) : cudaSuccess; }

struct PagedArgs {
    const void* query;
    const int32_t *query_start, *context, *table;
    int width, requests, tokens, heads, kv_heads, head_dim, block, pages;
    const int8_t *k_codes, *v_codes;
    const float *k_scales, *v_scales;
    float scale2;  // log2(e) times the score scale
    int window;
    void* out;
    int max_query;  // requests with more rows are left out
    int skip_rows;  // requests with at most this many rows (tokens times query heads of a kv head) belong to another kernel
};

template <typename T>
__device__ inline float row_entry(const void* p, size_t i);
template <>
__device__ inline float row_entry<float>(const void* p, size_t i) { return static_cast<const float*>(p)[i]; }
template <>
__device__ inline float row_entry<uint16_t>(const void* p, size_t i) { return bf16_bits_to_f32(static_cast<const uint16_t*>(p)[i]); }
// To the nearest bf16, ties to even, and NaN stays NaN (f32_to_bf16_bits, kmll's rule for weights, carries the NaN of the arithmetic units over
// into the sign).
__device__ inline uint16_t bf16_of(float v) {
    uint16_t b;
    asm("cvt.rn.bf16.f32 %0, %1;" : "=h"(b) : "f"(v));
    return b;
}
__device__ inline uint32_t bf16_pair_of(float x, float y) {
    uint32_t b;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(b) : "f"(y), "f"(x));
    return b;
}
__device__ inline void store_row(float* p, float v) { *p = v; }
__device__ inline void store_row(uint16_t* p, float v) { *p = bf16_of(v); }

// The first position that a row at `pos` attends (its distance from rows in front of position 0 may not be a number of 32 bits).
__device__ inline int window_start(int pos, int window) { return window > 0 ? max(0, max(pos, 0) - window + 1) : 0; }

// A request's rows and the positions they attend together.
struct PagedRequest {
    int first, rows;  // rows of the step, tokens
    int pos0;         // position of the first row (negative: rows that attend nothing)
    int lo, hi;       // positions lo .. hi - 1
    __device__ static PagedRequest of(const PagedArgs& a, int r) {
        PagedRequest q;
        q.first = a.query_start[r];
        q.rows = min(a.query_start[r + 1], a.tokens) - q.first;
        if (q.first < 0 || q.rows < 0 || q.rows > a.max_query) q.rows = 0;
        const int context = a.context[r];
        q.pos0 = context - q.rows;
        q.hi = max(0, min(context, a.width * a.block));
        q.lo = min(q.hi, window_start(q.pos0, a.window));
        return q;
    }
};

// The rows that a block of the prompt kernel takes: 256 (token, query head) rows of a request and kv head, and the key tiles they see.
constexpr int kPpUnit = 256, kPpKeys = 128;
struct PagedUnit {
    int row0, live;  // first row of the request's, how many
    int low, first;  // first position that a row attends, and the first position of tile 0 (whole groups of 16)
    __device__ static PagedUnit of(const PagedArgs& a, const PagedRequest& q, int group, int unit) {
        PagedUnit u;
        u.row0 = unit * kPpUnit;
        u.live = min(kPpUnit, q.rows * group - u.row0);
        u.low = window_start(q.pos0 + u.row0 / group, a.window);
        u.first = u.low & ~15;
        return u;
    }
    __device__ int tiles_to(const PagedRequest& q, int group, int row) const {  // key tiles that a row's position needs
        const int last = min(q.pos0 + (row0 + row) / group, q.hi - 1);
        return last >= low ? (last - first) / kPpKeys + 1 : 0;
    }
    __device__ int tiles(const PagedRequest& q, int group) const { return tiles_to(q, group, live - 1); }
};
// What the prompt kernel's blocks do, in the order in which they start: entry 0 is the number of entries, then (request, unit, part of how many << 16 | part, place of
// the unit's parts in the workspace).  A null list: none is wanted.
struct PagedOrder {
    int4* list;
    int capacity;     // entries
    int split_blocks; // parts (of all kv heads) that the workspace has room for
};

// paged_decode.cu: requests of at most kPagedDecodeRows rows, heads of 64 or 128
constexpr int kPagedDecodeRows = 16;
// A workspace begins with what has to be zero between calls, at places that no size of a call moves: a counter per (request, kv head), a counter per part of the
// prompt kernel, a bit per place for its sums.  Scratch follows.
constexpr int kPagedCounters = 65536, kPpSplitBlocks = 296;  // parts: two for each multiprocessor
constexpr int kPpSums = 160;  // places for sums: one for each block of the prompt kernel that runs, one on a multiprocessor
constexpr size_t kPagedZeroBytes = (size_t)kPagedCounters * 4 + ((kPpSplitBlocks + kPpSums / 32) * 4 + 255) / 256 * 256;
bool paged_decode_serves(int head_dim);
size_t paged_decode_scratch_bytes(int head_dim, int max_rows);
int paged_decode_launch(cudaStream_t stream, const PagedArgs& a, bool f32, int max_rows, int max_context, int* arrived, void* scratch, const PagedOrder& order);

// paged_prompt.cu: requests of more than a.skip_rows rows, heads of 64 or 128
bool paged_prompt_serves(const PagedArgs& a);
bool paged_prompt_fits(const PagedArgs& a);  // its blocks and rows in 16 and 31 bits
size_t paged_prompt_scratch_bytes(int heads, int kv_heads, int head_dim, int requests, int tokens);
PagedOrder paged_prompt_order(const PagedArgs& a, void* scratch);
int paged_prompt_launch(cudaStream_t stream, const PagedArgs& a, bool f32, int* arrived, void* scratch);
int paged_prompt_status(int* status_out);  // 1 after a wait inside a kernel of that file ran out, 0 otherwise

}  // namespace kmll
