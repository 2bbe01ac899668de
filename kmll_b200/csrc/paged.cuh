// What the files of the paged 8-bit cache share.
#pragma once

#include "common.cuh"

namespace kmll {

int check_paged_cache(const char* who, const void* k_codes, const void* k_scales, const void* v_codes, const void* v_scales, int pages, int block, int kv_heads, int head_dim);

}  // namespace kmll
