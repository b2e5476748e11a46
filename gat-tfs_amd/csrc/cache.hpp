// The paged 8-bit cache: what its append and its attention share (cache_append.hip, cache_attention.hip).
#pragma once
#include "context.hpp"

namespace gatgpu {

// Scales are powers of two from 2^kLeastScale to 2^kMostScale, so that a page whose scale grows loses nothing but what
// falls below e4m3's least value, and a scale enters a score or a weight as an exponent.
constexpr int kLeastScale = -64, kMostScale = 64;

__device__ inline int scale_exponent(float scale) {
    const int e = int(__float_as_uint(scale) >> 23 & 0xffu) - 127;
    return e < kLeastScale ? kLeastScale : e > kMostScale ? kMostScale : e;
}
__device__ inline float power_of_two(int e) { return __uint_as_float(uint32_t(e + 127) << 23); }  // -126 to 127

// Checks of a cache's shape and arrays (cache_append.hip).
int check_cache(gatgpu_ctx* c, const gatgpu_cache* cache, bool arrays);

}  // namespace gatgpu
