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

// The last i of [0, n) with first[i] <= x, for n >= 1, first[0] <= x: 64 places at a time, by a wave.
template <class V>
__device__ inline uint32_t last_at_most(const V* first, uint32_t n, V x, int lane) {
    uint32_t lo = 0;
    while (n > 1) {
        const uint32_t step = (n + kWave - 1) / kWave, i = uint32_t(lane) * step;
        const uint64_t below = __ballot(i < n && first[lo + i] <= x);
        const uint32_t at = uint32_t(__popcll(below) - 1) * step;  // (sorted: the lanes below are the first ones)
        lo += at;
        n = min(step, n - at);
    }
    return lo;
}

// Checks of a cache's shape and arrays (cache_append.hip).
int check_cache(gatgpu_ctx* c, const gatgpu_cache* cache, bool arrays);

}  // namespace gatgpu
