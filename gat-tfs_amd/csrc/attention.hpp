// Segment attention: what its kernels and its C entry points share.
//
// Rows.  Query row i of a segment carries `heads` vectors, of which `group`
// consecutive ones share a key/value head.  For one key/value head the kernels
// see the packed rows r = i * group + g (query i, head kv * group + g): the keys
// are then read once for all heads that share them, and one token of many heads
// fills a matrix tile.
//
// Visibility.  Every mask by position lets a query see a run of keys from the
// segment's start: lim(i) = Lk (full), or max(pos + 1, prefix) cut to [0, Lk]
// with pos = i + Lk - Lq (causal with a visible prefix).  Key j is seen iff
// j < lim(i) and, with a table bias, its pair's distance byte is not 255.
//
// Products (attention_tile.hpp).  v_mfma_f32_32x32x16_bf16 (bf16 storage) and v_mfma_f32_32x32x2_f32
// (FP32 storage): C has its column in lane % 32 and, in register r of lane half
// H = lane / 32, row 8 (r / 4) + 4 H + r % 4.  "Row" operands take 16 bytes a
// lane of row lane % 32 (16 bf16 or 8 FP32 of the contraction a step: half H
// holds the H-th 16 bytes of each 32).  "Column" operands contract over the 32
// rows of a C tile: its registers are, as they stand, the other operand of the
// next product, if the rows are taken in the order above; the LDS transpose read
// (four 16-bit rows a lane) gives the first operand in that same order, so no
// value crosses lanes between two products.
#pragma once
#include <type_traits>

#include "context.hpp"

namespace gatgpu {

// One segment of a plan.
struct AttnSeg {
    uint64_t q_begin, k_begin;  // first rows in the caller's arrays
    uint64_t base;              // query rows of the segments before it (rows of delta)
    uint64_t dist;              // byte offset of its distances
    uint32_t q_len, k_len, prefix, dist_ld;
};
// One tile of packed query rows over keys [k0, k1), or (backward) one tile of
// keys over packed query rows [r0, r1).
struct AttnTask {
    uint32_t seg, at, lo, hi;
};

// The capped score in units of log2, y = cap log2(e) tanh(u), u = x scale / cap, from the raw
// product x.  Where all of a tile is near 0 (scores of a few units under caps of 30 to 50) it is x
// times a polynomial in x^2, a Chebyshev fit of tanh(u) / u: of degree 2 up to |u| = 0.18
// (5.7e-8 off), of degree 4 up to 1/2 (1.4e-8); beyond by the exponential, which costs two
// quarter-rate operations a score more.
struct AttnCap {
    float in = 0.0f, out = 0.0f;          // scale / cap, cap log2(e)
    float near2 = -1.0f, near4 = -1.0f;   // largest |x| of the polynomials
    float poly2[3] = {}, poly4[5] = {};
    int bounded = 0;                      // scores are small enough for weights without a running maximum
};
AttnCap attention_cap(float scale, float cap);

struct AttnArgs {
    const AttnSeg* segs = nullptr;
    const AttnTask* tasks = nullptr;
    uint64_t ntasks = 0;
    int heads = 0, kv_heads = 0, group = 1, dim = 0;
    uint32_t group_mul = 0, group_shift = 0;  // row / group by multiplication (group_of)
    int causal = 0, bias_kind = 0, buckets = 0;
    int spread = 0;  // blocks of one task go to different XCDs (else to the same)
    float scale = 1.0f, cap = 0.0f;
    AttnCap capped;
    const void *q = nullptr, *k = nullptr, *v = nullptr;
    uint64_t qs = 0, ks = 0, vs = 0;  // row strides (elements)
    const float* bias = nullptr;
    const uint8_t* dist = nullptr;
    void *out = nullptr, *rest = nullptr;
    uint64_t os = 0;
    float* lse = nullptr;
    // tasks of a part of a tile's keys (or rows): their unfinished sums, and forward (max, sum) per task row
    float *part = nullptr, *stat = nullptr;
    // backward
    const void* dout = nullptr;
    uint64_t dos = 0;
    void *dq = nullptr, *dk = nullptr, *dv = nullptr;
    uint64_t dqs = 0, dks = 0, dvs = 0;
    float* delta = nullptr;  // [rows][heads]
    float* dbias = nullptr;  // [parts][kv_heads][group][buckets] partial sums, those of ...
    uint64_t first_part = 0; // ... this launch's tasks from here on
};

// Passes of the backward computation: over query rows, and over keys.
enum { kAttnBackwardQ = 1, kAttnBackwardKv = 2 };
// LDS bytes of a block of a backward pass; a block may have kAttnLds.
size_t attention_backward_lds_bf16(int pass, int dim, int waves, int bias, int group, int buckets);
size_t attention_backward_lds_fp32(int pass, int dim, int waves, int bias, int group, int buckets);
constexpr size_t kAttnLds = 160 * 1024;
// waves: 1 or 4 waves a block, 32 packed rows (keys) each.
hipError_t launch_attention_forward_bf16(const AttnArgs& a, int waves, hipStream_t s);
hipError_t launch_attention_forward_fp32(const AttnArgs& a, int waves, hipStream_t s);
// Blocks that cut the keys of 32 packed rows among their waves; the LDS of such a block.
hipError_t launch_attention_forward_cut_bf16(const AttnArgs& a, hipStream_t s);
hipError_t launch_attention_forward_cut_fp32(const AttnArgs& a, hipStream_t s);
size_t attention_forward_cut_lds_bf16(int dim, int bias, int group);
size_t attention_forward_cut_lds_fp32(int dim, int bias, int group);
hipError_t launch_attention_backward_q_bf16(const AttnArgs& a, int waves, hipStream_t s);
hipError_t launch_attention_backward_q_fp32(const AttnArgs& a, int waves, hipStream_t s);
hipError_t launch_attention_backward_kv_bf16(const AttnArgs& a, int waves, hipStream_t s);
hipError_t launch_attention_backward_kv_fp32(const AttnArgs& a, int waves, hipStream_t s);
// Short segments (task: segment, row of dbias, heads [lo, hi)): forward of at most 32 x blocks keys
// (1 or 2), backward of at most 32 x waves (1, 2 or 4), whose blocks take this much LDS.
hipError_t launch_attention_small_forward_bf16(const AttnArgs& a, int blocks, hipStream_t s);
hipError_t launch_attention_small_forward_fp32(const AttnArgs& a, int blocks, hipStream_t s);
hipError_t launch_attention_small_backward_bf16(const AttnArgs& a, int waves, hipStream_t s);
size_t attention_small_backward_lds_bf16(int dim, int waves, int bias, int group, int buckets);
hipError_t launch_attention_small_backward_fp32(const AttnArgs& a, int waves, hipStream_t s);
size_t attention_small_backward_lds_fp32(int dim, int waves, int bias, int group, int buckets);
// tiles: per split tile its segment and first row, and in lo / hi its first task and how many it has;
// rows: the most that one of them has.
hipError_t launch_attention_join(const AttnArgs& a, bool bf16, const AttnTask* tiles, uint64_t ntiles, uint32_t rows,
                                 hipStream_t s);
// Backward: the same tables for tiles of `height` rows (dq) or keys (dk, dv).
hipError_t launch_attention_grad_join(const AttnArgs& a, bool bf16, bool keys, const AttnTask* tiles, uint64_t ntiles, uint32_t height,
                                      hipStream_t s);
hipError_t launch_attention_bias_sum(const AttnArgs& a, uint64_t parts, float* dbias, hipStream_t s);

constexpr int kAttnMaxDim = 128, kAttnMaxBuckets = 64;
constexpr float kLog2e = 1.44269504088896341f, kLn2 = 0.693147180559945309f;

// Padded head width of the kernel that takes `dim`.
inline int attention_width(int dim) { return dim <= 32 ? 32 : dim <= 64 ? 64 : 128; }

// Widths of the forward kernel for short segments: a head's keys and values of 64 rows in registers.
template <class T>
constexpr bool attention_small_width(int width) {
    return width * int(sizeof(T)) <= 128;
}
// Waves of a block that cut its rows' keys among themselves: as many as the LDS of a CU holds tiles of.
template <class T>
constexpr int attention_cuts(int width) {
    return width * int(sizeof(T)) > 256 ? 4 : 8;
}
// a.group and what divides by it: (high half of n mul + n) >> shift for n < 2^31.
inline void set_group(AttnArgs& a, int group) {
    a.group = group;
    while ((1u << a.group_shift) < uint32_t(group)) ++a.group_shift;
    a.group_mul = uint32_t((uint64_t(1) << 32) * ((uint64_t(1) << a.group_shift) - uint64_t(group)) / uint64_t(group)) + 1;
}
// f(width, waves, bias, cap) as compile-time values.
template <class F>
hipError_t attn_dispatch(const AttnArgs& a, int waves, F f) {
    const auto by_cap = [&](auto d, auto nw, auto bias) {
        return a.cap > 0.0f ? f(d, nw, bias, std::true_type{}) : f(d, nw, bias, std::false_type{});
    };
    const auto by_bias = [&](auto d, auto nw) {
        switch (a.bias_kind) {
            case GATGPU_BIAS_LINEAR: return by_cap(d, nw, std::integral_constant<int, GATGPU_BIAS_LINEAR>{});
            case GATGPU_BIAS_TABLE: return by_cap(d, nw, std::integral_constant<int, GATGPU_BIAS_TABLE>{});
            default: return by_cap(d, nw, std::integral_constant<int, GATGPU_BIAS_NONE>{});
        }
    };
    const auto by_waves = [&](auto d) {
        return waves == 1 ? by_bias(d, std::integral_constant<int, 1>{}) : by_bias(d, std::integral_constant<int, 4>{});
    };
    switch (attention_width(a.dim)) {
        case 32: return by_waves(std::integral_constant<int, 32>{});
        case 64: return by_waves(std::integral_constant<int, 64>{});
        default: return by_waves(std::integral_constant<int, 128>{});
    }
}

inline uint64_t attn_blocks(const AttnArgs& a) {
    const uint64_t blocks = a.ntasks * uint64_t(a.kv_heads);
    return a.spread ? blocks : (blocks + 7) / 8 * 8;
}

}  // namespace gatgpu
