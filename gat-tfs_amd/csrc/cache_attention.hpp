// Attention over the paged 8-bit cache: operands, and what its kernels share (cache_attention.hip).
//
// A wave takes 64 keys by 16 packed rows (row index = query i of the request * group + head of the group) a step on
// v_mfma_f32_16x16x32.  The scores are formed as keys x rows, S^T = K Q^T, and the sums as O^T = V^T P^T, so that lane
// (n = lane % 16, g = lane / 16) owns row n's scores of the 16 keys 16 g + 4 a + r (operand a of 4, register r of 4):
//   K operand a:   lane (m, g) holds key 16 (m / 4) + 4 a + m % 4 at columns 64 b + 16 g + 8 s of step (b, s)
//   P operand:     lane (n, g) holds its own keys 16 g + 8 s ... + 7: the weights in the registers they were computed in
//   V operand:     lane (m, g) holds those keys of column 16 db + m: 16 bytes of a page's column, as they lie
// so keys and values come straight from memory, 16 bytes a lane, with no LDS and no exchange between lanes, and since a
// page is a multiple of 16 tokens, each lane's keys lie in one page.
//
// Numbers: e4m3 is exact in bf16 and in fp16.  Keys meet the queries in bf16 (FP32 queries as three bf16 parts, which
// hold all their bits).  Values meet the weights in fp16: weights are kept within 2^15 of a row's reference, where fp16
// is off by at most 2^-11 of the weight (bf16: 2^-8, as much as the output's own rounding), and lie below 2^-14 only where
// they are 2^-21 of the largest; FP32 calls take a second fp16 part for what that rounding took.  The scale of the values'
// page enters the weight as an exponent, p' = 2^(x + ev - ref), ref following the largest x + ev, so that no page's
// values leave fp16 or FP32, and the weights' sum takes p' 2^-ev.  That holds where the scales of a wave's (a block's) pages
// are not far apart: with exponents within kCacheSpread a weight counts in the sum unless it is below 2^-96 of the largest.
// Sums are joined by references that stand for the weights alone: see weighed.
#pragma once
#include "cache.hpp"
#include "cache_index.hpp"

namespace gatgpu {

typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2v_t __attribute__((ext_vector_type(2)));

struct CacheAttnArgs {
    CacheSizes c;
    uint32_t workers = 0;  // of a key/value head; 0: a block a row tile
    uint32_t least = 0;    // least work of a worker, where requests have as much: key tiles, times row tiles where these are of 16
    uint32_t row_tiles = 0;  // of a request, at most; for a block a row tile
    float scale = 0.0f;    // scale log2 e
    uint64_t ld = 0, qs = 0, os = 0;
    const void* q = nullptr;
    void* out = nullptr;
    float* lse = nullptr;
    const uint32_t *q_begin = nullptr, *k_len = nullptr, *table = nullptr;
    const uint8_t *k = nullptr, *v = nullptr;
    const float *k_scale = nullptr, *v_scale = nullptr;
    // Partial sums, of two pieces a worker and head: [piece][row tile][columns / 16][64][4] sums, [piece][row tile][2][16]
    // references and weights.
    float *part = nullptr, *stat = nullptr;
    uint4* meta = nullptr;  // [worker][head]: request, row tile, pieces (0: none) of the work that begins in the worker and ends in another
};
// One request's place (by scalar loads where r is the same in all lanes).
__device__ inline CacheRequest request_of(const CacheAttnArgs& a, uint32_t r) {
    return cache_request(a.c, read_only(a.q_begin)[r], read_only(a.q_begin)[r + 1], read_only(a.k_len)[r]);
}
// A value that is the same in all lanes, in a scalar register.
__device__ inline uint32_t uniform(uint32_t x) { return uint32_t(__builtin_amdgcn_readfirstlane(int(x))); }
__device__ inline uint64_t uniform(uint64_t x) { return uint64_t(uniform(uint32_t(x >> 32))) << 32 | uniform(uint32_t(x)); }

__device__ inline uint32_t f16x2(float lo, float hi) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2_t){lo, hi}, f16x2_t));
}
// Eight e4m3 bytes as bf16 (fp16) operands.
__device__ inline uint4 keys_operand(uint32_t lo, uint32_t hi) {
    return make_uint4(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true)));
}
__device__ inline uint4 values_operand(uint32_t lo, uint32_t hi) {
    return make_uint4(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true)));
}
__device__ inline f32x4_t mfma_bf16(uint4 a, uint4 b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}
__device__ inline f32x4_t mfma_f16(uint4 a, uint4 b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
}

// 0x80 at each NaN among four e4m3 bytes.
__device__ inline uint32_t nan_bytes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }
// The lowest n (0 to 4 and beyond) bytes of a word.
__device__ inline uint32_t low_bytes(int n) { return n <= 0 ? 0u : n >= 4 ? 0xffffffffu : (1u << (8 * n)) - 1; }

// A row's reference before anything was seen: finite, so that scores of -infinity weigh 0; how far above it a score may
// lie before it is raised, and how far below the score it is raised to.  References are whole numbers, so that rescaling
// is exact and a weight's exponent, x + (ev - ref), is rounded once.
constexpr float kCacheNoRef = -3.402823466e38f, kCacheRoom = 15.0f, kCacheSet = 7.0f;
// References from this size on are far: an exponent's rounding is a quarter and more of a step of 2, and soon wider than the room
// and the values' exponents.
constexpr float kCacheFar = 4194304.0f;
// How far apart the exponents of the values' scales may lie: keys of equal weights then have 2^-14 and more of fp16, its 11 bits
// (FP32: 2^-2 and more of two parts, 23 bits).  Beyond, and for rows whose reference is far, what a wave (a block) has is formed again,
// behind the others.  There each 16 keys of a row, of one page, have a reference of their own, a whole number at or above their
// largest score; scores are rounded before it leaves them, and the products with the values are shifted to the row's reference,
// the largest, and by the page's exponent as they are added.  So a weight is off by 2^-11 (FP32: 2^-22) or by 2^-38 of the 16
// keys' largest, whatever the pages' scales.
template <class T>
constexpr int kCacheSpread = sizeof(T) == 2 ? 20 : 8;
constexpr float kCacheUp = 14.0f;  // such weights are 2^14 at most
// A score that is rounded before anything leaves it, and its weight (NaN stays).
__device__ inline float far_score(float score, float by) {
#pragma clang fp contract(off)
    return score * by;
}
__device__ inline float far_weight(float score, float ref) {
#pragma clang fp contract(off)
    return __builtin_amdgcn_exp2f((score - ref) + kCacheUp);
}
// The reference of keys with this largest score.
__device__ inline float far_reference(float top) { return top > -INFINITY ? ceilf(top) : kCacheNoRef; }
// x 2^(from - to), for whole numbers from <= to: by an exponent, since the power alone may lie below FP32's numbers.
__device__ inline int shift_of(float from, float to) { return int(fmaxf(from - to, -1000.0f)); }
__device__ inline float shifted(float x, int by) { return __builtin_amdgcn_ldexpf(x, by); }
template <class V>
__device__ inline V shifted_all(V x, int by) {
#pragma unroll
    for (uint32_t i = 0; i < sizeof(V) / 4; ++i) x[i] = shifted(x[i], by);
    return x;
}
// Before sums are joined: a row's reference becomes that of its weights' sum, which is then 0.5 to 1 (the sums of products are a mean of
// values then).  Returns by what its sums are shifted.
__device__ inline int weighed(float& ref, float& sum) {
    const int e = __builtin_amdgcn_frexp_expf(sum);  // (0 for 0, infinity and NaN)
    ref += float(e);
    sum = shifted(sum, -e);
    return -e;
}

// What a page's scores are multiplied by: scale log2 e 2^exponent, kept among FP32's normal values, so that a masked score stays
// -infinity and one of 0 stays 0.
__device__ inline float score_factor(float scale, float page_scale) {
    return __builtin_amdgcn_fmed3f(scale * power_of_two(scale_exponent(page_scale)), 1.17549435e-38f, 3.402823466e38f);
}

// Columns col to col + 3 of a packed row, from the sums of its weights' products and of its weights.
template <class T>
__device__ inline void store4(const CacheAttnArgs& a, const CacheRequest& rq, uint32_t packed, uint32_t head, uint32_t col, f32x4_t o, float sum) {
    if (packed >= rq.rows * a.c.group || col >= a.c.dim) return;
    const uint32_t i = packed / a.c.group, h = head * a.c.group + packed % a.c.group;
    T* const to = static_cast<T*>(a.out) + uint64_t(rq.begin + i) * a.os + uint64_t(h) * a.c.dim + col;
    const float by = sum == 0.0f ? 0.0f : 1.0f / sum;
    if (sum == 0.0f) o = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    if constexpr (sizeof(T) == 2) *reinterpret_cast<uint2*>(to) = make_uint2(bf16x2(o[0] * by, o[1] * by), bf16x2(o[2] * by, o[3] * by));
    else *reinterpret_cast<float4*>(to) = make_float4(o[0] * by, o[1] * by, o[2] * by, o[3] * by);
}
__device__ inline void store_lse(const CacheAttnArgs& a, const CacheRequest& rq, uint32_t packed, uint32_t head, float ref, float sum) {
    if (!a.lse || packed >= rq.rows * a.c.group) return;
    const uint32_t i = packed / a.c.group, h = head * a.c.group + packed % a.c.group;
    a.lse[uint64_t(rq.begin + i) * a.c.heads + h] = sum == 0.0f ? -INFINITY : (ref + log2f(sum)) * 0.6931471805599453f;
}

// A value's first part before it is rounded to bf16, which is to stay finite, and what a part leaves of it: of an infinity or NaN nothing.
__device__ inline float first_part(float x) {
    constexpr float most = 3.38953139e38f;  // bf16's largest number
    return fabsf(x) < INFINITY ? __builtin_amdgcn_fmed3f(x, -most, most) : x;
}
__device__ inline float rest_of(float x, float part) { return fabsf(x) < INFINITY ? x - part : 0.0f; }
// Eight values of a query row from `col` on, as PARTS bf16 operands (FP32: three, which hold all its bits).
template <class T>
struct QueryParts {
    static constexpr int N = sizeof(T) == 2 ? 1 : 3;
    uint4 w[N];
};
template <class T>
__device__ inline QueryParts<T> load_query8(const T* row, uint32_t col, bool there) {
    QueryParts<T> q;
    if constexpr (sizeof(T) == 2) {
        q.w[0] = there ? *reinterpret_cast<const uint4*>(row + col) : make_uint4(0, 0, 0, 0);
    } else {
        float x[8] = {};
        if (there) {
            const float4 lo = *reinterpret_cast<const float4*>(row + col), hi = *reinterpret_cast<const float4*>(row + col + 4);
            x[0] = lo.x, x[1] = lo.y, x[2] = lo.z, x[3] = lo.w, x[4] = hi.x, x[5] = hi.y, x[6] = hi.z, x[7] = hi.w;
        }
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            uint32_t p[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                p[j] = k ? bf16x2(x[2 * j], x[2 * j + 1]) : bf16x2(first_part(x[2 * j]), first_part(x[2 * j + 1]));
                x[2 * j] = rest_of(x[2 * j], __uint_as_float(p[j] << 16));
                x[2 * j + 1] = rest_of(x[2 * j + 1], __uint_as_float(p[j] & 0xffff0000u));
            }
            q.w[k] = make_uint4(p[0], p[1], p[2], p[3]);
        }
    }
    return q;
}
// The queries of a packed row: its first element, the request's first row where there is none.
template <class T>
__device__ inline const T* query_row(const CacheAttnArgs& a, const CacheRequest& rq, uint32_t packed, uint32_t head) {
    const bool there = packed < rq.rows * a.c.group;
    const uint32_t i = there ? packed / a.c.group : 0, h = head * a.c.group + packed % a.c.group;
    return static_cast<const T*>(a.q) + uint64_t(rq.begin + i) * a.qs + uint64_t(h) * a.c.dim;
}

// Many rows a request (cache_attention_chunk.hip): workspace and launches.
struct ChunkPlan {
    uint32_t tiles = 0;    // at most, of packed rows
    uint32_t workers = 0;  // of a key/value head
    uint64_t begin = 0, request = 0, upto = 0, part = 0, stat = 0, meta = 0, bytes = 0;  // offsets in the workspace
};
ChunkPlan chunk_plan(int cus, const CacheSizes& c, bool bf16);
uint32_t chunk_rows(const CacheSizes& c, bool bf16);  // packed rows of a tile
hipError_t launch_cache_chunk(const CacheAttnArgs& a, bool bf16, const ChunkPlan& plan, void* workspace, hipStream_t s);

}  // namespace gatgpu
