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
// values leave fp16 or FP32, and the weights' sum takes p' 2^-ev.
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
    uint32_t workers = 0;  // of a key/value head; 0: a block a request
    uint32_t least = 0;    // tiles of a worker
    float scale = 0.0f;    // scale log2 e
    uint64_t ld = 0, qs = 0, os = 0;
    const void* q = nullptr;
    void* out = nullptr;
    float* lse = nullptr;
    const uint32_t *q_begin = nullptr, *k_len = nullptr, *table = nullptr;
    const uint8_t *k = nullptr, *v = nullptr;
    const float *k_scale = nullptr, *v_scale = nullptr;
    // Partial sums, of two pieces a worker and head: [piece][columns / 16][64][4] sums, [piece][2][16] references and weights.
    float *part = nullptr, *stat = nullptr;
    uint4* meta = nullptr;  // [worker][head]: request, row tile, pieces (0: none) of the task that begins in the worker and ends in another
};
__device__ inline CacheRequest request_of(const CacheAttnArgs& a, uint32_t r) { return cache_request(a.c, a.q_begin[r], a.q_begin[r + 1], a.k_len[r]); }

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

}  // namespace gatgpu
