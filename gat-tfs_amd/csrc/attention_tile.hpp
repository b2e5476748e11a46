// Segment attention: the pieces that its kernels are made of (attention.hpp says how
// rows, keys and products lie).
#pragma once
#include "attention.hpp"

namespace gatgpu {

typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));

template <class T>
struct AttnType;
template <>
struct AttnType<uint16_t> {  // bf16
    static constexpr int kPad = 32;  // bytes behind each LDS row: row and transpose reads without bank conflicts
    static constexpr int kPer = 8;   // elements in 16 bytes
};
template <>
struct AttnType<float> {
    static constexpr int kPad = 16;
    static constexpr int kPer = 4;
};

// Bytes of an LDS row of D elements.
template <class T, int D>
constexpr int lds_row() {
    return D * int(sizeof(T)) + AttnType<T>::kPad;
}

// acc += A rows x B rows over 32 bytes of the contraction.
template <class T>
__device__ inline f32x16_t mfma_rows(f32x16_t acc, uint4 a, uint4 b) {
    if constexpr (sizeof(T) == 2) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b),
                                                       acc, 0, 0, 0);
    } else {
        acc = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.x), __uint_as_float(b.x), acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.y), __uint_as_float(b.y), acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.z), __uint_as_float(b.z), acc, 0, 0, 0);
        return __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.w), __uint_as_float(b.w), acc, 0, 0, 0);
    }
}

// What a non-finite element of a column operand becomes.
//   kRaw:   itself (tiles without any)
//   kClean: 0
//   kUp:    1 for +inf and NaN, else 0 (finite ones too);  kDown: 1 for -inf and NaN
enum { kRaw = 0, kClean = 1, kUp = 2, kDown = 3 };
template <int MODE>
__device__ inline uint32_t filter_bf16(uint32_t h) {  // one bf16 in the low half
    const bool bad = (h & 0x7f80u) == 0x7f80u, nan = bad && (h & 0x7fu);
    if (MODE == kClean) return bad ? 0u : h;
    const bool neg = h & 0x8000u;
    return bad && (nan || neg == (MODE == kDown)) ? 0x3f80u : 0u;
}
template <class T, int MODE>
__device__ inline uint32_t filter_word(uint32_t w) {
    if (MODE == kRaw) return w;
    if constexpr (sizeof(T) == 2) {
        return filter_bf16<MODE>(w & 0xffffu) | filter_bf16<MODE>(w >> 16) << 16;
    } else {
        const bool bad = (w & 0x7f800000u) == 0x7f800000u, nan = bad && (w & 0x7fffffu);
        if (MODE == kClean) return bad ? 0u : w;
        const bool neg = w >> 31;
        return bad && (nan || neg == (MODE == kDown)) ? 0x3f800000u : 0u;
    }
}

// A column operand: 32 rows of a tile in LDS (the contraction, in the order of a C tile's rows) by
// 32 columns, lane l's column being col + l % 32.  `rows`: the first row, `row` bytes a row.
template <class T>
struct AttnCols {
    uint32_t w[8 * sizeof(T) / 2];
};
template <class T, int MODE = kRaw>
__device__ inline AttnCols<T> load_cols(const char* rows, int row, int col, int lane) {
    AttnCols<T> f;
    const int half = lane >> 5;
    if constexpr (sizeof(T) == 2) {
        typedef __attribute__((address_space(3))) s16x4_t lds4;
        const char* at = rows + (4 * half + (lane & 15) / 4) * row + (col + ((lane >> 4) & 1) * 16 + (lane & 3) * 4) * 2;
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const uint2 v = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(at + 8 * s * row)));
            f.w[2 * s] = filter_word<T, MODE>(v.x);
            f.w[2 * s + 1] = filter_word<T, MODE>(v.y);
        }
    } else {
        const char* at = rows + 4 * half * row + (col + (lane & 31)) * 4;
#pragma unroll
        for (int r = 0; r < 16; ++r)
            f.w[r] = filter_word<T, MODE>(*reinterpret_cast<const uint32_t*>(at + (8 * (r / 4) + r % 4) * row));
    }
    return f;
}
// acc[a's column][b's column] += the sum over the 32 rows.
template <class T>
__device__ inline f32x16_t mfma_cols(f32x16_t acc, const AttnCols<T>& a, const AttnCols<T>& b) {
    if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const uint4 x = make_uint4(a.w[4 * s], a.w[4 * s + 1], a.w[4 * s + 2], a.w[4 * s + 3]);
            const uint4 y = make_uint4(b.w[4 * s], b.w[4 * s + 1], b.w[4 * s + 2], b.w[4 * s + 3]);
            acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, x), __builtin_bit_cast(bf16x8_t, y),
                                                          acc, 0, 0, 0);
        }
    } else {
#pragma unroll
        for (int r = 0; r < 16; ++r)
            acc = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.w[r]), __uint_as_float(b.w[r]), acc, 0, 0, 0);
    }
    return acc;
}

// A C tile as the second operand of mfma_cols: rounded to bf16 for bf16 storage
// (at most 2^-8 of each weight, as the stored output's own rounding; over a row's
// keys the errors are random and add up to less), unrounded for FP32.
template <class T>
__device__ inline AttnCols<T> to_operand(const f32x16_t& c) {
    AttnCols<T> p;
    if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int i = 0; i < 8; ++i) p.w[i] = bf16x2(c[2 * i], c[2 * i + 1]);
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) p.w[i] = __float_as_uint(c[i]);
    }
    return p;
}
// What the rounding to bf16 took, as a second operand; and what that one's rounding took, which is exactly a third's.
__device__ inline void rest_operands(const f32x16_t& c, const AttnCols<uint16_t>& p, AttnCols<uint16_t>& r, AttnCols<uint16_t>* last) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float x = c[2 * i] - __uint_as_float(p.w[i] << 16), y = c[2 * i + 1] - __uint_as_float(p.w[i] & 0xffff0000u);
        r.w[i] = bf16x2(x, y);
        if (last) last->w[i] = bf16x2(x - __uint_as_float(r.w[i] << 16), y - __uint_as_float(r.w[i] & 0xffff0000u));
    }
}

// Weight tile of which every element that is not 0 counts as 1.
template <class T>
__device__ inline AttnCols<T> seen_operand(const f32x16_t& c) {
    f32x16_t one;
#pragma unroll
    for (int i = 0; i < 16; ++i) one[i] = c[i] == 0.0f ? 0.0f : 1.0f;
    return to_operand<T>(one);
}
// An operand of weights: 1 for each that is not 0.
template <class T>
__device__ inline AttnCols<T> nonzero_operand(const AttnCols<T>& w) {
    AttnCols<T> one;
#pragma unroll
    for (int i = 0; i < int(8 * sizeof(T) / 2); ++i) {
        if constexpr (sizeof(T) == 2) one.w[i] = (w.w[i] & 0xffffu ? 0x3f80u : 0u) | (w.w[i] >> 16 ? 0x3f800000u : 0u);
        else one.w[i] = w.w[i] ? 0x3f800000u : 0u;
    }
    return one;
}
// acc += weights p (as operand w) x columns of a tile that may hold NaN and infinities: one reaches
// the rows that give its own row of the tile some weight, and no other.
template <class T>
__device__ inline f32x16_t mfma_cols_careful(f32x16_t acc, const char* rows, int row, int col, int lane,
                                             const AttnCols<T>& w, const AttnCols<T>& seen) {
    acc = mfma_cols<T>(acc, load_cols<T, kClean>(rows, row, col, lane), w);
    const f32x16_t up = mfma_cols<T>(f32x16_t{}, load_cols<T, kUp>(rows, row, col, lane), seen);
#pragma unroll
    for (int r = 0; r < 16; ++r)
        if (up[r] > 0.0f) acc[r] += INFINITY;
    __builtin_amdgcn_sched_barrier(0);  // (one at a time: no registers for both)
    const f32x16_t down = mfma_cols<T>(f32x16_t{}, load_cols<T, kDown>(rows, row, col, lane), seen);
#pragma unroll
    for (int r = 0; r < 16; ++r)
        if (down[r] > 0.0f) acc[r] -= INFINITY;
    return acc;
}
// True if a lane's sums hold a NaN or an infinity.
template <int N>
__device__ inline bool nonfinite(const f32x16_t (&acc)[N]) {
    float zero = 0.0f;
#pragma unroll
    for (int d = 0; d < N; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) zero = fmaf(acc[d][r], 0.0f, zero);
    return zero != 0.0f;
}

__device__ inline float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// Capped scores of a tile from its raw products (AttnCap), less `less`.
__device__ inline void cap_scores(const AttnCap& c, f32x16_t& s, float less) {
    float top = 0.0f;
#pragma unroll
    for (int r = 0; r < 16; r += 2) top = fmaxf(fmaxf(top, fabsf(s[r])), fabsf(s[r + 1]));
    if (__all(top <= c.near2)) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const float t = s[r] * s[r];
            s[r] = fmaf(s[r], fmaf(fmaf(c.poly2[2], t, c.poly2[1]), t, c.poly2[0]), -less);
        }
    } else if (__all(top <= c.near4)) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const float t = s[r] * s[r];
            const float p = fmaf(fmaf(fmaf(fmaf(c.poly4[4], t, c.poly4[3]), t, c.poly4[2]), t, c.poly4[1]), t, c.poly4[0]);
            s[r] = fmaf(s[r], p, -less);
        }
    } else {  // tanh(u) = 1 - 2 / (1 + e^2u), exact at both ends, to 2^-23 between: 6e-6 of a score under a cap of 50, that
              // of one near the cap in FP32; small scores would keep more by the polynomial, a lane at a time, which took
              // 1430 us where this takes 1020 (16K nodes, 8 x 64, cap 3; 820 where all scores are small)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const float e = __builtin_amdgcn_exp2f(s[r] * c.in * (2.0f * kLog2e));
            s[r] = fmaf(c.out, 1.0f - 2.0f * __builtin_amdgcn_rcpf(1.0f + e), -less);
        }
    }
}

// A table entry in units of log2.  From kAttnHide down it hides its pairs, as -inf does: beside
// any other key its weight is 0 anyway, and a row of nothing else would have a log-sum whose
// FP32 steps are too wide to form its weights from again.
constexpr float kAttnHide = -1e6f;
__device__ inline float table_log2(float b) { return b <= kAttnHide ? -INFINITY : b * kLog2e; }
// The biases of a key/value head's query heads, one of 256 entries for each value of the distance
// byte: [group][256], -inf for hidden pairs.
__device__ inline void fill_table(const AttnArgs& a, int kv, float* table) {
    for (int i = int(threadIdx.x); i < a.group * 256; i += int(blockDim.x)) {
        const int d = i & 255;
        table[i] = d == GATGPU_HIDDEN
                       ? -INFINITY
                       : table_log2(a.bias[(kv * a.group + (i >> 8)) * a.buckets + min(d, a.buckets - 1)]);
    }
}
// A lane's distance bytes of one 32-key block: keys first + 8 i + (0 .. 3).  Behind the row's ld
// bytes they are some others of the row: no query sees those keys.  (A segment without keys has no
// distances at all.)
struct AttnDist {
    uint32_t w[4];
};
__device__ inline AttnDist load_dist(const uint8_t* row, uint32_t first, uint32_t ld) {
    AttnDist d{};
    if (ld == 0) return d;
#pragma unroll
    for (int i = 0; i < 4; ++i) d.w[i] = *reinterpret_cast<const uint32_t*>(row + min(first + 8 * i, ld - 4));
    return d;
}
__device__ inline uint32_t dist_of(const AttnDist& d, int r) { return d.w[r / 4] >> (8 * (r % 4)) & 255u; }

// Adds a block's score gradients to the lane's column of the bias gradient, [buckets][cols].  (Graphs of
// 130 to 1300 rows, the pass over query rows: 109 us so; 129 four at a time with equal buckets joined in
// registers; 490 with LDS additions without a return.)
__device__ inline void add_bins(float* column, int cols, int buckets, AttnDist d, const f32x16_t& y) {
#pragma unroll
    for (int i = 0; i < 4; ++i) asm("" : "+v"(d.w[i]));  // (the bytes are taken apart anew, not kept since the scores)
#pragma unroll
    for (int r = 0; r < 16; ++r) column[min(int(dist_of(d, r)), buckets - 1) * cols] += y[r];
}
// Scores of a block in units of log2, less `less`, from its raw products.  cc: their factor without
// a cap; gap: the row's position less the block's first key of the lane; table: the row's entries.
// A hidden pair's score is -inf; only CAREFUL keeps it so where its product is a NaN or +inf.
template <int BIAS, bool CAP, bool CAREFUL>
__device__ inline void tile_scores(const AttnCap& cap, f32x16_t& s, float cc, float less, float slope2, float gap,
                                   const AttnDist& d, const float* table) {
    if constexpr (CAP) cap_scores(cap, s, less);
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        float x = CAP ? s[r] : fmaf(s[r], cc, -less);
        if constexpr (BIAS == GATGPU_BIAS_LINEAR) x = fmaf(-slope2, fabsf(gap - float(8 * (r / 4) + r % 4)), x);
        if constexpr (BIAS == GATGPU_BIAS_TABLE) {
            const float t = table[dist_of(d, r)];
            x += t;
            if (CAREFUL && t == -INFINITY) x = t;
        }
        s[r] = x;
    }
}

// Weights p and score gradients y = p (dp - delta) of a block from its raw products s and dp;
// with CAP, s becomes 1 - tanh^2, the capped score's slope.  left: keys of the lane from its first
// on that the row sees (where masked).  CAREFUL: a weight of 0 has no gradient, whatever dp and the slope are.
template <int BIAS, bool CAP, bool CAREFUL>
__device__ inline void score_gradients(const AttnCap& cap, f32x16_t& s, const f32x16_t& dp, f32x16_t& y, f32x16_t* weights,
                                       float cc, float uncap, float slope2, float gap, const AttnDist& dist,
                                       const float* table, bool masked, int left, float lse2, float delta) {
    if constexpr (CAP) {
        cap_scores(cap, s, 0.0f);
        y = s;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const float t = s[r] * uncap;
            s[r] = fmaf(-t, t, 1.0f);
            y[r] -= lse2;
        }
    } else {
#pragma unroll
        for (int r = 0; r < 16; ++r) y[r] = fmaf(s[r], cc, -lse2);
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        if constexpr (BIAS == GATGPU_BIAS_LINEAR) y[r] = fmaf(-slope2, fabsf(gap - float(8 * (r / 4) + r % 4)), y[r]);
        if constexpr (BIAS == GATGPU_BIAS_TABLE) {
            const float t = table[dist_of(dist, r)];
            y[r] += t;
            if (CAREFUL && t == -INFINITY) y[r] = t;
        }
    }
    if (masked) {
#pragma unroll
        for (int r = 0; r < 16; ++r)
            if (8 * (r / 4) + r % 4 >= left) y[r] = -INFINITY;
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const float p = exp2_hw(y[r]);
        if (weights) (*weights)[r] = p;
        y[r] = CAREFUL && p == 0.0f ? 0.0f : p * (dp[r] - delta);
        if (CAP && CAREFUL && p == 0.0f) s[r] = 0.0f;
    }
}

// A C tile (rows: keys, columns: query rows) through LDS, one row a query row of 32 keys, from
// where load_cols takes it as an operand that contracts over the query rows.  The row's 8 (16)
// bytes behind its 32 elements keep both sides free of bank conflicts.
template <class T>
constexpr int attn_turn_row() {
    return sizeof(T) == 2 ? 72 : 144;
}
template <class T>
__device__ inline void turn_store(char* to, const AttnCols<T>& c, int lane) {
    char* row = to + (lane & 31) * attn_turn_row<T>() + 4 * (lane >> 5) * int(sizeof(T));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 2) *reinterpret_cast<uint2*>(row + 16 * i) = make_uint2(c.w[2 * i], c.w[2 * i + 1]);
        else *reinterpret_cast<uint4*>(row + 32 * i) = make_uint4(c.w[4 * i], c.w[4 * i + 1], c.w[4 * i + 2], c.w[4 * i + 3]);
    }
}

// Query of a packed row.
__device__ inline uint32_t group_of(const AttnArgs& a, uint32_t row) {
    return (__umulhi(row, a.group_mul) + row) >> a.group_shift;
}

// A barrier of the block for what its waves have in LDS.  Unlike __syncthreads it does not wait for
// requests to memory: the next tile's loads and the last one's stores stay in flight across it.
__device__ inline void lds_barrier() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}
// Rows of a tile in LDS.
template <class T, int NW>
constexpr int attn_tile_rows() {
    return NW == 1 || sizeof(T) == 4 ? 32 : 64;
}
// Two buffers spare a barrier a tile; FP32 tiles are too large for them, and one wave needs none.
template <class T, int NW>
constexpr int attn_buffers() {
    return sizeof(T) == 2 && NW > 1 ? 2 : 1;
}

// Waves a SIMD that the registers are held to, where a wave's sums, operands and scores fit.
template <class T, int D, int NW>
constexpr int attn_waves() {
    return sizeof(T) == 2 && (D < 128 || NW == 4) ? 2 : 1;
}

// Tile of BK rows (keys, or packed query rows) of one head on its way from memory to LDS: loads
// of 16 bytes a thread, requested a tile ahead.  Rows from `end` on and columns from `dim` on are 0.
// A thread's first place in a tile is the same in every tile, its others lie a fixed number of rows
// further, and a tile's address is the block's own; where these do not fit 31 bits, or those rows
// are no whole number of queries, addresses are formed anew.
template <class T, int D, int NW, int BK>
struct AttnStage {
    static constexpr int kCpr = D * int(sizeof(T)) / 16, kPerThread = BK * kCpr / (NW * 64), kRowStep = NW * 64 / kCpr;
    static __device__ uint32_t thread() { return NW == 1 ? threadIdx.x & 63u : threadIdx.x; }
    uint4 r[kPerThread];
    uint32_t at;    // byte offset of the first place in a tile
    uint32_t step;  // bytes from place to place, 0: addresses are formed anew
    __device__ __forceinline__ void place(const AttnArgs& a, uint64_t stride, int group) {
        const uint64_t bytes = stride * sizeof(T) * uint64_t(BK);
        step = kRowStep % group == 0 && bytes < (uint64_t(1) << 31)
                   ? uint32_t(stride * sizeof(T)) * uint32_t(kRowStep / group)
                   : 0u;
        const uint32_t row = thread() / uint32_t(kCpr), q = group == 1 ? row : group_of(a, row);
        at = uint32_t((q * stride + (row - q * uint32_t(group)) * uint32_t(a.dim)) * sizeof(T)) +
             thread() % uint32_t(kCpr) * 16u;
    }
    // Rows first .. first + BK of `base`; first is a multiple of BK.
    __device__ __forceinline__ void load(const AttnArgs& a, const T* base, uint64_t stride, int group, uint32_t first, uint32_t end) {
        const bool wide = a.dim == D;
        if (__builtin_expect(step != 0, 1)) {
            const char* tile = reinterpret_cast<const char*>(base) + uint64_t(first / uint32_t(kRowStep)) * step;
            if (wide && first + BK <= end) {
#pragma unroll
                for (int i = 0; i < kPerThread; ++i) r[i] = *reinterpret_cast<const uint4*>(tile + uint64_t(i) * step + at);
                return;
            }
#pragma unroll
            for (int i = 0; i < kPerThread; ++i) {
                const int chunk = int(thread()) + i * NW * 64;
                const bool in = first + uint32_t(chunk / kCpr) < end && chunk % kCpr * AttnType<T>::kPer < a.dim;
                r[i] = in ? *reinterpret_cast<const uint4*>(tile + uint64_t(i) * step + at) : make_uint4(0, 0, 0, 0);
            }
            return;
        }
#pragma unroll
        for (int i = 0; i < kPerThread; ++i) {
            const int chunk = int(thread()) + i * NW * 64, c = chunk % kCpr * AttnType<T>::kPer;
            const uint32_t row = first + uint32_t(chunk / kCpr), q = group == 1 ? row : group_of(a, row);
            r[i] = row < end && c < a.dim ? *reinterpret_cast<const uint4*>(base + q * stride +
                                                                           (row - q * uint32_t(group)) * uint32_t(a.dim) + c)
                                          : make_uint4(0, 0, 0, 0);
        }
    }
    __device__ __forceinline__ void store(char* lds) const {
#pragma unroll
        for (int i = 0; i < kPerThread; ++i) {
            const int chunk = int(thread()) + i * NW * 64;
            *reinterpret_cast<uint4*>(lds + chunk / kCpr * lds_row<T, D>() + chunk % kCpr * 16) = r[i];
        }
    }
};

// What a lane knows of its packed query row.
struct AttnRow {
    int query, local, head;  // query of the segment, head within the group, head
    int pos, lim;            // position among the keys; keys [0, lim) are seen
};
__device__ inline AttnRow attn_row(const AttnArgs& a, const AttnSeg& s, uint32_t row, int kv) {
    AttnRow w;
    w.query = int(group_of(a, row));
    w.local = int(row) - w.query * a.group;
    w.head = kv * a.group + w.local;
    w.pos = w.query + int(s.k_len) - int(s.q_len);
    w.lim = a.causal ? min(int(s.k_len), max(w.pos + 1, int(s.prefix))) : int(s.k_len);
    return w;
}

// What rounding to the bf16 `b` took from x: the difference of their FP32 patterns, -2^15 to 2^15, halved to 15 bits, so that
// both give x to 23 bits (a bf16 rest would give 17).  Bit 14 stays 0: as a bf16 a rest is never a NaN.
__device__ inline uint32_t rest_bits(float x, uint32_t b) {
    const int t = max(-32768, min(32767, int(__float_as_uint(x) - (b << 16))));
    const uint32_t u = uint32_t(t + 32768) >> 1;
    return (u & 0x4000u) << 1 | (u & 0x3fffu);
}
__device__ inline float with_rest(uint32_t b, uint32_t rest) {
    return __uint_as_float((b << 16) + 2 * ((rest >> 1 & 0x4000u) | (rest & 0x3fffu)) - 32768u);
}

// Rows of a C tile set (columns: rows of the output, registers: dim) times `factor`, rounded to
// the storage type, to the lane's row at base + at.  bf16: the wave's halves swap 8 bytes, so that
// each lane stores 16.  Every lane of the wave takes part; rows with `in` are stored.  REST: what
// the rounding took instead.
template <class T, int DB, bool REST = false>
__device__ inline void store_rows(void* base, uint64_t at, const f32x16_t (&acc)[DB], float factor, int half, int dim, bool in) {
    if constexpr (sizeof(T) == 2) {
        uint16_t* to = static_cast<uint16_t*>(base) + at;
        const auto pack = [&](float x, float y) {
            x *= factor;
            y *= factor;
            uint32_t u = bf16x2(x, y);
            if (REST) u = rest_bits(x, u & 0xffffu) | rest_bits(y, u >> 16) << 16;
            return u;
        };
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                uint32_t w[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] = pack(acc[d][8 * j + 2 * e], acc[d][8 * j + 2 * e + 1]);
                const auto x = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false);
                const auto y = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
                const int c = d * 32 + 16 * j + 8 * half;
                if (in && c < dim) *reinterpret_cast<uint4*>(to + c) = make_uint4(x[0], y[0], x[1], y[1]);
            }
    } else {
        float* to = static_cast<float*>(base) + at;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int c = d * 32 + 8 * i + 4 * half;
                if (in && c < dim)
                    *reinterpret_cast<float4*>(to + c) = make_float4(acc[d][4 * i] * factor, acc[d][4 * i + 1] * factor,
                                                                     acc[d][4 * i + 2] * factor, acc[d][4 * i + 3] * factor);
            }
    }
}
// A row's output, what its rounding took and its log-sum, from its sums.  l == 0: it saw nothing.
template <class T, int DB>
__device__ inline void store_out(const AttnArgs& a, const AttnSeg& seg, const AttnRow& w, const f32x16_t (&acc)[DB], float m,
                                 float l, int half, bool in) {
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const uint64_t row = seg.q_begin + uint64_t(w.query), to = row * a.os + uint64_t(w.head) * a.dim;
    store_rows<T, DB>(a.out, to, acc, inv, half, a.dim, in);
    if constexpr (sizeof(T) == 2) {
        if (a.rest) store_rows<T, DB, true>(a.rest, to, acc, inv, half, a.dim, in);
    }
    if (a.lse && half == 0 && in)
        a.lse[row * uint64_t(a.heads) + w.head] = l == 0.0f ? -INFINITY : (m + __log2f(l)) * kLn2;
}

// Four consecutive columns of an output row, rounded to the storage type.
template <class T>
__device__ inline void store4(void* base, uint64_t at, float a, float b, float c, float d) {
    if constexpr (sizeof(T) == 2)
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(base) + at) = make_uint2(bf16x2(a, b), bf16x2(c, d));
    else *reinterpret_cast<float4*>(static_cast<float*>(base) + at) = make_float4(a, b, c, d);
}

// A row's FP32 sums to row `at` of a workspace of rows of 32 DB columns, where a launch joins them.
template <int DB>
__device__ inline void store_part(float* part, uint64_t at, const f32x16_t (&acc)[DB], int half, bool in) {
    if (!in) return;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            store4<float>(part, at * (32 * DB) + uint64_t(d * 32 + 8 * i + 4 * half), acc[d][4 * i], acc[d][4 * i + 1],
                          acc[d][4 * i + 2], acc[d][4 * i + 3]);
}

// Block b's (task, key/value head).  Blocks go to the 8 XCDs in turn.  spread:
// heads of a task side by side, so an XCD sees few heads (of 8: one) of all tasks
// and keeps that head's keys in its L2; else each XCD takes a run of tasks with
// all their heads, whose rows are parts of the same lines.
__device__ inline bool attn_task(const AttnArgs& a, uint64_t& task, int& kv) {
    const uint64_t blocks = a.ntasks * uint64_t(a.kv_heads);
    uint64_t b = blockIdx.x;
    if (!a.spread) {
        const uint64_t per = (blocks + 7) / 8;
        b = (b % 8) * per + b / 8;
        if (b / per != blockIdx.x % 8 || b >= blocks) return false;
    }
    if (b >= blocks) return false;
    task = b / uint64_t(a.kv_heads);
    kv = int(b % uint64_t(a.kv_heads));
    return true;
}

}  // namespace gatgpu
