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
// Products.  v_mfma_f32_32x32x16_bf16 (bf16 storage) and v_mfma_f32_32x32x2_f32
// (FP32 storage): C has its column in lane % 32 and, in register r of lane half
// H = lane / 32, row 8 (r / 4) + 4 H + r % 4.  "Row" operands take 16 bytes a
// lane of row lane % 32 (16 bf16 or 8 FP32 of the contraction a step: half H
// holds the H-th 16 bytes of each 32).  "Column" operands contract over the 32
// rows of a C tile: its registers are, as they stand, the other operand of the
// next product, if the rows are taken in the order above; the LDS transpose read
// (four 16-bit rows a lane) gives the first operand in that same order, so no
// value crosses lanes between two products.
#pragma once
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

struct AttnArgs {
    const AttnSeg* segs = nullptr;
    const AttnTask* tasks = nullptr;
    uint64_t ntasks = 0;
    int heads = 0, kv_heads = 0, group = 1, dim = 0;
    int causal = 0, bias_kind = 0, buckets = 0;
    int spread = 0;  // blocks of one task go to different XCDs (else to the same)
    float scale = 1.0f, cap = 0.0f;
    const void *q = nullptr, *k = nullptr, *v = nullptr;
    uint64_t qs = 0, ks = 0, vs = 0;  // row strides (elements)
    const float* bias = nullptr;
    const uint8_t* dist = nullptr;
    void *out = nullptr, *rest = nullptr;
    uint64_t os = 0;
    float* lse = nullptr;
    // split over keys: unnormalised partial sums and (max, sum) per task row
    float *part = nullptr, *stat = nullptr;
    // backward
    const void* dout = nullptr;
    uint64_t dos = 0;
    void *dq = nullptr, *dk = nullptr, *dv = nullptr;
    uint64_t dqs = 0, dks = 0, dvs = 0;
    float* delta = nullptr;  // [rows][heads]
    float* dbias = nullptr;  // [tasks][kv_heads][group][buckets] partial sums
};

// waves: 1 or 4 waves a block, 32 packed rows (keys) each.
hipError_t launch_attention_forward(const AttnArgs& a, bool bf16, int waves, hipStream_t s);
// tiles: per split tile its segment and first row, and in lo / hi its first task and how many it has.
hipError_t launch_attention_join(const AttnArgs& a, bool bf16, const AttnTask* tiles, uint64_t ntiles, hipStream_t s);
hipError_t launch_attention_backward_q(const AttnArgs& a, bool bf16, int waves, hipStream_t s);
hipError_t launch_attention_backward_kv(const AttnArgs& a, bool bf16, int waves, hipStream_t s);
hipError_t launch_attention_bias_sum(const AttnArgs& a, float* dbias, hipStream_t s);

constexpr int kAttnMaxDim = 128, kAttnMaxBuckets = 64;
constexpr float kLog2e = 1.44269504088896341f, kLn2 = 0.693147180559945309f;

// Padded head width of the kernel that takes `dim`.
inline int attention_width(int dim) { return dim <= 32 ? 32 : dim <= 64 ? 64 : 128; }

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

// Column operand of one 32-row block and 32 columns, times the C-layout tile p:
// acc[column][lane's column of p] += sum over the 32 rows.  `rows`: LDS address
// of the block's first row, `row` bytes a row, `col` the first of the 32 columns.
template <class T, int MODE>
__device__ inline f32x16_t mfma_cols(f32x16_t acc, const char* rows, int row, int col, const uint32_t (&p)[8 * sizeof(T) / 2],
                                     int lane) {
    const int half = lane >> 5;
    if constexpr (sizeof(T) == 2) {
        typedef __attribute__((address_space(3))) s16x4_t lds4;
        const char* at = rows + (4 * half + (lane & 15) / 4) * row + (col + ((lane >> 4) & 1) * 16 + (lane & 3) * 4) * 2;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const uint2 a0 = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(at + 16 * s * row)));
            const uint2 a1 =
                __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(at + (16 * s + 8) * row)));
            const uint4 a = make_uint4(filter_word<T, MODE>(a0.x), filter_word<T, MODE>(a0.y), filter_word<T, MODE>(a1.x),
                                       filter_word<T, MODE>(a1.y));
            const uint4 b = make_uint4(p[4 * s], p[4 * s + 1], p[4 * s + 2], p[4 * s + 3]);
            acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b),
                                                          acc, 0, 0, 0);
        }
    } else {
        const char* at = rows + 4 * half * row + (col + (lane & 31)) * 4;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const uint32_t a = *reinterpret_cast<const uint32_t*>(at + (8 * (r / 4) + r % 4) * row);
            acc = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(filter_word<T, MODE>(a)), __uint_as_float(p[r]), acc,
                                                       0, 0, 0);
        }
    }
    return acc;
}

// A C tile as the second operand of mfma_cols: rounded to bf16 for bf16 storage
// (at most 2^-8 of each weight, as the stored output's own rounding; over a row's
// keys the errors are random and add up to less), unrounded for FP32.
template <class T>
__device__ inline void to_operand(const f32x16_t& c, uint32_t (&p)[8 * sizeof(T) / 2]) {
    if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = bf16x2(c[2 * i], c[2 * i + 1]);
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) p[i] = __float_as_uint(c[i]);
    }
}

// Weight tile of which every element that is not 0 counts as 1.
template <class T>
__device__ inline void seen_operand(const f32x16_t& c, uint32_t (&p)[8 * sizeof(T) / 2]) {
    f32x16_t one;
#pragma unroll
    for (int i = 0; i < 16; ++i) one[i] = c[i] == 0.0f ? 0.0f : 1.0f;
    to_operand<T>(one, p);
}

// Nonzero if 16 bytes hold a NaN or an infinity.
template <class T>
__device__ inline uint32_t nonfinite16(uint4 w) {
    constexpr uint32_t mask = sizeof(T) == 2 ? 0x7f807f80u : 0x7f800000u, one = sizeof(T) == 2 ? 0x00800080u : 0x00800000u;
    const uint32_t any = ((w.x & mask) + one) | ((w.y & mask) + one) | ((w.z & mask) + one) | ((w.w & mask) + one);
    return any & (sizeof(T) == 2 ? 0x80008000u : 0x80000000u);
}

// 2^x and the capped score: cap tanh(x) = cap (1 - 2 / (1 + e^2x)), exact at both ends.
__device__ inline float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ inline float tanh_hw(float x) {
    return 1.0f - 2.0f * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x * (2.0f * kLog2e)));
}

// A table entry in units of log2.  From kAttnHide down it hides its pairs, as -inf does: beside
// any other key its weight is 0 anyway, and a row of nothing else would have a log-sum whose
// FP32 steps are too wide to form its weights from again.
constexpr float kAttnHide = -1e6f;
__device__ inline float table_log2(float b) { return b <= kAttnHide ? -INFINITY : b * kLog2e; }

// Four consecutive columns of an output row, rounded to the storage type.
template <class T>
__device__ inline void store4(void* base, uint64_t at, float a, float b, float c, float d) {
    if constexpr (sizeof(T) == 2)
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(base) + at) = make_uint2(bf16x2(a, b), bf16x2(c, d));
    else *reinterpret_cast<float4*>(static_cast<float*>(base) + at) = make_float4(a, b, c, d);
}

// Tile of BK rows (keys, or packed query rows) of one head on its way from memory to LDS: loads
// of 16 bytes a thread, requested a tile ahead.  Rows from `end` on and columns from `dim` on are 0.
template <class T, int D, int NW, int BK>
struct AttnStage {
    static constexpr int kCpr = D * int(sizeof(T)) / 16, kPerThread = BK * kCpr / (NW * 64);
    uint4 r[kPerThread];
    __device__ void load(const T* base, uint64_t stride, uint32_t first, uint32_t end, int dim) {
#pragma unroll
        for (int i = 0; i < kPerThread; ++i) {
            const int chunk = int(threadIdx.x) + i * NW * 64, c = chunk % kCpr * AttnType<T>::kPer;
            const uint32_t row = first + uint32_t(chunk / kCpr);
            r[i] = row < end && c < dim ? *reinterpret_cast<const uint4*>(base + row * stride + c) : make_uint4(0, 0, 0, 0);
        }
    }
    // The same of packed rows: `group` vectors of `dim` side by side in each row of the array.
    __device__ void load_packed(const T* base, uint64_t stride, uint32_t first, uint32_t end, int dim, int group) {
        if (group == 1) return load(base, stride, first, end, dim);
#pragma unroll
        for (int i = 0; i < kPerThread; ++i) {
            const int chunk = int(threadIdx.x) + i * NW * 64, c = chunk % kCpr * AttnType<T>::kPer;
            const uint32_t row = first + uint32_t(chunk / kCpr), q = row / uint32_t(group);
            r[i] = row < end && c < dim
                       ? *reinterpret_cast<const uint4*>(base + q * stride + (row - q * uint32_t(group)) * uint32_t(dim) + c)
                       : make_uint4(0, 0, 0, 0);
        }
    }
    // Nonzero if the thread's part holds a NaN or an infinity.
    __device__ uint32_t nonfinite() const {
        uint32_t any = 0;
#pragma unroll
        for (int i = 0; i < kPerThread; ++i) any |= nonfinite16<T>(r[i]);
        return any;
    }
    __device__ void store(char* lds) const {
#pragma unroll
        for (int i = 0; i < kPerThread; ++i) {
            const int chunk = int(threadIdx.x) + i * NW * 64;
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
    w.query = int(row / uint32_t(a.group));
    w.local = int(row % uint32_t(a.group));
    w.head = kv * a.group + w.local;
    w.pos = w.query + int(s.k_len) - int(s.q_len);
    w.lim = a.causal ? min(int(s.k_len), max(w.pos + 1, int(s.prefix))) : int(s.k_len);
    return w;
}

// Factors of a score in units of log2: x = scale q.k log2(e), or cap log2(e) tanh(scale q.k / cap).
struct AttnScore {
    float cc, cap_in, cap_out;  // scale log2(e); scale / cap; cap log2(e)
    __device__ explicit AttnScore(const AttnArgs& a)
        : cc(a.scale * kLog2e), cap_in(a.cap > 0.0f ? a.scale / a.cap : 0.0f), cap_out(a.cap * kLog2e) {}
};

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
inline uint64_t attn_blocks(const AttnArgs& a) {
    const uint64_t blocks = a.ntasks * uint64_t(a.kv_heads);
    return a.spread ? blocks : (blocks + 7) / 8 * 8;
}

}  // namespace gatgpu
