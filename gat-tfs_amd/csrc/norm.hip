// Layer norm, forward and backward.
//
//   h = x (+ residual, rounded to the storage type),  mean and var over the row's columns,
//   r = 1 / sqrt(var + eps),  n = (h - mean) r,  t = n gamma + beta,  y = t or ELU(t)
//   dt = dy (ELU'(t)),  dgamma = sum dt n,  dbeta = sum dt,  g = dt gamma,
//   dx = r (g - mean(g) - n mean(g n)) (+ dsum)
//
// Bound by bytes: a row is read once into registers (TPR threads a row, ITEMS chunks of
// VEC elements a thread), its mean and then its centred squares are summed from there, and
// it is written once.  The backward pass gives each block a fixed set of rows and keeps its
// columns' sums of dgamma and dbeta in registers over them; blocks leave one partial row
// each, which a second launch adds in one fixed order.  Sums are FP32.
#include <algorithm>
#include <cmath>
#include <string>
#include <type_traits>

#include "context.hpp"
#include "norm.hpp"

namespace gatgpu {
namespace {

// Chunks of 16 bytes; FREE: at any element's address, for rows of no whole chunks or off 16 bytes (29817 x 566 bf16,
// forward: 30 us, 71 an element at a time; 169K x 255, training: 192, x 256 in whole chunks: 143).
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef u32x4_t u32x4_at2 __attribute__((aligned(2)));
typedef u32x4_t u32x4_at4 __attribute__((aligned(4)));
template <class T, bool FREE>
__device__ inline u32x4_t load16(const T* p) {
    if constexpr (!FREE) return *reinterpret_cast<const u32x4_t*>(p);
    else if constexpr (sizeof(T) == 2) return *reinterpret_cast<const u32x4_at2*>(p);
    else return *reinterpret_cast<const u32x4_at4*>(p);
}
template <class T, bool FREE>
__device__ inline void store16(T* p, u32x4_t v) {
    if constexpr (!FREE) *reinterpret_cast<u32x4_t*>(p) = v;
    else if constexpr (sizeof(T) == 2) *reinterpret_cast<u32x4_at2*>(p) = v;
    else *reinterpret_cast<u32x4_at4*>(p) = v;
}
template <class T>
__device__ inline float widen(T x) {
    if constexpr (sizeof(T) == 2) return bf16_widen(x);
    else return x;
}
template <class T>
__device__ inline void store_one(T* p, float v) {
    if constexpr (sizeof(T) == 2) *p = bf16_rne(v);
    else *p = v;
}
// Chunks of one row as they lie in memory: requested a row ahead.
template <class T, int VEC>
struct Raw {
    u32x4_t w;
};
template <class T>
struct Raw<T, 1> {
    T w;
};
template <class T, int VEC, bool FREE>
__device__ inline Raw<T, VEC> load_raw(const T* p) {
    if constexpr (VEC == 1) return {p[0]};
    else return {load16<T, FREE>(p)};
}
template <class T, int VEC>
__device__ inline void unpack(const Raw<T, VEC>& r, float (&v)[VEC]) {
    if constexpr (VEC == 1) {
        v[0] = widen(r.w);
    } else if constexpr (sizeof(T) == 2) {  // 8
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(r.w[i] << 16);
            v[2 * i + 1] = __uint_as_float(r.w[i] & 0xffff0000u);
        }
    } else {  // 4
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(r.w[i]);
    }
}
// Elements `skip` on of a chunk (the others belong to the chunk before).
template <class T, int VEC, bool FREE>
__device__ inline void store_vec(T* p, const float (&v)[VEC], uint32_t skip) {
    if constexpr (VEC == 1) {
        store_one(p, v[0]);
    } else {
        if (FREE && skip) {
#pragma unroll
            for (uint32_t e = 0; e < VEC; ++e)
                if (e >= skip) store_one(p + e, v[e]);
            return;
        }
        u32x4_t w;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 2) w[i] = bf16x2(v[2 * i], v[2 * i + 1]);
            else w[i] = __float_as_uint(v[i]);
        }
        store16<T, FREE>(p, w);
    }
}
// First column of a chunk at column c: a row of no whole number of chunks ends with one that begins
// before its place and shares its first columns (skip) with the chunk ahead of it.
template <int VEC, bool FREE>
__device__ inline uint32_t chunk_begin(uint32_t c, uint32_t W) {
    return FREE ? min(c, W - uint32_t(VEC)) : c;
}
// FP32 weights of VEC columns.
template <int VEC>
__device__ inline void load_weights(const float* p, uint64_t at, float none, float (&v)[VEC]) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = p ? p[at + e] : none;
}
template <class T>
__device__ inline float round_to(float x) {
    if constexpr (sizeof(T) == 2) return bf16_widen(bf16_rne(x));
    else return x;
}
// The sum of x over the TPR threads of a row, in every one of them.
template <int TPR>
__device__ inline float row_sum(float x, float* lds) {
#pragma unroll
    for (int d = (TPR < 64 ? TPR : 64) / 2; d; d /= 2) x += __shfl_xor(x, d);
    if constexpr (TPR > 64) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
        __syncthreads();
        x = 0.0f;
#pragma unroll
        for (int w = 0; w < TPR / 64; ++w) x += lds[w];
    }
    return x;
}
template <int TPR>
__device__ inline float2 row_sum2(float2 x, float2* lds) {
#pragma unroll
    for (int d = (TPR < 64 ? TPR : 64) / 2; d; d /= 2) {
        x.x += __shfl_xor(x.x, d);
        x.y += __shfl_xor(x.y, d);
    }
    if constexpr (TPR > 64) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
        __syncthreads();
        x = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < TPR / 64; ++w) {
            x.x += lds[w].x;
            x.y += lds[w].y;
        }
    }
    return x;
}
template <class T>
__device__ inline float elu_to(float t) {
    if constexpr (sizeof(T) == 2) return elu_bf16(t);
    else return elu(t);
}

// Blocks of a launch of n: a dimension has at most 2^32 - 1 threads.  Blocks behind the last have no row.
constexpr uint64_t kNormGridX = uint64_t(1) << 20;
dim3 norm_grid(uint64_t n) {
    const uint64_t y = (n + kNormGridX - 1) / kNormGridX;
    return dim3(uint32_t((n + y - 1) / y), uint32_t(y));
}
__device__ inline uint64_t norm_block() { return uint64_t(blockIdx.y) * gridDim.x + blockIdx.x; }

template <class T, int VEC, int TPR, int ITEMS, bool FREE>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void k_norm_fwd(const NormArgs a) {
    constexpr int BLOCK = TPR < 256 ? 256 : TPR;
    __shared__ float lds[BLOCK / 64];
    const uint64_t row = norm_block() * (BLOCK / TPR) + threadIdx.x / TPR;
    if (row >= a.rows) return;  // (whole row groups; of rows wider than a wave whole blocks)
    const uint32_t t = threadIdx.x % TPR, W = a.width;
    const T* x = static_cast<const T*>(a.x) + row * a.xs;
    float v[ITEMS][VEC];
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        const uint32_t c = (i * TPR + t) * VEC;
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[i][e] = 0.0f;
        if (c < W) unpack<T, VEC>(load_raw<T, VEC, FREE>(x + chunk_begin<VEC, FREE>(c, W)), v[i]);
    }
    if (a.residual) {
        const T* res = static_cast<const T*>(a.residual) + row * a.rs;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const uint32_t c = (i * TPR + t) * VEC;
            if (c < W) {
                const uint32_t s = chunk_begin<VEC, FREE>(c, W);
                float r[VEC];
                unpack<T, VEC>(load_raw<T, VEC, FREE>(res + s), r);
#pragma unroll
                for (int e = 0; e < VEC; ++e) v[i][e] = round_to<T>(v[i][e] + r[e]);
                if (a.sum) store_vec<T, VEC, FREE>(static_cast<T*>(a.sum) + row * a.ss + s, v[i], c - s);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        const uint32_t c = (i * TPR + t) * VEC, skip = c < W ? c - chunk_begin<VEC, FREE>(c, W) : 0;
#pragma unroll
        for (int e = 0; e < VEC; ++e) sum += FREE && uint32_t(e) < skip ? 0.0f : v[i][e];
    }
    const float inv = 1.0f / float(W), mean = row_sum<TPR>(sum, lds) * inv;
    sum = 0.0f;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        const uint32_t c = (i * TPR + t) * VEC;
        if (c >= W) continue;
        const uint32_t skip = c - chunk_begin<VEC, FREE>(c, W);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const float d = FREE && uint32_t(e) < skip ? 0.0f : v[i][e] - mean;
            sum = fmaf(d, d, sum);
        }
    }
    const float rstd = 1.0f / sqrtf(row_sum<TPR>(sum, lds) * inv + a.eps);
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        const uint32_t c = (i * TPR + t) * VEC;
        if (c >= W) continue;
        const uint32_t s = chunk_begin<VEC, FREE>(c, W);
        float g[VEC], b[VEC];
        load_weights<VEC>(a.gamma, s, 1.0f, g);
        load_weights<VEC>(a.beta, s, 0.0f, b);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const float y = fmaf((v[i][e] - mean) * rstd, g[e], b[e]);
            v[i][e] = a.elu ? elu_to<T>(y) : y;
        }
        store_vec<T, VEC, FREE>(static_cast<T*>(a.y) + row * a.ys + s, v[i], c - s);
    }
    if (t == 0) {
        if (a.mean) a.mean[row] = mean;
        if (a.rstd) a.rstd[row] = rstd;
    }
}

// Rows of any width, a block a row: passes over the row where it lies.
template <class T>
__global__ __launch_bounds__(1024) void k_norm_fwd_any(const NormArgs a) {
    __shared__ float lds[16];
    const uint64_t row = norm_block();
    if (row >= a.rows) return;
    const uint32_t W = a.width;
    const T* x = static_cast<const T*>(a.x) + row * a.xs;
    const T* res = a.residual ? static_cast<const T*>(a.residual) + row * a.rs : nullptr;
    const auto h = [&](uint32_t c) {
        const float v = widen(x[c]);
        return res ? round_to<T>(v + widen(res[c])) : v;
    };
    float sum = 0.0f;
    for (uint32_t c = threadIdx.x; c < W; c += 1024) sum += h(c);
    const float mean = row_sum<1024>(sum, lds) / float(W);
    sum = 0.0f;
    for (uint32_t c = threadIdx.x; c < W; c += 1024) sum = fmaf(h(c) - mean, h(c) - mean, sum);
    const float rstd = 1.0f / sqrtf(row_sum<1024>(sum, lds) / float(W) + a.eps);
    for (uint32_t c = threadIdx.x; c < W; c += 1024) {
        const float v = h(c), g = a.gamma ? a.gamma[c] : 1.0f, b = a.beta ? a.beta[c] : 0.0f;
        if (a.sum) store_one(static_cast<T*>(a.sum) + row * a.ss + c, v);
        const float y = fmaf((v - mean) * rstd, g, b);
        store_one(static_cast<T*>(a.y) + row * a.ys + c, a.elu ? elu_to<T>(y) : y);
    }
    if (threadIdx.x == 0) {
        if (a.mean) a.mean[row] = mean;
        if (a.rstd) a.rstd[row] = rstd;
    }
}

template <class T, int VEC, int TPR, int ITEMS, bool FREE>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void k_norm_bwd(const NormArgs a) {
    constexpr int BLOCK = TPR < 256 ? 256 : TPR, GROUPS = BLOCK / TPR;
    __shared__ float2 lds[BLOCK / 64];
    __shared__ float cols[GROUPS > 1 ? GROUPS * TPR * VEC : 1];
    const uint32_t t = threadIdx.x % TPR, group = threadIdx.x / TPR, W = a.width;
    const float inv = 1.0f / float(W);
    float dg[ITEMS][VEC], db[ITEMS][VEC], w[ITEMS][VEC];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        const uint32_t c = (i * TPR + t) * VEC;
#pragma unroll
        for (int e = 0; e < VEC; ++e) dg[i][e] = db[i][e] = w[i][e] = 0.0f;
        if (c < W) load_weights<VEC>(a.gamma, chunk_begin<VEC, FREE>(c, W), 1.0f, w[i]);
    }
    Raw<T, VEC> hr[ITEMS], yr[ITEMS], sr[ITEMS];
    float mean = 0.0f, rstd = 0.0f;
    const auto request = [&](uint64_t row) {
        if (row >= a.rows) return;
        mean = a.mean[row];
        rstd = a.rstd[row];
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const uint32_t c = (i * TPR + t) * VEC;
            if (c >= W) continue;
            const uint32_t s = chunk_begin<VEC, FREE>(c, W);
            hr[i] = load_raw<T, VEC, FREE>(static_cast<const T*>(a.h) + row * a.hs + s);
            yr[i] = load_raw<T, VEC, FREE>(static_cast<const T*>(a.dy) + row * a.dys + s);
            if (a.dsum) sr[i] = load_raw<T, VEC, FREE>(static_cast<const T*>(a.dsum) + row * a.dss + s);
        }
    };
    // (Rows beyond the last leave a row group's lanes idle, not its reductions: all threads make
    // the same rounds.)
    const uint64_t step = uint64_t(gridDim.x) * GROUPS, first = uint64_t(blockIdx.x) * GROUPS;
    request(first + group);
    for (uint64_t r0 = first; r0 < a.rows; r0 += step) {
        const uint64_t row = r0 + group;
        const bool in = row < a.rows;
        float n[ITEMS][VEC], g[ITEMS][VEC];
        Raw<T, VEC> ar[ITEMS];
        float2 s = make_float2(0.0f, 0.0f);
        const float scale = rstd, shift = mean;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const uint32_t c = (i * TPR + t) * VEC;
#pragma unroll
            for (int e = 0; e < VEC; ++e) n[i][e] = g[i][e] = 0.0f;
            if (!in || c >= W) continue;
            unpack<T, VEC>(hr[i], n[i]);
            unpack<T, VEC>(yr[i], g[i]);
            ar[i] = sr[i];
        }
        request(row + step);
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const uint32_t c = (i * TPR + t) * VEC;
            if (!in || c >= W) continue;
            const uint32_t begin = chunk_begin<VEC, FREE>(c, W), skip = c - begin;
            float b[VEC];
            if (a.elu) load_weights<VEC>(a.beta, begin, 0.0f, b);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                n[i][e] = (n[i][e] - shift) * scale;
                if (FREE && uint32_t(e) < skip) n[i][e] = g[i][e] = 0.0f;
                if (a.elu) {
                    const float y = fmaf(n[i][e], w[i][e], b[e]);
                    g[i][e] *= y < 0.0f ? exp_w(y) : 1.0f;
                }
                dg[i][e] = fmaf(g[i][e], n[i][e], dg[i][e]);
                db[i][e] += g[i][e];
                g[i][e] *= w[i][e];
                s.x += g[i][e];
                s.y = fmaf(g[i][e], n[i][e], s.y);
            }
        }
        s = row_sum2<TPR>(s, lds);
        s.x *= inv;
        s.y *= inv;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const uint32_t c = (i * TPR + t) * VEC;
            if (!in || c >= W) continue;
            float add[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) add[e] = 0.0f;
            if (a.dsum) unpack<T, VEC>(ar[i], add);
#pragma unroll
            for (int e = 0; e < VEC; ++e) g[i][e] = fmaf(scale, g[i][e] - s.x - n[i][e] * s.y, add[e]);
            const uint32_t begin = chunk_begin<VEC, FREE>(c, W);
            store_vec<T, VEC, FREE>(static_cast<T*>(a.dx) + row * a.dxs + begin, g[i], c - begin);
        }
    }
    if (!a.part) return;
    // The block's column sums: row groups added in order.
    float* to = a.part + uint64_t(blockIdx.x) * 2 * W;
#pragma unroll
    for (int which = 0; which < 2; ++which)
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const uint32_t c = (i * TPR + t) * VEC;
            float v[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[e] = which ? db[i][e] : dg[i][e];
            if constexpr (GROUPS > 1) {
                __syncthreads();
#pragma unroll
                for (int e = 0; e < VEC; ++e) cols[(group * VEC + e) * TPR + t] = v[e];
                __syncthreads();
                if (group == 0)
#pragma unroll
                    for (int e = 0; e < VEC; ++e)
                        for (int q = 1; q < GROUPS; ++q) v[e] += cols[(q * VEC + e) * TPR + t];
            }
            if (group == 0 && c < W) {
                const uint32_t begin = chunk_begin<VEC, FREE>(c, W);
                if (!FREE || begin == c) {
#pragma unroll
                    for (int e = 0; e < VEC; ++e) to[uint64_t(which) * W + c + e] = v[e];
                } else {
#pragma unroll
                    for (int e = 0; e < VEC; ++e)
                        if (uint32_t(e) >= c - begin) to[uint64_t(which) * W + begin + e] = v[e];
                }
            }
        }
}

template <class T>
__global__ __launch_bounds__(1024) void k_norm_bwd_any(const NormArgs a) {
    __shared__ float2 lds[16];
    const uint64_t row = norm_block();
    if (row >= a.rows) return;
    const uint32_t W = a.width;
    const float mean = a.mean[row], rstd = a.rstd[row];
    const T* h = static_cast<const T*>(a.h) + row * a.hs;
    const T* dy = static_cast<const T*>(a.dy) + row * a.dys;
    const auto terms = [&](uint32_t c, float& n, float& dt) {
        n = (widen(h[c]) - mean) * rstd;
        dt = widen(dy[c]);
        if (a.elu) {
            const float y = fmaf(n, a.gamma ? a.gamma[c] : 1.0f, a.beta ? a.beta[c] : 0.0f);
            if (y < 0.0f) dt *= exp_w(y);
        }
    };
    float2 s = make_float2(0.0f, 0.0f);
    for (uint32_t c = threadIdx.x; c < W; c += 1024) {
        float n, dt;
        terms(c, n, dt);
        dt *= a.gamma ? a.gamma[c] : 1.0f;
        s.x += dt;
        s.y = fmaf(dt, n, s.y);
    }
    s = row_sum2<1024>(s, lds);
    for (uint32_t c = threadIdx.x; c < W; c += 1024) {
        float n, dt;
        terms(c, n, dt);
        const float add = a.dsum ? widen(static_cast<const T*>(a.dsum)[row * a.dss + c]) : 0.0f;
        dt *= a.gamma ? a.gamma[c] : 1.0f;
        store_one(static_cast<T*>(a.dx) + row * a.dxs + c, fmaf(rstd, dt - s.x / float(W) - n * (s.y / float(W)), add));
    }
}
// Column sums of rows of any width: block (columns, row strip), a thread a column.  It runs
// before k_norm_bwd_any, whose dx may take dy's place.
template <class T>
__global__ __launch_bounds__(256) void k_norm_cols_any(const NormArgs a) {
    const uint32_t c = blockIdx.x * 256 + threadIdx.x, W = a.width;
    if (c >= W) return;
    const float w = a.gamma ? a.gamma[c] : 1.0f, b = a.beta ? a.beta[c] : 0.0f;
    float dg = 0.0f, db = 0.0f;
    for (uint64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
        const float n = (widen(static_cast<const T*>(a.h)[row * a.hs + c]) - a.mean[row]) * a.rstd[row];
        float d = widen(static_cast<const T*>(a.dy)[row * a.dys + c]);
        if (a.elu) {
            const float y = fmaf(n, w, b);
            if (y < 0.0f) d *= exp_w(y);
        }
        dg = fmaf(d, n, dg);
        db += d;
    }
    a.part[uint64_t(blockIdx.y) * 2 * W + c] = dg;
    a.part[uint64_t(blockIdx.y) * 2 * W + W + c] = db;
}

// dgamma, dbeta: 32 columns a block, 32 threads a column over the partial rows, added in one
// fixed order.
__global__ __launch_bounds__(1024) void k_norm_sum(const float* __restrict__ part, uint32_t blocks, uint32_t W, float* dgamma,
                                                   float* dbeta) {
    const uint64_t first = norm_block() * 32, c = first + (threadIdx.x & 31);
    const uint32_t g = threadIdx.x >> 5;
    __shared__ float lds[32][33];
    float sum = 0.0f;
    if (c < 2 * uint64_t(W)) {
        float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        uint32_t b = g;
        for (; b + 96 < blocks; b += 128)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[i] += part[uint64_t(b + 32 * i) * 2 * W + c];
        for (; b < blocks; b += 32) s[0] += part[uint64_t(b) * 2 * W + c];
        sum = (s[0] + s[1]) + (s[2] + s[3]);
    }
    lds[g][threadIdx.x & 31] = sum;
    __syncthreads();
    // Column g's sums in lanes 0 to 31 of a half wave
    sum = lds[threadIdx.x & 31][g];
#pragma unroll
    for (int d = 16; d; d /= 2) sum += __shfl_xor(sum, d);
    const uint64_t at = first + g;
    if ((threadIdx.x & 31) || at >= 2 * uint64_t(W)) return;
    if (at < W) {
        if (dgamma) dgamma[at] = sum;
    } else if (dbeta) dbeta[at - W] = sum;
}

// Threads a row and chunks a thread for a row of `chunks` chunks: the fewest threads that keep
// a thread at 4 chunks, 0 where no kernel holds the row.
struct NormShape {
    int tpr, items;
};
NormShape norm_shape(uint64_t chunks) {
    const NormShape all[] = {{16, 1}, {32, 1}, {64, 1}, {64, 2}, {256, 1}, {256, 2}, {512, 2}, {1024, 2}, {1024, 4}};
    for (const NormShape& s : all)
        if (chunks <= uint64_t(s.tpr) * s.items) return s;
    return {0, 0};
}
bool aligned(const void* p, uint64_t stride, int size) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride * uint64_t(size) % 16 == 0;
}

// f(tpr, items) of a shape as compile-time values.
template <int VEC, class F>
void with_shape(NormShape s, F f) {
    const auto as = [&](auto tpr, auto items) {
        if (s.tpr == tpr && s.items == items) f(tpr, items);
    };
    as(std::integral_constant<int, 16>{}, std::integral_constant<int, 1>{});
    if constexpr (VEC > 1) {  // (narrower rows than a chunk have at most 7 columns)
        as(std::integral_constant<int, 32>{}, std::integral_constant<int, 1>{});
        as(std::integral_constant<int, 64>{}, std::integral_constant<int, 1>{});
        as(std::integral_constant<int, 64>{}, std::integral_constant<int, 2>{});
        as(std::integral_constant<int, 256>{}, std::integral_constant<int, 1>{});
        as(std::integral_constant<int, 256>{}, std::integral_constant<int, 2>{});
        as(std::integral_constant<int, 512>{}, std::integral_constant<int, 2>{});
        as(std::integral_constant<int, 1024>{}, std::integral_constant<int, 2>{});
        as(std::integral_constant<int, 1024>{}, std::integral_constant<int, 4>{});
    }
}
// f(elements a load, whether loads are free of alignment) for rows of W columns.
template <class T, class F>
hipError_t with_chunks(uint32_t W, bool wide, F f) {
    constexpr int VEC = 16 / int(sizeof(T));
    if (W < uint32_t(VEC)) return f(std::integral_constant<int, 1>{}, std::false_type{}, norm_shape(W));
    const NormShape s = norm_shape((uint64_t(W) + VEC - 1) / VEC);
    return wide ? f(std::integral_constant<int, VEC>{}, std::false_type{}, s) : f(std::integral_constant<int, VEC>{}, std::true_type{}, s);
}

template <class T>
hipError_t forward(const NormArgs& a, bool wide, hipStream_t st) {
    return with_chunks<T>(a.width, wide, [&](auto vec, auto free, NormShape s) {
        constexpr int VEC = decltype(vec)::value;
        if (!s.tpr) {
            k_norm_fwd_any<T><<<norm_grid(a.rows), 1024, 0, st>>>(a);
            return hipGetLastError();
        }
        with_shape<VEC>(s, [&](auto tpr, auto items) {
            constexpr int TPR = decltype(tpr)::value, BLOCK = TPR < 256 ? 256 : TPR;
            k_norm_fwd<T, VEC, TPR, decltype(items)::value, decltype(free)::value>
                <<<norm_grid((a.rows + BLOCK / TPR - 1) / (BLOCK / TPR)), BLOCK, 0, st>>>(a);
        });
        return hipGetLastError();
    });
}
template <class T>
hipError_t backward(const NormArgs& a, bool wide, uint32_t blocks, hipStream_t st) {
    return with_chunks<T>(a.width, wide, [&](auto vec, auto free, NormShape s) {
        constexpr int VEC = decltype(vec)::value;
        if (!s.tpr) {
            if (a.part) k_norm_cols_any<T><<<dim3((a.width + 255) / 256, blocks), 256, 0, st>>>(a);
            if (a.rows) k_norm_bwd_any<T><<<norm_grid(a.rows), 1024, 0, st>>>(a);
            return hipGetLastError();
        }
        with_shape<VEC>(s, [&](auto tpr, auto items) {
            constexpr int TPR = decltype(tpr)::value;
            k_norm_bwd<T, VEC, TPR, decltype(items)::value, decltype(free)::value><<<blocks, TPR < 256 ? 256 : TPR, 0, st>>>(a);
        });
        return hipGetLastError();
    });
}

}  // namespace

// Blocks are persistent, so no more than run at once: three of 256 threads a CU (131 registers a
// thread).  169K x 256 bf16, residual and ELU: 768 blocks 80 us, 512 97, 1024 108, 2048 91.
// Wider rows take blocks of 256 to 1024 threads, one or two a CU (8190 x 8192: 106 us at 256 blocks and at 512).  Few rows: a block
// a row where a block holds one at a time (100 x 2000, forward and backward: 10.7 us; 13.7 with four rows a block).
// A partial row costs 16 bytes a column, written and read, a row 6 to 16 a column.
uint32_t norm_blocks(uint64_t rows, uint64_t width) {
    const uint64_t most = width > 1024 ? 512 : 768;
    const uint64_t least = width > 1024 ? 1 : 4;  // rows a block
    return uint32_t(std::max<uint64_t>(1, std::min({most, std::max<uint64_t>(256, rows / 32), (rows + least - 1) / least})));
}

hipError_t launch_norm_forward(const NormArgs& a, bool bf16, hipStream_t s) {
    const int size = bf16 ? 2 : 4, vec = 16 / size;
    const bool wide = a.width % uint32_t(vec) == 0 && aligned(a.x, a.xs, size) && aligned(a.y, a.ys, size) &&
                      (!a.residual || aligned(a.residual, a.rs, size)) && (!a.sum || aligned(a.sum, a.ss, size));
    return bf16 ? forward<uint16_t>(a, wide, s) : forward<float>(a, wide, s);
}

hipError_t launch_norm_backward(const NormArgs& a, bool bf16, uint32_t blocks, float* dgamma, float* dbeta, hipStream_t s) {
    const int size = bf16 ? 2 : 4, vec = 16 / size;
    const bool wide = a.width % uint32_t(vec) == 0 && aligned(a.h, a.hs, size) && aligned(a.dy, a.dys, size) &&
                      aligned(a.dx, a.dxs, size) && (!a.dsum || aligned(a.dsum, a.dss, size));
    const hipError_t e = bf16 ? backward<uint16_t>(a, wide, blocks, s) : backward<float>(a, wide, blocks, s);
    if (e != hipSuccess || !a.part) return e;
    return launch_column_sums(a.part, blocks, a.width, dgamma, dbeta, s);
}

hipError_t launch_column_sums(const float* part, uint32_t blocks, uint32_t width, float* a, float* b, hipStream_t s) {
    k_norm_sum<<<norm_grid((2 * uint64_t(width) + 31) / 32), 1024, 0, s>>>(part, blocks, width, a, b);
    return hipGetLastError();
}

}  // namespace gatgpu

namespace {

using namespace gatgpu;

// Rows of the call's storage type: there, aligned to its elements, wide enough, on the device.
int check_rows(gatgpu_ctx* c, const gatgpu_norm_io* io, const char* name, const void* p, uint64_t stride) {
    if (!p) return fail(c, GATGPU_EINVAL, std::string("null ") + name);
    if (reinterpret_cast<uintptr_t>(p) % (io->precision == GATGPU_BF16 ? 2 : 4))
        return fail(c, GATGPU_EINVAL, std::string(name) + " is not aligned to its elements");
    if (stride < io->width || stride > (uint64_t(1) << 44)) return fail(c, GATGPU_EINVAL, std::string(name) + " has a bad row stride");
    return check_device_array(c, p, name);
}
int check_floats(gatgpu_ctx* c, const char* name, const void* p) {
    if (reinterpret_cast<uintptr_t>(p) % 4) return fail(c, GATGPU_EINVAL, std::string(name) + " must be 4-byte aligned");
    return check_device_array(c, p, name);
}
int check_call(gatgpu_ctx* c, const gatgpu_norm_io* io) {
    if (!io) return fail(c, GATGPU_EINVAL, "null arrays");
    if (io->precision != GATGPU_FP32 && io->precision != GATGPU_BF16) return fail(c, GATGPU_EINVAL, "bad precision");
    if (io->width == 0 || io->width > (1u << 30)) return fail(c, GATGPU_EINVAL, "width must be 1 to 2^30");
    if (io->rows >= (uint64_t(1) << 31)) return fail(c, GATGPU_EOVERFLOW, "more than 2^31 - 1 rows");
    if (!(io->eps >= 0.0f) || !std::isfinite(io->eps)) return fail(c, GATGPU_EINVAL, "eps must be finite and not negative");
    if (io->gamma)
        if (int r = check_floats(c, "gamma", io->gamma)) return r;
    if (io->beta)
        if (int r = check_floats(c, "beta", io->beta)) return r;
    return GATGPU_OK;
}
NormArgs make_args(const gatgpu_norm_io* io) {
    NormArgs a;
    a.rows = io->rows;
    a.width = io->width;
    a.elu = io->elu != 0;
    a.eps = io->eps;
    a.gamma = io->gamma;
    a.beta = io->beta;
    a.mean = io->mean;
    a.rstd = io->rstd;
    return a;
}

}  // namespace

extern "C" {

int gatgpu_norm_forward(gatgpu_ctx* c, const gatgpu_norm_io* io) {
    if (!c) return fail(nullptr, GATGPU_EINVAL, "null context");
    DeviceGuard on(c->device);
    if (!on.ok) return fail(c, GATGPU_EDEVICE, "cannot select the context's device");
    if (int r = check_call(c, io)) return r;
    if (!io->rows) return GATGPU_OK;
    if (int r = check_rows(c, io, "x", io->x, io->x_stride)) return r;
    if (int r = check_rows(c, io, "y", io->y, io->y_stride)) return r;
    if (io->residual)
        if (int r = check_rows(c, io, "residual", io->residual, io->residual_stride)) return r;
    if (io->sum) {
        if (!io->residual) return fail(c, GATGPU_EINVAL, "sum without a residual");
        if (int r = check_rows(c, io, "sum", io->sum, io->sum_stride)) return r;
    }
    if (io->mean)
        if (int r = check_floats(c, "mean", io->mean)) return r;
    if (io->rstd)
        if (int r = check_floats(c, "rstd", io->rstd)) return r;
    NormArgs a = make_args(io);
    a.x = io->x;
    a.xs = io->x_stride;
    a.residual = io->residual;
    a.rs = io->residual_stride;
    a.sum = io->sum;
    a.ss = io->sum_stride;
    a.y = io->y;
    a.ys = io->y_stride;
    HIPCHECK(c, launch_norm_forward(a, io->precision == GATGPU_BF16, c->stream));
    return GATGPU_OK;
}

int gatgpu_norm_workspace(gatgpu_ctx* c, uint64_t rows, uint32_t width, uint64_t* bytes) {
    if (!c) return fail(nullptr, GATGPU_EINVAL, "null context");
    if (!bytes) return fail(c, GATGPU_EINVAL, "null output");
    *bytes = uint64_t(norm_blocks(rows, width)) * 2 * uint64_t(width) * 4;
    return GATGPU_OK;
}

int gatgpu_norm_backward(gatgpu_ctx* c, const gatgpu_norm_io* io, void* ws, uint64_t bytes) {
    if (!c) return fail(nullptr, GATGPU_EINVAL, "null context");
    DeviceGuard on(c->device);
    if (!on.ok) return fail(c, GATGPU_EDEVICE, "cannot select the context's device");
    if (int r = check_call(c, io)) return r;
    NormArgs a = make_args(io);
    a.h = io->residual ? io->sum : io->x;
    a.hs = io->residual ? io->sum_stride : io->x_stride;
    a.dy = io->dy;
    a.dys = io->dy_stride;
    a.dsum = io->dsum;
    a.dss = io->dsum_stride;
    a.dx = io->dx;
    a.dxs = io->dx_stride;
    if (io->rows) {
        if (int r = check_rows(c, io, io->residual ? "sum" : "x", a.h, a.hs)) return r;
        if (int r = check_rows(c, io, "dy", io->dy, io->dy_stride)) return r;
        if (int r = check_rows(c, io, "dx", io->dx, io->dx_stride)) return r;
        if (io->dsum)
            if (int r = check_rows(c, io, "dsum", io->dsum, io->dsum_stride)) return r;
        if (!io->mean || !io->rstd) return fail(c, GATGPU_EINVAL, "null mean or rstd");
        if (int r = check_floats(c, "mean", io->mean)) return r;
        if (int r = check_floats(c, "rstd", io->rstd)) return r;
    }
    const uint32_t blocks = norm_blocks(io->rows, io->width);
    if (io->dgamma || io->dbeta) {
        if (io->dgamma)
            if (int r = check_floats(c, "dgamma", io->dgamma)) return r;
        if (io->dbeta)
            if (int r = check_floats(c, "dbeta", io->dbeta)) return r;
        const uint64_t need = uint64_t(blocks) * 2 * uint64_t(io->width) * 4;
        if (bytes < need)
            return fail(c, GATGPU_EINVAL, "workspace of " + std::to_string(bytes) + " bytes, " + std::to_string(need) + " needed");
        if (!ws || reinterpret_cast<uintptr_t>(ws) % 16) return fail(c, GATGPU_EINVAL, "workspace must be 16-byte aligned device memory");
        if (int r = check_device_array(c, ws, "workspace")) return r;
        a.part = static_cast<float*>(ws);
    }
    if (!io->rows && !a.part) return GATGPU_OK;
    HIPCHECK(c, launch_norm_backward(a, io->precision == GATGPU_BF16, blocks, io->dgamma, io->dbeta, c->stream));
    return GATGPU_OK;
}

}  // extern "C"
