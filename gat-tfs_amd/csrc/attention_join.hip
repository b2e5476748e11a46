// Segment attention: the joins of partial results, and the choice of a kernel's storage type.
#include <cmath>

#include "attention_tile.hpp"

namespace gatgpu {
namespace {

// Joins the key ranges of a split tile's rows: a wave a row and key/value head, a lane a range's
// weight and D / 64 columns of the sums.  Ranges are added in order.
template <class T, int D>
__global__ __launch_bounds__(64) void k_attn_join(const AttnArgs a, const AttnTask* __restrict__ tiles, uint32_t per_tile) {
    const uint32_t cell = blockIdx.x / per_tile;  // (tile, head)
    const AttnTask tile = tiles[cell / uint32_t(a.kv_heads)];
    const int kv = int(cell % uint32_t(a.kv_heads)), lane = int(threadIdx.x);
    const AttnSeg seg = a.segs[tile.seg];
    const uint32_t rows = seg.q_len * uint32_t(a.group), local = blockIdx.x % per_tile, row = tile.at + local;
    if (row >= rows) return;
    const AttnRow w = attn_row(a, seg, row, kv);
    constexpr int N = D > 64 ? D / 64 : 1;
    const uint64_t step = uint64_t(a.kv_heads) * 32, first = (uint64_t(tile.lo) * uint64_t(a.kv_heads) + uint64_t(kv)) * 32 + local;
    float m = -INFINITY;
    for (uint32_t t = uint32_t(lane); t < tile.hi; t += 64) m = fmaxf(m, a.stat[(first + t * step) * 2]);
#pragma unroll
    for (int d = 32; d; d /= 2) m = fmaxf(m, __shfl_xor(m, d));
    const float ref = m == -INFINITY ? 0.0f : m;
    float l = 0.0f, o[N] = {};
    const bool mine = D >= 64 || lane < D;
    const int col = lane * N;
    for (uint32_t t0 = 0; t0 < tile.hi; t0 += 64) {
        const uint32_t t = t0 + uint32_t(lane), n = min(64u, tile.hi - t0);
        float f = 0.0f, part_l = 0.0f;
        if (t < tile.hi) {
            const float2 st = *reinterpret_cast<const float2*>(a.stat + (first + t * step) * 2);
            f = st.y == 0.0f ? 0.0f : exp2_hw(st.x - ref);  // (a range of which nothing is seen)
            part_l = st.y * f;
        }
        for (uint32_t i = 0; i < n; i += 16) {  // 16 ranges' columns in flight
            float v[16][N];
#pragma unroll
            for (int u = 0; u < 16; ++u)
#pragma unroll
                for (int e = 0; e < N; ++e)
                    v[u][e] = mine ? a.part[(first + (t0 + min(i + u, n - 1)) * step) * D + uint64_t(col + e)] : 0.0f;
#pragma unroll
            for (int u = 0; u < 16; ++u) {
                if (i + u >= n) break;
                const float fi = __shfl(f, int(i) + u);
                l += __shfl(part_l, int(i) + u);
#pragma unroll
                for (int e = 0; e < N; ++e) o[e] = fmaf(v[u][e], fi, o[e]);
            }
        }
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const uint64_t at = (seg.q_begin + uint64_t(w.query)) * a.os + uint64_t(w.head) * a.dim + uint64_t(col);
    if (mine && col < a.dim) {  // (dim is a multiple of 8)
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const float v = o[e] * inv;
            if constexpr (sizeof(T) == 2) {
                const uint16_t b = bf16_hw(v);
                static_cast<uint16_t*>(a.out)[at + e] = b;
                if (a.rest) static_cast<uint16_t*>(a.rest)[at + e] = uint16_t(rest_bits(v, b));
            } else {
                static_cast<float*>(a.out)[at + e] = v;
            }
        }
    }
    if (a.lse && lane == 0)
        a.lse[(seg.q_begin + uint64_t(w.query)) * uint64_t(a.heads) + w.head] =
            l == 0.0f ? -INFINITY : (m + __log2f(l)) * kLn2;
}

// Adds the partial gradients of a split tile, in order: a wave a row and key/value head.  KEYS: dk and dv
// of `height` keys a tile, else dq of `height` packed query rows.
template <class T, int D, bool KEYS>
__global__ __launch_bounds__(64) void k_attn_grad_join(const AttnArgs a, const AttnTask* __restrict__ tiles, uint32_t height) {
    constexpr int N = D > 64 ? D / 64 : 1, PLANES = KEYS ? 2 : 1;
    const uint32_t local = blockIdx.x % height, cell = blockIdx.x / height;
    const AttnTask tile = tiles[cell / uint32_t(a.kv_heads)];
    const int kv = int(cell % uint32_t(a.kv_heads)), col = int(threadIdx.x) * N;
    const AttnSeg seg = a.segs[tile.seg];
    const uint32_t row = tile.at + local;
    if (row >= (KEYS ? seg.k_len : seg.q_len * uint32_t(a.group)) || col >= a.dim) return;
    const uint64_t step = uint64_t(a.kv_heads) * PLANES * height * D;
#pragma unroll
    for (int plane = 0; plane < PLANES; ++plane) {
        const float* p = a.part + (((uint64_t(tile.lo) * uint64_t(a.kv_heads) + uint64_t(kv)) * PLANES + plane) * height + local) * D + col;
        float sum[N] = {};
        for (uint32_t t = 0; t < tile.hi; t += 8) {  // 8 ranges in flight
            float x[8][N];
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i)
#pragma unroll
                for (int e = 0; e < N; ++e) x[i][e] = t + i < tile.hi ? p[(t + i) * step + e] : 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int e = 0; e < N; ++e) sum[e] += x[i][e];
        }
        void* base;
        uint64_t at;
        if (KEYS) {
            base = plane ? a.dv : a.dk;
            at = (seg.k_begin + row) * (plane ? a.dvs : a.dks) + uint64_t(kv) * uint64_t(a.dim);
        } else {
            const AttnRow w = attn_row(a, seg, row, kv);
            base = a.dq;
            at = (seg.q_begin + uint64_t(w.query)) * a.dqs + uint64_t(w.head) * uint64_t(a.dim);
        }
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const float v = sum[e] * (plane ? 1.0f : a.scale);
            if constexpr (sizeof(T) == 2) static_cast<uint16_t*>(base)[at + uint64_t(col + e)] = bf16_hw(v);
            else static_cast<float*>(base)[at + uint64_t(col + e)] = v;
        }
    }
}

// dbias[head][bucket]: partial sums of all parts, in one fixed order.  A block takes 8 cells, 128
// threads a cell.
__global__ __launch_bounds__(1024) void k_attn_bias_sum(const float* __restrict__ part, uint64_t parts, uint32_t cells,
                                                        float* __restrict__ dbias) {
    const uint32_t c = blockIdx.x * 8 + (threadIdx.x & 7), g = threadIdx.x >> 3;
    __shared__ float lds[128][9];
    float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (c < cells) {
        uint64_t p = g;
        for (; p + 384 < parts; p += 512)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[i] += part[(p + 128 * i) * cells + c];
        for (; p < parts; p += 128) s[0] += part[p * cells + c];
    }
    lds[g][threadIdx.x & 7] = (s[0] + s[1]) + (s[2] + s[3]);
    __syncthreads();
    const uint32_t cell = threadIdx.x >> 7, lane = threadIdx.x & 127;  // two waves a cell
    float sum = lds[lane][cell];
#pragma unroll
    for (int d = 32; d; d /= 2) sum += __shfl_xor(sum, d);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6][0] = sum;
    __syncthreads();
    if (lane == 0 && blockIdx.x * 8 + cell < cells) dbias[blockIdx.x * 8 + cell] = lds[2 * cell][0] + lds[2 * cell + 1][0];
}

template <class T, int D>
hipError_t grad_join(const AttnArgs& a, bool keys, const AttnTask* tiles, uint64_t ntiles, uint32_t height, hipStream_t s) {
    const uint32_t blocks = uint32_t(ntiles * uint64_t(a.kv_heads) * height);
    if (keys) k_attn_grad_join<T, D, true><<<blocks, 64, 0, s>>>(a, tiles, height);
    else k_attn_grad_join<T, D, false><<<blocks, 64, 0, s>>>(a, tiles, height);
    return hipGetLastError();
}
template <class T, int D>
hipError_t join(const AttnArgs& a, const AttnTask* tiles, uint64_t ntiles, uint32_t rows, hipStream_t s) {
    k_attn_join<T, D><<<uint32_t(ntiles * uint64_t(a.kv_heads) * rows), 64, 0, s>>>(a, tiles, rows);
    return hipGetLastError();
}

}  // namespace

AttnCap attention_cap(float scale, float cap) {
    AttnCap c;
    if (!(cap > 0.0f)) return c;
    const double fit2[3] = {0.9999999439, -0.3333021063, 0.1307500945};
    const double fit4[5] = {0.9999999871, -0.3333307189, 0.13324829, -0.05298924118, 0.01714131905};
    const double in = double(scale) / double(cap), out = double(cap) * 1.4426950408889634;
    c.in = float(in);
    c.out = float(out);
    bool fits = true;
    double f = out * in;
    for (int k = 0; k < 5; ++k, f *= in * in) {
        if (k < 3) c.poly2[k] = float(fit2[k] * f);
        c.poly4[k] = float(fit4[k] * f);
        fits = fits && std::isfinite(c.poly4[k]);
    }
    if (fits) {
        c.near2 = float(0.18 / in);
        c.near4 = float(0.5 / in);
    }
    // 2^y and sums of 2^30 of them stay inside FP32, and 2^-y far above its smallest values.  (The forward kernel sees to
    // their products with large and small values.)
    c.bounded = out <= 90.0;
    return c;
}

hipError_t launch_attention_join(const AttnArgs& a, bool bf16, const AttnTask* tiles, uint64_t ntiles, uint32_t rows,
                                 hipStream_t s) {
    switch (attention_width(a.dim)) {
        case 32: return bf16 ? join<uint16_t, 32>(a, tiles, ntiles, rows, s) : join<float, 32>(a, tiles, ntiles, rows, s);
        case 64: return bf16 ? join<uint16_t, 64>(a, tiles, ntiles, rows, s) : join<float, 64>(a, tiles, ntiles, rows, s);
        default: return bf16 ? join<uint16_t, 128>(a, tiles, ntiles, rows, s) : join<float, 128>(a, tiles, ntiles, rows, s);
    }
}
hipError_t launch_attention_grad_join(const AttnArgs& a, bool bf16, bool keys, const AttnTask* tiles, uint64_t ntiles, uint32_t height,
                                      hipStream_t s) {
    switch (attention_width(a.dim)) {
        case 32:
            return bf16 ? grad_join<uint16_t, 32>(a, keys, tiles, ntiles, height, s) : grad_join<float, 32>(a, keys, tiles, ntiles, height, s);
        case 64:
            return bf16 ? grad_join<uint16_t, 64>(a, keys, tiles, ntiles, height, s) : grad_join<float, 64>(a, keys, tiles, ntiles, height, s);
        default:
            return bf16 ? grad_join<uint16_t, 128>(a, keys, tiles, ntiles, height, s) : grad_join<float, 128>(a, keys, tiles, ntiles, height, s);
    }
}
hipError_t launch_attention_bias_sum(const AttnArgs& a, uint64_t parts, float* dbias, hipStream_t s) {
    const uint32_t cells = uint32_t(a.heads) * uint32_t(a.buckets);
    k_attn_bias_sum<<<(cells + 7) / 8, 1024, 0, s>>>(a.dbias, parts, cells, dbias);
    return hipGetLastError();
}

}  // namespace gatgpu
