// Segment attention: the joins of partial results, and the choice of a kernel's storage type.
#include <cmath>

#include "attention_tile.hpp"

namespace gatgpu {
namespace {

// Joins the key ranges of a split tile: 32 rows, 8 threads each.
template <class T, int D>
__global__ __launch_bounds__(256) void k_attn_join(const AttnArgs a, const AttnTask* __restrict__ tiles) {
    const AttnTask tile = tiles[blockIdx.x / uint32_t(a.kv_heads)];
    const int kv = int(blockIdx.x % uint32_t(a.kv_heads));
    const AttnSeg seg = a.segs[tile.seg];
    const uint32_t rows = seg.q_len * uint32_t(a.group), row = tile.at + threadIdx.x / 8;
    if (row >= rows) return;
    const AttnRow w = attn_row(a, seg, row, kv);
    constexpr int N = D / 32;  // float4 a thread: columns 4 (8 i + threadIdx.x % 8)
    const uint64_t step = uint64_t(a.kv_heads) * 32;
    const uint64_t first = (uint64_t(tile.lo) * uint64_t(a.kv_heads) + uint64_t(kv)) * 32 + threadIdx.x / 8;
    float m = -INFINITY;
    for (uint32_t t = 0; t < tile.hi; ++t) m = fmaxf(m, a.stat[(first + t * step) * 2]);
    const float ref = m == -INFINITY ? 0.0f : m;
    float l = 0.0f;
    float4 o[N];
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = make_float4(0, 0, 0, 0);
    for (uint32_t t = 0; t < tile.hi; ++t) {
        const float2 st = *reinterpret_cast<const float2*>(a.stat + (first + t * step) * 2);
        const float f = exp2_hw(st.x - ref);
        if (st.y == 0.0f) continue;  // a range of which nothing is seen
        l += st.y * f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float4 p = *reinterpret_cast<const float4*>(a.part + (first + t * step) * D + 4 * (8 * i + threadIdx.x % 8));
            o[i].x += p.x * f;
            o[i].y += p.y * f;
            o[i].z += p.z * f;
            o[i].w += p.w * f;
        }
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const uint64_t to = (seg.q_begin + uint64_t(w.query)) * a.os + uint64_t(w.head) * a.dim;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int at = 4 * (8 * i + int(threadIdx.x) % 8);
        if (at >= a.dim) continue;
        const float v[4] = {o[i].x * inv, o[i].y * inv, o[i].z * inv, o[i].w * inv};
        store4<T>(a.out, to + at, v[0], v[1], v[2], v[3]);
        if (sizeof(T) == 2 && a.rest) {
            float d[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) d[e] = v[e] - bf16_widen(bf16_hw(v[e]));
            store4<T>(a.rest, to + at, d[0], d[1], d[2], d[3]);
        }
    }
    if (a.lse && threadIdx.x % 8 == 0)
        a.lse[(seg.q_begin + uint64_t(w.query)) * uint64_t(a.heads) + w.head] =
            l == 0.0f ? -INFINITY : (m + __log2f(l)) * kLn2;
}

// dbias[head][bucket]: partial sums of all parts, in one fixed order.  A block takes 32 cells, 32
// threads a cell.
__global__ __launch_bounds__(1024) void k_attn_bias_sum(const float* __restrict__ part, uint64_t parts, uint32_t cells,
                                                        float* __restrict__ dbias) {
    const uint32_t c = blockIdx.x * 32 + (threadIdx.x & 31), g = threadIdx.x >> 5;
    __shared__ float lds[32][33];
    float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (c < cells) {
        uint64_t p = g;
        for (; p + 96 < parts; p += 128)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[i] += part[(p + 32 * i) * cells + c];
        for (; p < parts; p += 32) s[0] += part[p * cells + c];
    }
    lds[g][threadIdx.x & 31] = (s[0] + s[1]) + (s[2] + s[3]);
    __syncthreads();
    float sum = lds[threadIdx.x & 31][g];
#pragma unroll
    for (int d = 16; d; d /= 2) sum += __shfl_xor(sum, d);
    if ((threadIdx.x & 31) == 0 && blockIdx.x * 32 + g < cells) dbias[blockIdx.x * 32 + g] = sum;
}

template <class T, int D>
hipError_t join(const AttnArgs& a, const AttnTask* tiles, uint64_t ntiles, hipStream_t s) {
    k_attn_join<T, D><<<uint32_t(ntiles * uint64_t(a.kv_heads)), 256, 0, s>>>(a, tiles);
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
    // 2^y and sums of 2^30 of them stay inside FP32, and 2^-y far above its smallest values.
    c.bounded = out <= 90.0;
    return c;
}

hipError_t launch_attention_join(const AttnArgs& a, bool bf16, const AttnTask* tiles, uint64_t ntiles, hipStream_t s) {
    switch (attention_width(a.dim)) {
        case 32: return bf16 ? join<uint16_t, 32>(a, tiles, ntiles, s) : join<float, 32>(a, tiles, ntiles, s);
        case 64: return bf16 ? join<uint16_t, 64>(a, tiles, ntiles, s) : join<float, 64>(a, tiles, ntiles, s);
        default: return bf16 ? join<uint16_t, 128>(a, tiles, ntiles, s) : join<float, 128>(a, tiles, ntiles, s);
    }
}
hipError_t launch_attention_bias_sum(const AttnArgs& a, uint64_t parts, float* dbias, hipStream_t s) {
    const uint32_t cells = uint32_t(a.heads) * uint32_t(a.buckets);
    k_attn_bias_sum<<<(cells + 31) / 32, 1024, 0, s>>>(a.dbias, parts, cells, dbias);
    return hipGetLastError();
}

}  // namespace gatgpu
