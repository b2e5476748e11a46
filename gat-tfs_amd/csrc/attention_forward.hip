// Segment attention, forward: one pass over a row's keys with the running maximum
// and sum of the softmax.
//
//   x_j = scale q.k_j,  y_j = cap tanh(x_j / cap),  s_j = y_j + bias(distance)
//   m' = max(m, max s_j),  l' = l 2^(m - m') + sum 2^(s_j - m'),  O' = O 2^(m - m') + sum 2^(s_j - m') v_j
// (in units of log2) and out = O / l, lse = ln 2 (m + log2 l).
//
// A wave holds 32 packed query rows; scores are formed transposed (keys x rows), so
// that a lane owns half a row's scores, its statistics are plain registers and the
// weights are the operand of the second product as they stand (attention.hpp).  Four
// waves share tiles of 64 keys through LDS; short segments and split key ranges run
// one wave a block on tiles of 32.  m, l and O are FP32.
#include "attention.hpp"

namespace gatgpu {
namespace {

template <class T, int D, int NW>
__global__ __launch_bounds__(NW * 64) void k_attn_fwd(const AttnArgs a) {
    constexpr int BK = NW == 1 ? 32 : 64, NB = BK / 32, ROW = lds_row<T, D>(), NF = D * int(sizeof(T)) / 32, DB = D / 32;
    constexpr int NBUF = sizeof(T) == 2 ? 2 : 1, NP = 8 * sizeof(T) / 2;
    __shared__ __align__(16) char lds_k[NBUF][BK * ROW];
    __shared__ __align__(16) char lds_v[NBUF][BK * ROW];
    __shared__ uint32_t bad_tile[NBUF];  // the tile (counted from 1) whose values hold a NaN or an infinity
    extern __shared__ float table[];     // [group][buckets], in units of log2

    uint64_t task_id;
    int kv;
    if (!attn_task(a, task_id, kv)) return;
    const AttnTask task = a.tasks[task_id];
    const AttnSeg seg = a.segs[task.seg];
    const int lane = int(threadIdx.x) & 63, wave = int(threadIdx.x) >> 6, l32 = lane & 31, half = lane >> 5;
    const uint32_t rows = seg.q_len * uint32_t(a.group), row0 = task.at + uint32_t(wave) * 32;
    const bool idle = row0 >= rows;
    const uint32_t row = min(row0 + uint32_t(l32), rows - 1);
    const AttnRow w = attn_row(a, seg, row, kv);
    // Rows are in order of their queries, so the wave's limits are those of its first and last lane.
    const int lim_first = __builtin_amdgcn_readlane(w.lim, 0), lim_last = __builtin_amdgcn_readlane(w.lim, 31);
    const int dim = a.dim;

    if (threadIdx.x < NBUF) bad_tile[threadIdx.x] = 0;
    if (a.bias_kind == GATGPU_BIAS_TABLE)
        for (int i = int(threadIdx.x); i < a.group * a.buckets; i += NW * 64)
            table[i] = table_log2(a.bias[kv * a.group * a.buckets + i]);

    __syncthreads();

    uint4 qf[NF];
    {
        const T* q = static_cast<const T*>(a.q) + (seg.q_begin + uint64_t(w.query)) * a.qs + uint64_t(w.head) * dim;
#pragma unroll
        for (int f = 0; f < NF; ++f) {
            const int at = (2 * f + half) * AttnType<T>::kPer;
            qf[f] = at < dim ? *reinterpret_cast<const uint4*>(q + at) : make_uint4(0, 0, 0, 0);
        }
    }
    const T* kbase = static_cast<const T*>(a.k) + seg.k_begin * a.ks + uint64_t(kv) * dim;
    const T* vbase = static_cast<const T*>(a.v) + seg.k_begin * a.vs + uint64_t(kv) * dim;
    const uint8_t* drow = a.dist ? a.dist + seg.dist + uint64_t(w.query) * seg.dist_ld : nullptr;
    const AttnScore sc(a);
    const float slope2 = a.bias_kind == GATGPU_BIAS_LINEAR ? a.bias[w.head] * kLog2e : 0.0f;
    const float* trow = table + w.local * a.buckets;

    f32x16_t acc[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d) acc[d] = f32x16_t{};
    float m = -INFINITY, l = 0.0f;

    AttnStage<T, D, NW, BK> sk, sv;
    const uint32_t end = task.hi;
    sk.load(kbase, a.ks, task.lo, end, dim);
    sv.load(vbase, a.vs, task.lo, end, dim);
    uint32_t tile = 0;
    for (uint32_t k0 = task.lo; k0 < end; k0 += BK, ++tile) {
        const int buf = NBUF == 2 ? int(tile & 1) : 0;
        if (NBUF == 1) __syncthreads();
        sk.store(lds_k[buf]);
        sv.store(lds_v[buf]);
        if (sv.nonfinite()) bad_tile[buf] = tile + 1;
        __syncthreads();
        if (k0 + BK < end) {
            sk.load(kbase, a.ks, k0 + BK, end, dim);
            sv.load(vbase, a.vs, k0 + BK, end, dim);
        }
        if (idle || int(k0) >= lim_last) continue;  // (uniform over the wave; no barrier follows in the tile)
        const bool bad = bad_tile[buf] == tile + 1;

        uint32_t dist[NB][4];
        if (a.bias_kind == GATGPU_BIAS_TABLE) {
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t key = k0 + b * 32 + 8 * i + 4 * half;
                    dist[b][i] = key < seg.dist_ld ? *reinterpret_cast<const uint32_t*>(drow + key) : ~0u;
                }
        }
        f32x16_t s[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            s[b] = f32x16_t{};
#pragma unroll
            for (int f = 0; f < NF; ++f) {
                const uint4 kf = *reinterpret_cast<const uint4*>(lds_k[buf] + (b * 32 + l32) * ROW + f * 32 + half * 16);
                s[b] = mfma_rows<T>(s[b], kf, qf[f]);
            }
        }
        float cc = sc.cc;
        if (a.cap > 0.0f) {
            cc = 1.0f;
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r) s[b][r] = sc.cap_out * tanh_hw(s[b][r] * sc.cap_in);
        }
        if (a.bias_kind == GATGPU_BIAS_LINEAR) {
            const float base = float(w.pos - int(k0) - 4 * half);
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    s[b][r] = s[b][r] * cc - slope2 * fabsf(base - float(b * 32 + 8 * (r / 4) + r % 4));
            cc = 1.0f;
        } else if (a.bias_kind == GATGPU_BIAS_TABLE) {
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const uint32_t d = dist[b][r / 4] >> (8 * (r % 4)) & 255u;
                    const float t = trow[min(int(d), a.buckets - 1)];
                    s[b][r] = d == 255u ? -INFINITY : s[b][r] * cc + t;
                }
            cc = 1.0f;
        }
        if (int(k0) + BK > lim_first) {
            const int left = w.lim - int(k0) - 4 * half;
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (b * 32 + 8 * (r / 4) + r % 4 >= left) s[b][r] = -INFINITY;
        }
        float top = s[0][0];
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r) top = fmaxf(top, s[b][r]);
        top = xor32_max(top) * cc;
        const float next = fmaxf(m, top), ref = next == -INFINITY ? 0.0f : next;  // nothing seen yet: every weight is 0
        if (__any(next > m)) {
            const float fall = exp2_hw(m - ref);
            l *= fall;
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[d][r] *= fall;
        }
        m = next;
        float sum = 0.0f;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                s[b][r] = exp2_hw(s[b][r] * cc - ref);
                sum += s[b][r];
            }
        l += sum;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            uint32_t p[NP];
            to_operand<T>(s[b], p);
            const char* vrows = lds_v[buf] + b * 32 * ROW;
            if (__builtin_expect(!bad, 1)) {
#pragma unroll
                for (int d = 0; d < DB; ++d) acc[d] = mfma_cols<T, kRaw>(acc[d], vrows, ROW, d * 32, p, lane);
            } else {
                // A NaN or an infinity reaches the rows that give its key some weight, and no other.
                uint32_t one[NP];
                seen_operand<T>(s[b], one);
#pragma unroll
                for (int d = 0; d < DB; ++d) {
                    acc[d] = mfma_cols<T, kClean>(acc[d], vrows, ROW, d * 32, p, lane);
                    const f32x16_t up = mfma_cols<T, kUp>(f32x16_t{}, vrows, ROW, d * 32, one, lane);
                    const f32x16_t down = mfma_cols<T, kDown>(f32x16_t{}, vrows, ROW, d * 32, one, lane);
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        if (up[r] > 0.0f) acc[d][r] += INFINITY;
                        if (down[r] > 0.0f) acc[d][r] -= INFINITY;
                    }
                }
            }
        }
    }
    if (idle) return;
    l = xor32_add(l);
    if (a.part) {  // a range of the keys: joined by k_attn_join
        const uint64_t at = (task_id * uint64_t(a.kv_heads) + uint64_t(kv)) * (NW * 32) + uint64_t(wave * 32 + l32);
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                store4<float>(a.part, at * D + d * 32 + 8 * i + 4 * half, acc[d][4 * i], acc[d][4 * i + 1], acc[d][4 * i + 2],
                              acc[d][4 * i + 3]);
        if (half == 0) *reinterpret_cast<float2*>(a.stat + at * 2) = make_float2(m, l);
        return;
    }
    if (row0 + uint32_t(l32) >= rows) return;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // nothing seen: 0
    const uint64_t to = (seg.q_begin + uint64_t(w.query)) * a.os + uint64_t(w.head) * dim;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int at = d * 32 + 8 * i + 4 * half;
            if (at >= dim) continue;
            float o[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = acc[d][4 * i + e] * inv;
            store4<T>(a.out, to + at, o[0], o[1], o[2], o[3]);
            if (sizeof(T) == 2 && a.rest) {  // what the rounding took
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] -= bf16_widen(bf16_hw(o[e]));
                store4<T>(a.rest, to + at, o[0], o[1], o[2], o[3]);
            }
        }
    if (a.lse && half == 0)
        a.lse[(seg.q_begin + uint64_t(w.query)) * uint64_t(a.heads) + w.head] =
            l == 0.0f ? -INFINITY : (m + __log2f(l)) * kLn2;
}

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

template <class T, int D>
hipError_t forward(const AttnArgs& a, int waves, hipStream_t s) {
    const size_t dyn = a.bias_kind == GATGPU_BIAS_TABLE ? size_t(a.group) * a.buckets * 4 : 0;
    const dim3 grid{uint32_t(attn_blocks(a))};
    if (waves == 1) k_attn_fwd<T, D, 1><<<grid, 64, dyn, s>>>(a);
    else k_attn_fwd<T, D, 4><<<grid, 256, dyn, s>>>(a);
    return hipGetLastError();
}
template <class T, int D>
hipError_t join(const AttnArgs& a, const AttnTask* tiles, uint64_t ntiles, hipStream_t s) {
    k_attn_join<T, D><<<uint32_t(ntiles * uint64_t(a.kv_heads)), 256, 0, s>>>(a, tiles);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_attention_forward(const AttnArgs& a, bool bf16, int waves, hipStream_t s) {
    switch (attention_width(a.dim)) {
        case 32: return bf16 ? forward<uint16_t, 32>(a, waves, s) : forward<float, 32>(a, waves, s);
        case 64: return bf16 ? forward<uint16_t, 64>(a, waves, s) : forward<float, 64>(a, waves, s);
        default: return bf16 ? forward<uint16_t, 128>(a, waves, s) : forward<float, 128>(a, waves, s);
    }
}
hipError_t launch_attention_join(const AttnArgs& a, bool bf16, const AttnTask* tiles, uint64_t ntiles, hipStream_t s) {
    switch (attention_width(a.dim)) {
        case 32: return bf16 ? join<uint16_t, 32>(a, tiles, ntiles, s) : join<float, 32>(a, tiles, ntiles, s);
        case 64: return bf16 ? join<uint16_t, 64>(a, tiles, ntiles, s) : join<float, 64>(a, tiles, ntiles, s);
        default: return bf16 ? join<uint16_t, 128>(a, tiles, ntiles, s) : join<float, 128>(a, tiles, ntiles, s);
    }
}

}  // namespace gatgpu
