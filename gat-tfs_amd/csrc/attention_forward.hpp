// Segment attention, forward: one pass over a row's keys with the running maximum
// and sum of the softmax.
//
//   x_j = scale q.k_j,  y_j = cap tanh(x_j / cap),  s_j = y_j + bias(distance)
//   l' = l 2^(m - m') + sum 2^(s_j - m'),  O' = O 2^(m - m') + sum 2^(s_j - m') v_j,  m' a score near the maximum
// (in units of log2) and out = O / l, lse = ln 2 (m + log2 l).  Capped scores without a bias
// stay within cap: they need no maximum, m is 0 throughout.  (Their weights of 2^-90 to 2^90 fit FP32, but not always
// their products with the values: rows whose sums overflow, or lie low, are taken again with the maximum.)
//
// A wave holds 32 packed query rows; scores are formed transposed (keys x rows), so
// that a lane owns half a row's scores, its statistics are plain registers and the
// weights are the operand of the second product as they stand.  Four waves share tiles
// of 64 keys through LDS, requested a tile ahead; few rows run one wave a block, or eight with a range
// of the keys each, on tiles of 32.  m, l and O are FP32.
//
// Bound by the vector instructions of the scores (four or more and a quarter-rate exponential each) beside the
// products: one graph of 16K nodes, 8 x 64, capped, takes 800 to 830 us, 660 to 690 TFLOP/s where a large product reaches 1086;
// 48 single tokens over up to 24K keys 182 us, the keys' and values' bytes at 5 TB/s.
//
// The loop checks no element for NaN or infinity: a bad value in a tile shows in the sums of
// every row that met it (0 x NaN), and then the block goes over its keys again, letting it
// reach only the rows that see it.
#pragma once
#include "attention_tile.hpp"

namespace gatgpu {
namespace {

// REST: the weights enter the sums as two bf16 each, for the backward pass's delta; with a table as three, which are all of
// FP32's bits, since the table's gradient is FP32.  (24 graphs of 130 to 1300 rows, 8 x 64, both passes: 278 us and that
// gradient 1.3e-6 off with two, 287 us and 3.8e-7 with three.)
// CUTS > 1: each wave of the block walks its own range of the keys, by itself; then they are joined.
template <class T, int D, int NW, int CUTS, int BIAS, bool CAP, bool REST>
__global__ __launch_bounds__(NW * CUTS * 64, (attn_waves<T, D, NW>())) void k_attn_fwd(const AttnArgs a) {
    static_assert(NW == 1 || CUTS == 1, "");
    constexpr int BK = attn_tile_rows<T, NW>(), NB = BK / 32, ROW = lds_row<T, D>(), NF = D * int(sizeof(T)) / 32,
                  DB = D / 32, NBUF = attn_buffers<T, NW>();
    constexpr int SUM = D + 4;  // floats of a row of a wave's sums
    static_assert(CUTS == 1 || 32 * SUM * 4 <= 2 * BK * ROW, "");
    __shared__ __align__(16) char lds[CUTS][2][NBUF][BK * ROW];  // of a wave or block: K, V
    __shared__ float2 lds_stat[CUTS][32];
    extern __shared__ float table[];  // TABLE: [group][256]

    uint64_t task_id;
    int kv;
    if (!attn_task(a, task_id, kv)) return;
    const AttnTask task = a.tasks[task_id];
    const AttnSeg seg = a.segs[task.seg];
    const int lane = int(threadIdx.x) & 63, id = __builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6),
              wave = NW == 1 ? 0 : id, cut = CUTS == 1 ? 0 : id, l32 = lane & 31, half = lane >> 5;
    char(*const lds_k)[BK * ROW] = lds[cut][0];
    char(*const lds_v)[BK * ROW] = lds[cut][1];
    const uint32_t rows = seg.q_len * uint32_t(a.group), row0 = task.at + uint32_t(wave) * 32;
    const bool idle = row0 >= rows;
    const AttnRow w = attn_row(a, seg, min(row0 + uint32_t(l32), rows - 1), kv);
    // Rows are in order of their queries, so the wave's limits are those of its first and last lane.
    const int lim_first = __builtin_amdgcn_readlane(w.lim, 0), lim_last = __builtin_amdgcn_readlane(w.lim, 31);
    const int dim = a.dim;
    const T* kbase = static_cast<const T*>(a.k) + seg.k_begin * a.ks + uint64_t(kv) * dim;
    const T* vbase = static_cast<const T*>(a.v) + seg.k_begin * a.vs + uint64_t(kv) * dim;
    const uint32_t per = CUTS == 1 ? 0 : ((task.hi - task.lo + 31) / 32 + CUTS - 1) / CUTS * 32;  // keys a wave
    const uint32_t begin = min(task.hi, task.lo + uint32_t(cut) * per), end = CUTS == 1 ? task.hi : min(task.hi, begin + per);
    AttnStage<T, D, NW, BK> sk, sv;
    sk.place(a, a.ks, 1);
    sv.place(a, a.vs, 1);
    sk.load(a, kbase, a.ks, 1, begin, end);
    sv.load(a, vbase, a.vs, 1, begin, end);

    uint4 qf[NF];
    {
        const T* q = static_cast<const T*>(a.q) + (seg.q_begin + uint64_t(w.query)) * a.qs + uint64_t(w.head) * dim;
#pragma unroll
        for (int f = 0; f < NF; ++f) {
            const int at = (2 * f + half) * AttnType<T>::kPer;
            qf[f] = at < dim ? *reinterpret_cast<const uint4*>(q + at) : make_uint4(0, 0, 0, 0);
        }
    }
    const uint8_t* drow = BIAS == GATGPU_BIAS_TABLE ? a.dist + seg.dist + uint64_t(w.query) * seg.dist_ld : nullptr;
    AttnDist dist[NB], next_dist[NB];
    if constexpr (BIAS == GATGPU_BIAS_TABLE) {
#pragma unroll
        for (int b = 0; b < NB; ++b) next_dist[b] = load_dist(drow, begin + b * 32 + 4 * half, seg.dist_ld);
        fill_table(a, kv, table);
    }
    const float cc = a.scale * kLog2e;
    const float slope2 = BIAS == GATGPU_BIAS_LINEAR ? a.bias[w.head] * kLog2e : 0.0f;
    const float* trow = table + w.local * 256;
    const bool bounded = CAP && BIAS == GATGPU_BIAS_NONE && a.capped.bounded;

    // Orders the LDS traffic of the waves that share tiles.
    const auto sync = [] {
        if constexpr (NW == 1) wave_sync();
        else lds_barrier();
    };
    f32x16_t acc[DB];
    float m, l;
    const auto pass = [&](auto careful) __attribute__((always_inline)) {
        constexpr bool CAREFUL = decltype(careful)::value;
#pragma unroll
        for (int d = 0; d < DB; ++d) acc[d] = f32x16_t{};
        m = bounded && !CAREFUL ? 0.0f : -INFINITY;
        l = 0.0f;
        uint32_t tile = 0;
        for (uint32_t k0 = begin; k0 < end; k0 += BK, ++tile) {
            const int buf = NBUF == 2 ? int(tile & 1) : 0;
            if (NBUF == 1) sync();
            sk.store(lds_k[buf]);
            sv.store(lds_v[buf]);
#pragma unroll
            for (int b = 0; b < NB; ++b) dist[b] = next_dist[b];
            sync();
            if (k0 + BK < end) {
                sk.load(a, kbase, a.ks, 1, k0 + BK, end);
                sv.load(a, vbase, a.vs, 1, k0 + BK, end);
                if constexpr (BIAS == GATGPU_BIAS_TABLE) {
#pragma unroll
                    for (int b = 0; b < NB; ++b) next_dist[b] = load_dist(drow, k0 + BK + b * 32 + 4 * half, seg.dist_ld);
                }
            }
            if (idle || int(k0) >= lim_last) continue;  // (uniform over the wave; no barrier follows in the tile)
            const float ref = m == -INFINITY ? 0.0f : m;
            f32x16_t s[NB];
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                s[b] = f32x16_t{};
#pragma unroll
                for (int f = 0; f < NF; ++f)
                    s[b] = mfma_rows<T>(
                        s[b], *reinterpret_cast<const uint4*>(lds_k[buf] + (b * 32 + l32) * ROW + f * 32 + half * 16), qf[f]);
                tile_scores<BIAS, CAP, CAREFUL>(a.capped, s[b], cc, ref, slope2, float(w.pos - int(k0) - b * 32 - 4 * half),
                                                dist[b], trow);
                if (REST && D == 128) __builtin_amdgcn_sched_barrier(0);
            }
            if (int(k0) + BK > lim_first) {
                const int left = w.lim - int(k0) - 4 * half;
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        if (b * 32 + 8 * (r / 4) + r % 4 >= left) s[b][r] = -INFINITY;
            }
            if (CAREFUL || !bounded) {
                // The reference m is the maximum of an earlier tile.  It is raised, and the sums with it,
                // only when a score passes it by 2^8: weights of up to 2^8 are as exact as those up to 1.
                float top = s[0][0];
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int r = 0; r < 16; r += 2) top = fmaxf(fmaxf(top, s[b][r]), s[b][r + 1]);
                top = xor32_max(top);
                const bool fresh = m == -INFINITY;  // the row has seen nothing yet
                if (__any(fresh || top > 8.0f)) {
                    const float up = fresh ? top : fmaxf(top, 0.0f), down = up == -INFINITY ? 0.0f : up;
                    const float fall = fresh ? 0.0f : exp2_hw(-up);
                    m = fresh ? top : m + up;
                    l *= fall;
#pragma unroll
                    for (int d = 0; d < DB; ++d)
#pragma unroll
                        for (int r = 0; r < 16; ++r) acc[d][r] *= fall;
#pragma unroll
                    for (int b = 0; b < NB; ++b)
#pragma unroll
                        for (int r = 0; r < 16; ++r) s[b][r] -= down;
                }
            }
            float sum = 0.0f;
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    s[b][r] = exp2_hw(s[b][r]);
                    sum += s[b][r];
                }
            l += sum;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const AttnCols<T> p = to_operand<T>(s[b]);
                const char* vrows = lds_v[buf] + b * 32 * ROW;
                if constexpr (CAREFUL) {
                    const AttnCols<T> seen = seen_operand<T>(s[b]);
#pragma unroll
                    for (int d = 0; d < DB; ++d) acc[d] = mfma_cols_careful<T>(acc[d], vrows, ROW, d * 32, lane, p, seen);
                } else if (!REST) {
#pragma unroll
                    for (int d = 0; d < DB; ++d) acc[d] = mfma_cols<T>(acc[d], load_cols<T>(vrows, ROW, d * 32, lane), p);
                }
                if constexpr (REST) {
                    AttnCols<T> lo, last;
                    rest_operands(s[b], p, lo, BIAS == GATGPU_BIAS_TABLE ? &last : nullptr);
                    if (D == 128) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int d = 0; d < DB; ++d) {
                        const AttnCols<T> v = load_cols<T, CAREFUL ? kClean : kRaw>(vrows, ROW, d * 32, lane);
                        if (!CAREFUL) acc[d] = mfma_cols<T>(acc[d], v, p);
                        acc[d] = mfma_cols<T>(acc[d], v, lo);
                        if constexpr (BIAS == GATGPU_BIAS_TABLE) acc[d] = mfma_cols<T>(acc[d], v, last);
                        if (D == 128) __builtin_amdgcn_sched_barrier(0);
                    }
                }
            }
        }
    };
    if constexpr (BIAS == GATGPU_BIAS_TABLE) lds_barrier();
    pass(std::false_type{});
    bool bad = !idle && nonfinite(acc);
    if (bounded) {  // a row of low scores only: values below 2^-86 would leave FP32
        const float sum = xor32_add(l);
        bad = bad || (sum > 0.0f && sum < 0x1p-40f);
    }
    if (__builtin_expect(NW == 1 ? __any(bad) : __syncthreads_or(bad), 0)) {
        sync();
        sk.load(a, kbase, a.ks, 1, begin, end);
        sv.load(a, vbase, a.vs, 1, begin, end);
        if constexpr (BIAS == GATGPU_BIAS_TABLE) {
#pragma unroll
            for (int b = 0; b < NB; ++b) next_dist[b] = load_dist(drow, begin + b * 32 + 4 * half, seg.dist_ld);
        }
        pass(std::true_type{});
    }
    if (idle) return;
    l = xor32_add(l);
    if constexpr (CUTS > 1) {
        sync();
        float* sums = reinterpret_cast<float*>(&lds[cut][0][0][0]) + l32 * SUM + 4 * half;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                store4<float>(sums, d * 32 + 8 * i, acc[d][4 * i], acc[d][4 * i + 1], acc[d][4 * i + 2], acc[d][4 * i + 3]);
        if (half == 0) lds_stat[cut][l32] = make_float2(m, l);
        lds_barrier();
        // Four columns of a row a thread, the ranges in order.
        const int here = int(min(32u, rows - row0));
        for (int c = int(threadIdx.x); c < here * (D / 4); c += CUTS * 64) {
            const int r = c / (D / 4), col = c % (D / 4) * 4;
            if (col >= dim) continue;
            float top = -INFINITY;
#pragma unroll
            for (int i = 0; i < CUTS; ++i) top = fmaxf(top, lds_stat[i][r].x);
            const float ref = top == -INFINITY ? 0.0f : top;
            float sum = 0.0f, o[4] = {};
#pragma unroll
            for (int i = 0; i < CUTS; ++i) {
                const float2 st = lds_stat[i][r];
                const float f = st.y == 0.0f ? 0.0f : exp2_hw(st.x - ref);  // (a range of which nothing is seen)
                const float4 x = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(&lds[i][0][0][0]) + r * SUM + col);
                sum = fmaf(st.y, f, sum);
                o[0] = fmaf(x.x, f, o[0]);
                o[1] = fmaf(x.y, f, o[1]);
                o[2] = fmaf(x.z, f, o[2]);
                o[3] = fmaf(x.w, f, o[3]);
            }
            const AttnRow row = attn_row(a, seg, row0 + uint32_t(r), kv);
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
            const uint64_t to = seg.q_begin + uint64_t(row.query), at = to * a.os + uint64_t(row.head) * dim + uint64_t(col);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] *= inv;
            store4<T>(a.out, at, o[0], o[1], o[2], o[3]);
            if constexpr (sizeof(T) == 2) {
                if (a.rest) {
                    uint32_t t[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) t[e] = rest_bits(o[e], bf16_hw(o[e]));
                    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.rest) + at) = make_uint2(t[0] | t[1] << 16, t[2] | t[3] << 16);
                }
            }
            if (a.lse && col == 0) a.lse[to * uint64_t(a.heads) + row.head] = sum == 0.0f ? -INFINITY : (top + __log2f(sum)) * kLn2;
        }
        return;
    }
    if (a.part) {  // a range of the keys: joined by k_attn_join
        const uint64_t at = (task_id * uint64_t(a.kv_heads) + uint64_t(kv)) * (NW * 32) + uint64_t(wave * 32 + l32);
        const bool in = row0 + uint32_t(l32) < rows;
        store_part<DB>(a.part, at, acc, half, in);
        if (half == 0 && in) *reinterpret_cast<float2*>(a.stat + at * 2) = make_float2(m, l);
        return;
    }
    store_out<T, DB>(a, seg, w, acc, m, l, half, row0 + uint32_t(l32) < rows);
}

template <class T, int D, int NW, int CUTS, int BIAS, bool CAP>
hipError_t forward_as(const AttnArgs& a, hipStream_t s) {
    const size_t dyn = BIAS == GATGPU_BIAS_TABLE ? size_t(a.group) * 1024 : 0;
    const uint32_t blocks = uint32_t(attn_blocks(a)), threads = NW * CUTS * 64;
    if constexpr (sizeof(T) == 2) {
        if (a.rest) {
            k_attn_fwd<T, D, NW, CUTS, BIAS, CAP, true><<<blocks, threads, dyn, s>>>(a);
            return hipGetLastError();
        }
    }
    k_attn_fwd<T, D, NW, CUTS, BIAS, CAP, false><<<blocks, threads, dyn, s>>>(a);
    return hipGetLastError();
}

template <class T>
hipError_t forward(const AttnArgs& a, int waves, hipStream_t s) {
    return attn_dispatch(a, waves, [&](auto d, auto nw, auto bias, auto cap) {
        return forward_as<T, decltype(d)::value, decltype(nw)::value, 1, decltype(bias)::value, decltype(cap)::value>(a, s);
    });
}
template <class T>
hipError_t forward_cut(const AttnArgs& a, hipStream_t s) {
    return attn_dispatch(a, 1, [&](auto d, auto, auto bias, auto cap) {
        constexpr int D = decltype(d)::value;
        return forward_as<T, D, 1, attention_cuts<T>(D), decltype(bias)::value, decltype(cap)::value>(a, s);
    });
}
// LDS of a block of forward_cut.
template <class T>
size_t forward_cut_lds(int dim, int bias, int group) {
    AttnArgs a;
    a.dim = dim;
    size_t bytes = 0;
    (void)attn_dispatch(a, 1, [&](auto d, auto, auto, auto) {
        constexpr int D = decltype(d)::value;
        bytes = size_t(attention_cuts<T>(D)) * (2 * 32 * lds_row<T, D>() + 32 * sizeof(float2));
        return hipSuccess;
    });
    return bytes + (bias == GATGPU_BIAS_TABLE ? size_t(group) * 1024 : 0);
}

}  // namespace
}  // namespace gatgpu
