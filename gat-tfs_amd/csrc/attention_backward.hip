// Segment attention, backward, in two passes without atomics, so that results do
// not depend on an order of arrival.
//
//   p_ij = 2^(s_ij - lse_i),  dp_ij = dout_i.v_j,  delta_i = dout_i.out_i,  ds_ij = p_ij (dp_ij - delta_i)
//   dbias = sum of ds over the pairs of a distance,  dx_ij = ds_ij (1 - tanh^2)
//   dq_i = scale sum_j dx_ij k_j,  dk_j = scale sum_i dx_ij q_i,  dv_j = sum_i p_ij dout_i
//
// The first pass (k_attn_bwd_q) holds 32 query rows a wave and walks the keys, as the
// forward pass does; it forms delta on its way and sums the bias gradient in LDS, a
// column a lane.  The second (k_attn_bwd_kv) holds 32 keys a wave and walks the packed
// query rows of all heads that share them, which sums the shared heads' gradients.
// Scores and dp are formed in both: 7 products a pair where 5 would do with atomic
// sums of dq.
#include "attention.hpp"

namespace gatgpu {
namespace {

// Sum of products of 16 bytes of a and b (+ c).
template <class T>
__device__ inline float dot16(uint4 a, uint4 b, uint4 c) {
    const uint32_t av[4] = {a.x, a.y, a.z, a.w}, bv[4] = {b.x, b.y, b.z, b.w}, cv[4] = {c.x, c.y, c.z, c.w};
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 2) {
            sum = fmaf(__uint_as_float(av[i] << 16), __uint_as_float(bv[i] << 16) + __uint_as_float(cv[i] << 16), sum);
            sum = fmaf(__uint_as_float(av[i] & 0xffff0000u),
                       __uint_as_float(bv[i] & 0xffff0000u) + __uint_as_float(cv[i] & 0xffff0000u), sum);
        } else {
            sum = fmaf(__uint_as_float(av[i]), __uint_as_float(bv[i]), sum);
        }
    }
    return sum;
}

template <class T, int D, int NW>
__global__ __launch_bounds__(NW * 64) void k_attn_bwd_q(const AttnArgs a) {
    constexpr int BK = NW == 1 ? 32 : 64, NB = BK / 32, ROW = lds_row<T, D>(), NF = D * int(sizeof(T)) / 32, DB = D / 32;
    constexpr int NBUF = sizeof(T) == 2 ? 2 : 1, NP = 8 * sizeof(T) / 2, COLS = NW * 64;
    __shared__ __align__(16) char lds_k[NBUF][BK * ROW];
    __shared__ __align__(16) char lds_v[NBUF][BK * ROW];
    __shared__ uint32_t bad_tile[NBUF];  // the tile (from 1) with a NaN or an infinity
    extern __shared__ float dyn[];       // table [group][buckets], then its gradient [buckets][COLS]

    uint64_t task_id;
    int kv;
    if (!attn_task(a, task_id, kv)) return;
    const AttnTask task = a.tasks[task_id];
    const AttnSeg seg = a.segs[task.seg];
    const int lane = int(threadIdx.x) & 63, wave = int(threadIdx.x) >> 6, l32 = lane & 31, half = lane >> 5;
    const uint32_t rows = seg.q_len * uint32_t(a.group), row0 = task.at + uint32_t(wave) * 32;
    const bool idle = row0 >= rows, live = row0 + uint32_t(l32) < rows;
    const AttnRow w = attn_row(a, seg, min(row0 + uint32_t(l32), rows - 1), kv);
    const int lim_first = __builtin_amdgcn_readlane(w.lim, 0), lim_last = __builtin_amdgcn_readlane(w.lim, 31);
    const int dim = a.dim;
    const bool tabled = a.bias_kind == GATGPU_BIAS_TABLE, binned = tabled && a.dbias;
    float* bins = dyn + (tabled ? a.group * a.buckets : 0);

    if (threadIdx.x < NBUF) bad_tile[threadIdx.x] = 0;
    if (tabled)
        for (int i = int(threadIdx.x); i < a.group * a.buckets; i += COLS)
            dyn[i] = table_log2(a.bias[kv * a.group * a.buckets + i]);
    if (binned)
        for (int b = 0; b < a.buckets; ++b) bins[b * COLS + threadIdx.x] = 0.0f;
    __syncthreads();

    const uint64_t grow = seg.q_begin + uint64_t(w.query);
    float lse2 = a.lse[grow * uint64_t(a.heads) + w.head];
    const bool dead = !live || lse2 == -INFINITY;  // sees nothing: its weights are 0
    lse2 = dead ? INFINITY : lse2 * kLog2e;
    uint4 qf[NF], dof[NF];
    float delta = 0.0f;
    {
        const T* q = static_cast<const T*>(a.q) + grow * a.qs + uint64_t(w.head) * dim;
        const T* d = static_cast<const T*>(a.dout) + grow * a.dos + uint64_t(w.head) * dim;
        const T* o = static_cast<const T*>(a.out) + grow * a.os + uint64_t(w.head) * dim;
        const T* e = a.rest ? static_cast<const T*>(a.rest) + grow * a.os + uint64_t(w.head) * dim : nullptr;
#pragma unroll
        for (int f = 0; f < NF; ++f) {
            const int at = (2 * f + half) * AttnType<T>::kPer;
            const bool in = at < dim;
            qf[f] = in ? *reinterpret_cast<const uint4*>(q + at) : make_uint4(0, 0, 0, 0);
            dof[f] = in && !dead ? *reinterpret_cast<const uint4*>(d + at) : make_uint4(0, 0, 0, 0);
            if (in && !dead)
                delta += dot16<T>(dof[f], *reinterpret_cast<const uint4*>(o + at),
                                  sizeof(T) == 2 && e ? *reinterpret_cast<const uint4*>(e + at) : make_uint4(0, 0, 0, 0));
        }
    }
    delta = xor32_add(delta);
    if (live && half == 0) a.delta[(seg.base + uint64_t(w.query)) * uint64_t(a.heads) + w.head] = delta;

    const T* kbase = static_cast<const T*>(a.k) + seg.k_begin * a.ks + uint64_t(kv) * dim;
    const T* vbase = static_cast<const T*>(a.v) + seg.k_begin * a.vs + uint64_t(kv) * dim;
    const uint8_t* drow = a.dist ? a.dist + seg.dist + uint64_t(w.query) * seg.dist_ld : nullptr;
    const AttnScore sc(a);
    const float slope2 = a.bias_kind == GATGPU_BIAS_LINEAR ? a.bias[w.head] * kLog2e : 0.0f;
    const float* trow = dyn + w.local * a.buckets;

    f32x16_t acc[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d) acc[d] = f32x16_t{};
    AttnStage<T, D, NW, BK> sk, sv;
    const uint32_t end = task.hi;
    sk.load(kbase, a.ks, 0, end, dim);
    sv.load(vbase, a.vs, 0, end, dim);
    uint32_t tile = 0;
    for (uint32_t k0 = 0; k0 < end; k0 += BK, ++tile) {
        const int buf = NBUF == 2 ? int(tile & 1) : 0;
        if (NBUF == 1) __syncthreads();
        sk.store(lds_k[buf]);
        sv.store(lds_v[buf]);
        if (sk.nonfinite() | sv.nonfinite()) bad_tile[buf] = tile + 1;
        __syncthreads();
        if (k0 + BK < end) {
            sk.load(kbase, a.ks, k0 + BK, end, dim);
            sv.load(vbase, a.vs, k0 + BK, end, dim);
        }
        if (idle || int(k0) >= lim_last) continue;
        const bool bad = bad_tile[buf] == tile + 1;
        const bool masked = int(k0) + BK > lim_first;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            uint32_t dist[4];
            if (tabled) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t key = k0 + b * 32 + 8 * i + 4 * half;
                    dist[i] = key < seg.dist_ld ? *reinterpret_cast<const uint32_t*>(drow + key) : ~0u;
                }
            }
            f32x16_t s = f32x16_t{}, dp = f32x16_t{};
#pragma unroll
            for (int f = 0; f < NF; ++f) {
                const int at = (b * 32 + l32) * ROW + f * 32 + half * 16;
                s = mfma_rows<T>(s, *reinterpret_cast<const uint4*>(lds_k[buf] + at), qf[f]);
                dp = mfma_rows<T>(dp, *reinterpret_cast<const uint4*>(lds_v[buf] + at), dof[f]);
            }
            // y: the biased score in units of log2 over cc; s keeps tanh for its slope.
            float cc = sc.cc;
            f32x16_t y = s;
            if (a.cap > 0.0f) {
                cc = 1.0f;
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    s[r] = tanh_hw(s[r] * sc.cap_in);
                    y[r] = s[r] * sc.cap_out;
                }
            }
            if (a.bias_kind == GATGPU_BIAS_LINEAR) {
                const float base = float(w.pos - int(k0) - b * 32 - 4 * half);
#pragma unroll
                for (int r = 0; r < 16; ++r) y[r] = y[r] * cc - slope2 * fabsf(base - float(8 * (r / 4) + r % 4));
                cc = 1.0f;
            } else if (tabled) {
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const uint32_t d = dist[r / 4] >> (8 * (r % 4)) & 255u;
                    y[r] = d == 255u ? -INFINITY : y[r] * cc + trow[min(int(d), a.buckets - 1)];
                }
                cc = 1.0f;
            }
            if (masked) {
                const int left = w.lim - int(k0) - b * 32 - 4 * half;
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (8 * (r / 4) + r % 4 >= left) y[r] = -INFINITY;
            }
            // A weight of 0 has no gradient, whatever its key or value holds.
            if (masked || tabled || bad) {
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const float p = exp2_hw(y[r] * cc - lse2);
                    y[r] = p == 0.0f ? 0.0f : p * (dp[r] - delta);
                }
            } else {
#pragma unroll
                for (int r = 0; r < 16; ++r) y[r] = exp2_hw(y[r] * cc - lse2) * (dp[r] - delta);
            }
            if (binned && live) {
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const uint32_t d = dist[r / 4] >> (8 * (r % 4)) & 255u;
                    bins[min(int(d), a.buckets - 1) * COLS + threadIdx.x] += y[r];
                }
            }
            if (a.cap > 0.0f) {
#pragma unroll
                for (int r = 0; r < 16; ++r) y[r] *= 1.0f - s[r] * s[r];
            }
            uint32_t p[NP];
            to_operand<T>(y, p);
            const char* krows = lds_k[buf] + b * 32 * ROW;
#pragma unroll
            for (int d = 0; d < DB; ++d)
                acc[d] = __builtin_expect(!bad, 1) ? mfma_cols<T, kRaw>(acc[d], krows, ROW, d * 32, p, lane)
                                                   : mfma_cols<T, kClean>(acc[d], krows, ROW, d * 32, p, lane);
        }
    }
    if (live) {
        const uint64_t to = grow * a.dqs + uint64_t(w.head) * dim;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int at = d * 32 + 8 * i + 4 * half;
                if (at < dim)
                    store4<T>(a.dq, to + at, acc[d][4 * i] * a.scale, acc[d][4 * i + 1] * a.scale,
                              acc[d][4 * i + 2] * a.scale, acc[d][4 * i + 3] * a.scale);
            }
    }
    if (!binned) return;
    // Each bucket's columns, by head of the group, in one fixed order.
    __syncthreads();
    float* to = a.dbias + (task_id * uint64_t(a.kv_heads) + uint64_t(kv)) * uint64_t(a.group * a.buckets);
    for (int b = wave; b < a.buckets; b += NW)
        for (int g = 0; g < a.group; ++g) {
            float sum = 0.0f;
#pragma unroll
            for (int v = 0; v < NW; ++v) {
                const float x = bins[b * COLS + v * 64 + lane];
                sum += int((task.at + uint32_t(v) * 32 + uint32_t(l32)) % uint32_t(a.group)) == g ? x : 0.0f;
            }
#pragma unroll
            for (int d = 32; d; d /= 2) sum += __shfl_xor(sum, d);
            if (lane == 0) to[g * a.buckets + b] = sum;
        }
}

template <class T, int D, int NW>
__global__ __launch_bounds__(NW * 64) void k_attn_bwd_kv(const AttnArgs a) {
    constexpr int BQ = NW == 1 ? 32 : 64, NB = BQ / 32, ROW = lds_row<T, D>(), NF = D * int(sizeof(T)) / 32, DB = D / 32;
    constexpr int NBUF = sizeof(T) == 2 ? 2 : 1, NP = 8 * sizeof(T) / 2;
    __shared__ __align__(16) char lds_q[NBUF][BQ * ROW];
    __shared__ __align__(16) char lds_o[NBUF][BQ * ROW];
    // Per packed row of a tile: log-sum in units of log2 (+inf: weighs nothing), delta, keys seen,
    // position, slope, table row, query
    __shared__ __align__(16) float r_lse[NBUF][BQ], r_delta[NBUF][BQ], r_slope[NBUF][BQ], r_pos[NBUF][BQ];
    __shared__ __align__(16) int r_lim[NBUF][BQ], r_tab[NBUF][BQ], r_query[NBUF][BQ];
    __shared__ uint32_t bad_tile[NBUF];
    extern __shared__ float dyn[];  // table [group][buckets]

    uint64_t task_id;
    int kv;
    if (!attn_task(a, task_id, kv)) return;
    const AttnTask task = a.tasks[task_id];
    const AttnSeg seg = a.segs[task.seg];
    const int tid = int(threadIdx.x), lane = tid & 63, wave = tid >> 6, l32 = lane & 31, half = lane >> 5;
    const uint32_t key0 = task.at + uint32_t(wave) * 32, key = key0 + uint32_t(l32);
    const bool idle = key0 >= seg.k_len;
    const int dim = a.dim;
    const bool tabled = a.bias_kind == GATGPU_BIAS_TABLE;
    if (tid < NBUF) bad_tile[tid] = 0;
    if (tabled)
        for (int i = tid; i < a.group * a.buckets; i += NW * 64) dyn[i] = table_log2(a.bias[kv * a.group * a.buckets + i]);

    uint4 kf[NF], vf[NF];
    const uint64_t grow = seg.k_begin + min(key, seg.k_len - 1);
    {
        const T* k = static_cast<const T*>(a.k) + grow * a.ks + uint64_t(kv) * dim;
        const T* v = static_cast<const T*>(a.v) + grow * a.vs + uint64_t(kv) * dim;
#pragma unroll
        for (int f = 0; f < NF; ++f) {
            const int at = (2 * f + half) * AttnType<T>::kPer;
            kf[f] = at < dim ? *reinterpret_cast<const uint4*>(k + at) : make_uint4(0, 0, 0, 0);
            vf[f] = at < dim ? *reinterpret_cast<const uint4*>(v + at) : make_uint4(0, 0, 0, 0);
        }
    }
    const T* qbase = static_cast<const T*>(a.q) + seg.q_begin * a.qs + uint64_t(kv) * uint64_t(a.group * dim);
    const T* obase = static_cast<const T*>(a.dout) + seg.q_begin * a.dos + uint64_t(kv) * uint64_t(a.group * dim);
    const uint8_t* dcol = tabled ? a.dist + seg.dist + min(key, seg.dist_ld - 1) : nullptr;
    const AttnScore sc(a);
    const uint32_t rows = seg.q_len * uint32_t(a.group), end = min(task.hi, rows);

    f32x16_t acc_k[DB], acc_v[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d) acc_k[d] = acc_v[d] = f32x16_t{};

    AttnStage<T, D, NW, BQ> sq, so;
    float n_lse = 0.0f, n_delta = 0.0f;
    const auto row_load = [&](uint32_t r0) {
        if (tid < BQ) {
            const uint32_t r = r0 + uint32_t(tid);
            n_lse = INFINITY;
            n_delta = 0.0f;
            if (r < end) {
                const uint32_t q = r / uint32_t(a.group);
                const uint64_t h = uint64_t(kv) * uint64_t(a.group) + (r - q * uint32_t(a.group));
                const float x = a.lse[(seg.q_begin + q) * uint64_t(a.heads) + h];
                n_lse = x == -INFINITY ? INFINITY : x * kLog2e;
                n_delta = a.delta[(seg.base + q) * uint64_t(a.heads) + h];
            }
        }
    };
    if (task.lo < end) {
        sq.load_packed(qbase, a.qs, task.lo, end, dim, a.group);
        so.load_packed(obase, a.dos, task.lo, end, dim, a.group);
        row_load(task.lo);
    }
    uint32_t tile = 0;
    __syncthreads();
    for (uint32_t r0 = task.lo; r0 < end; r0 += BQ, ++tile) {
        const int buf = NBUF == 2 ? int(tile & 1) : 0;
        if (NBUF == 1) __syncthreads();
        sq.store(lds_q[buf]);
        so.store(lds_o[buf]);
        if (sq.nonfinite() | so.nonfinite()) bad_tile[buf] = tile + 1;
        if (tid < BQ) {
            const AttnRow w = attn_row(a, seg, min(r0 + uint32_t(tid), rows - 1), kv);
            r_lse[buf][tid] = n_lse;
            r_delta[buf][tid] = n_delta;
            r_lim[buf][tid] = w.lim;
            r_pos[buf][tid] = float(w.pos - int(key0));  // from the first wave's keys
            r_tab[buf][tid] = w.local * a.buckets;
            r_query[buf][tid] = w.query;
            if (a.bias_kind == GATGPU_BIAS_LINEAR) r_slope[buf][tid] = a.bias[w.head] * kLog2e;
        }
        __syncthreads();
        if (r0 + BQ < end) {
            sq.load_packed(qbase, a.qs, r0 + BQ, end, dim, a.group);
            so.load_packed(obase, a.dos, r0 + BQ, end, dim, a.group);
            row_load(r0 + BQ);
        }
        if (idle) continue;
        const bool bad = bad_tile[buf] == tile + 1;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const int lim_first = __builtin_amdgcn_readfirstlane(r_lim[buf][b * 32]);
            const int lim_last = __builtin_amdgcn_readfirstlane(r_lim[buf][b * 32 + 31]);
            if (int(key0) >= lim_last) continue;
            const bool masked = int(key0) + 32 > lim_first;
            const int rb = b * 32 + 4 * half;  // the lane's first row of the block
            f32x16_t s = f32x16_t{}, dp = f32x16_t{};
#pragma unroll
            for (int f = 0; f < NF; ++f) {
                const int at = (b * 32 + l32) * ROW + f * 32 + half * 16;
                s = mfma_rows<T>(s, *reinterpret_cast<const uint4*>(lds_q[buf] + at), kf[f]);
                dp = mfma_rows<T>(dp, *reinterpret_cast<const uint4*>(lds_o[buf] + at), vf[f]);
            }
            float cc = sc.cc;
            f32x16_t y = s;
            if (a.cap > 0.0f) {
                cc = 1.0f;
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    s[r] = tanh_hw(s[r] * sc.cap_in);
                    y[r] = s[r] * sc.cap_out;
                }
            }
            if (a.bias_kind == GATGPU_BIAS_LINEAR) {
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int at = rb + 8 * (r / 4) + r % 4;
                    y[r] = y[r] * cc - r_slope[buf][at] * fabsf(r_pos[buf][at] - float(wave * 32 + l32));
                }
                cc = 1.0f;
            } else if (tabled) {
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int at = rb + 8 * (r / 4) + r % 4;
                    const int d = dcol[uint64_t(r_query[buf][at]) * seg.dist_ld];
                    y[r] = d == 255 ? -INFINITY : y[r] * cc + dyn[r_tab[buf][at] + min(d, a.buckets - 1)];
                }
                cc = 1.0f;
            }
            if (masked) {
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (int(key) >= r_lim[buf][rb + 8 * (r / 4) + r % 4]) y[r] = -INFINITY;
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) y[r] = exp2_hw(y[r] * cc - r_lse[buf][rb + 8 * (r / 4) + r % 4]);
            const char* orows = lds_o[buf] + b * 32 * ROW;
            const char* qrows = lds_q[buf] + b * 32 * ROW;
            uint32_t p[NP];
            to_operand<T>(y, p);
            if (__builtin_expect(!bad, 1)) {
#pragma unroll
                for (int d = 0; d < DB; ++d) acc_v[d] = mfma_cols<T, kRaw>(acc_v[d], orows, ROW, d * 32, p, lane);
            } else {
                uint32_t one[NP];
                seen_operand<T>(y, one);
#pragma unroll
                for (int d = 0; d < DB; ++d) {
                    acc_v[d] = mfma_cols<T, kClean>(acc_v[d], orows, ROW, d * 32, p, lane);
                    const f32x16_t up = mfma_cols<T, kUp>(f32x16_t{}, orows, ROW, d * 32, one, lane);
                    const f32x16_t down = mfma_cols<T, kDown>(f32x16_t{}, orows, ROW, d * 32, one, lane);
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        if (up[r] > 0.0f) acc_v[d][r] += INFINITY;
                        if (down[r] > 0.0f) acc_v[d][r] -= INFINITY;
                    }
                }
            }
            // A weight of 0 has no gradient, whatever its row holds.
            if (masked || tabled || bad) {
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    y[r] = y[r] == 0.0f ? 0.0f : y[r] * (dp[r] - r_delta[buf][rb + 8 * (r / 4) + r % 4]);
            } else {
#pragma unroll
                for (int r = 0; r < 16; ++r) y[r] *= dp[r] - r_delta[buf][rb + 8 * (r / 4) + r % 4];
            }
            if (a.cap > 0.0f) {
#pragma unroll
                for (int r = 0; r < 16; ++r) y[r] *= 1.0f - s[r] * s[r];
            }
            to_operand<T>(y, p);
#pragma unroll
            for (int d = 0; d < DB; ++d)
                acc_k[d] = __builtin_expect(!bad, 1) ? mfma_cols<T, kRaw>(acc_k[d], qrows, ROW, d * 32, p, lane)
                                                     : mfma_cols<T, kClean>(acc_k[d], qrows, ROW, d * 32, p, lane);
        }
    }
    if (key >= seg.k_len) return;
    const uint64_t tk = grow * a.dks + uint64_t(kv) * dim, tv = grow * a.dvs + uint64_t(kv) * dim;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int at = d * 32 + 8 * i + 4 * half;
            if (at >= dim) continue;
            store4<T>(a.dk, tk + at, acc_k[d][4 * i] * a.scale, acc_k[d][4 * i + 1] * a.scale, acc_k[d][4 * i + 2] * a.scale,
                      acc_k[d][4 * i + 3] * a.scale);
            store4<T>(a.dv, tv + at, acc_v[d][4 * i], acc_v[d][4 * i + 1], acc_v[d][4 * i + 2], acc_v[d][4 * i + 3]);
        }
}

// dbias[head][bucket]: the first pass's partial sums of all tasks, in one fixed order; a block a
// (head, bucket).
__global__ __launch_bounds__(256) void k_attn_bias_sum(const AttnArgs a, float* __restrict__ dbias) {
    const int cell = int(blockIdx.x), head = cell / a.buckets, kv = head / a.group;
    const uint64_t step = uint64_t(a.heads) * a.buckets;
    const uint64_t at = uint64_t(kv) * (a.group * a.buckets) + uint64_t(cell - kv * a.group * a.buckets);
    float sum = 0.0f;
    for (uint64_t t = threadIdx.x; t < a.ntasks; t += 256) sum += a.dbias[t * step + at];
    __shared__ float part[256];
    part[threadIdx.x] = sum;
    __syncthreads();
    for (int d = 128; d; d /= 2) {
        if (int(threadIdx.x) < d) part[threadIdx.x] += part[threadIdx.x + d];
        __syncthreads();
    }
    if (threadIdx.x == 0) dbias[cell] = part[0];
}

template <class T, int D>
hipError_t backward_q(const AttnArgs& a, int waves, hipStream_t s) {
    const size_t table = a.bias_kind == GATGPU_BIAS_TABLE ? size_t(a.group) * a.buckets * 4 : 0;
    const size_t dyn = table + (table && a.dbias ? size_t(a.buckets) * waves * 64 * 4 : 0);
    const dim3 grid{uint32_t(attn_blocks(a))};
    if (waves == 1) k_attn_bwd_q<T, D, 1><<<grid, 64, dyn, s>>>(a);
    else k_attn_bwd_q<T, D, 4><<<grid, 256, dyn, s>>>(a);
    return hipGetLastError();
}
template <class T, int D>
hipError_t backward_kv(const AttnArgs& a, int waves, hipStream_t s) {
    const size_t dyn = a.bias_kind == GATGPU_BIAS_TABLE ? size_t(a.group) * a.buckets * 4 : 0;
    const dim3 grid{uint32_t(attn_blocks(a))};
    if (waves == 1) k_attn_bwd_kv<T, D, 1><<<grid, 64, dyn, s>>>(a);
    else k_attn_bwd_kv<T, D, 4><<<grid, 256, dyn, s>>>(a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_attention_backward_q(const AttnArgs& a, bool bf16, int waves, hipStream_t s) {
    switch (attention_width(a.dim)) {
        case 32: return bf16 ? backward_q<uint16_t, 32>(a, waves, s) : backward_q<float, 32>(a, waves, s);
        case 64: return bf16 ? backward_q<uint16_t, 64>(a, waves, s) : backward_q<float, 64>(a, waves, s);
        default: return bf16 ? backward_q<uint16_t, 128>(a, waves, s) : backward_q<float, 128>(a, waves, s);
    }
}
hipError_t launch_attention_backward_kv(const AttnArgs& a, bool bf16, int waves, hipStream_t s) {
    switch (attention_width(a.dim)) {
        case 32: return bf16 ? backward_kv<uint16_t, 32>(a, waves, s) : backward_kv<float, 32>(a, waves, s);
        case 64: return bf16 ? backward_kv<uint16_t, 64>(a, waves, s) : backward_kv<float, 64>(a, waves, s);
        default: return bf16 ? backward_kv<uint16_t, 128>(a, waves, s) : backward_kv<float, 128>(a, waves, s);
    }
}
hipError_t launch_attention_bias_sum(const AttnArgs& a, float* dbias, hipStream_t s) {
    k_attn_bias_sum<<<uint32_t(a.heads * a.buckets), 256, 0, s>>>(a, dbias);
    return hipGetLastError();
}

}  // namespace gatgpu
