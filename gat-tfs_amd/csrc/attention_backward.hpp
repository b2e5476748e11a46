// Segment attention, backward, in two passes without atomics, so that results do
// not depend on an order of arrival.
//
//   p_ij = 2^(s_ij - lse_i),  dp_ij = dout_i.v_j,  delta_i = dout_i.out_i,  ds_ij = p_ij (dp_ij - delta_i)
//   dbias = sum of ds over the pairs of a distance,  dx_ij = ds_ij (1 - tanh^2)
//   dq_i = scale sum_j dx_ij k_j,  dk_j = scale sum_i dx_ij q_i,  dv_j = sum_i p_ij dout_i
//
// The first pass (k_attn_bwd_q) holds 32 query rows a wave and walks the keys, as the
// forward pass does; it forms delta on its way and sums the bias gradient in LDS, a
// column a lane.  The second (k_attn_bwd_kv) holds 32 keys a pair of waves and walks the packed
// query rows of all heads that share them, which sums the shared heads' gradients; its
// weights and score gradients pass through LDS, whose transpose read makes them operands
// that contract over the rows.
// Scores and dp are formed in both: 7 products a pair where 5 would do with atomic
// sums of dq.  (24 graphs of 130 to 1300 rows, 8 x 64, table: 110 us and 115; four sequences of 4K, 16 x 128,
// capped: 600 and 960.)
//
// Weights and score gradients enter the products with Q, K and dout rounded to bf16 (2^-8 of each; the
// gradients' own stored rounding is as large), the bias gradient unrounded.
//
// Where a pass has few blocks, each takes a range of its tile's keys (rows) and leaves FP32 sums, which
// k_attn_grad_join adds in order.
//
// As in the forward pass, no element is checked for NaN or infinity on the way: they show in
// the sums, and the block then goes over its tiles again.  (A bad row of K in the first pass, of Q
// in the second, counts as 0 in the product with the score gradients, which hold a NaN wherever
// the row is seen; rows that give it no weight are left as they were.)
#pragma once
#include "attention_tile.hpp"

namespace gatgpu {
namespace {

// Sum of products of 16 bytes of a and b; bf16 and `rested`: of b with its rest c.
template <class T>
__device__ inline float dot16(uint4 a, uint4 b, uint4 c, bool rested) {
    const uint32_t av[4] = {a.x, a.y, a.z, a.w}, bv[4] = {b.x, b.y, b.z, b.w}, cv[4] = {c.x, c.y, c.z, c.w};
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 2) {
            const float lo = rested ? with_rest(bv[i] & 0xffffu, cv[i] & 0xffffu) : __uint_as_float(bv[i] << 16);
            const float hi = rested ? with_rest(bv[i] >> 16, cv[i] >> 16) : __uint_as_float(bv[i] & 0xffff0000u);
            sum = fmaf(__uint_as_float(av[i] << 16), lo, sum);
            sum = fmaf(__uint_as_float(av[i] & 0xffff0000u), hi, sum);
        } else {
            sum = fmaf(__uint_as_float(av[i]), __uint_as_float(bv[i]), sum);
        }
    }
    return sum;
}

template <class T, int D, int NW, int BIAS, bool CAP>
__global__ __launch_bounds__(NW * 64, (attn_waves<T, D, NW>())) void k_attn_bwd_q(const AttnArgs a) {
    constexpr int BK = attn_tile_rows<T, NW>(), NB = BK / 32, ROW = lds_row<T, D>(), NF = D * int(sizeof(T)) / 32,
                  DB = D / 32, NBUF = attn_buffers<T, NW>(), COLS = NW * 64;
    constexpr bool TABLE = BIAS == GATGPU_BIAS_TABLE;
    __shared__ __align__(16) char lds_k[NBUF][BK * ROW];
    __shared__ __align__(16) char lds_v[NBUF][BK * ROW];
    extern __shared__ float table[];  // TABLE: [group][256], then the table's gradient [buckets][COLS]

    uint64_t task_id;
    int kv;
    if (!attn_task(a, task_id, kv)) return;
    const AttnTask task = a.tasks[task_id];
    const AttnSeg seg = a.segs[task.seg];
    const int lane = int(threadIdx.x) & 63, wave = NW == 1 ? 0 : __builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6),
              l32 = lane & 31, half = lane >> 5;
    const uint32_t rows = seg.q_len * uint32_t(a.group), row0 = task.at + uint32_t(wave) * 32;
    const bool idle = row0 >= rows, live = row0 + uint32_t(l32) < rows;
    const AttnRow w = attn_row(a, seg, min(row0 + uint32_t(l32), rows - 1), kv);
    const int lim_first = __builtin_amdgcn_readlane(w.lim, 0), lim_last = __builtin_amdgcn_readlane(w.lim, 31);
    const int dim = a.dim;
    const bool binned = TABLE && a.dbias;
    float* bins = table + a.group * 256;
    const T* kbase = static_cast<const T*>(a.k) + seg.k_begin * a.ks + uint64_t(kv) * dim;
    const T* vbase = static_cast<const T*>(a.v) + seg.k_begin * a.vs + uint64_t(kv) * dim;
    const uint32_t begin = task.lo, end = task.hi;
    AttnStage<T, D, NW, BK> sk, sv;
    sk.place(a, a.ks, 1);
    sv.place(a, a.vs, 1);
    sk.load(a, kbase, a.ks, 1, begin, end);
    sv.load(a, vbase, a.vs, 1, begin, end);

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
            const bool in = at < dim && !dead;
            qf[f] = in ? *reinterpret_cast<const uint4*>(q + at) : make_uint4(0, 0, 0, 0);
            dof[f] = in ? *reinterpret_cast<const uint4*>(d + at) : make_uint4(0, 0, 0, 0);
            if (in)
                delta += dot16<T>(dof[f], *reinterpret_cast<const uint4*>(o + at),
                                  sizeof(T) == 2 && e ? *reinterpret_cast<const uint4*>(e + at) : make_uint4(0, 0, 0, 0), e != nullptr);
        }
    }
    delta = xor32_add(delta);
    if (live && half == 0 && begin == 0) a.delta[(seg.base + uint64_t(w.query)) * uint64_t(a.heads) + w.head] = delta;

    const uint8_t* drow = TABLE ? a.dist + seg.dist + uint64_t(w.query) * seg.dist_ld : nullptr;
    AttnDist dist[NB], next_dist[NB];
    if constexpr (TABLE) {
#pragma unroll
        for (int b = 0; b < NB; ++b) next_dist[b] = load_dist(drow, begin + b * 32 + 4 * half, seg.dist_ld);
        fill_table(a, kv, table);
    }
    const float cc = a.scale * kLog2e;
    const float slope2 = BIAS == GATGPU_BIAS_LINEAR ? a.bias[w.head] * kLog2e : 0.0f;
    const float uncap = CAP ? 1.0f / a.capped.out : 0.0f;
    const float* trow = table + w.local * 256;

    f32x16_t acc[DB];
    const auto pass = [&](auto careful) __attribute__((always_inline)) {
        constexpr bool CAREFUL = decltype(careful)::value;
#pragma unroll
        for (int d = 0; d < DB; ++d) acc[d] = f32x16_t{};
        if (binned)
            for (int b = 0; b < a.buckets; ++b) bins[b * COLS + threadIdx.x] = 0.0f;
        uint32_t tile = 0;
        for (uint32_t k0 = begin; k0 < end; k0 += BK, ++tile) {
            const int buf = NBUF == 2 ? int(tile & 1) : 0;
            if (NBUF == 1) lds_barrier();
            sk.store(lds_k[buf]);
            sv.store(lds_v[buf]);
#pragma unroll
            for (int b = 0; b < NB; ++b) dist[b] = next_dist[b];
            lds_barrier();
            if (k0 + BK < end) {
                sk.load(a, kbase, a.ks, 1, k0 + BK, end);
                sv.load(a, vbase, a.vs, 1, k0 + BK, end);
                if constexpr (TABLE) {
#pragma unroll
                    for (int b = 0; b < NB; ++b) next_dist[b] = load_dist(drow, k0 + BK + b * 32 + 4 * half, seg.dist_ld);
                }
            }
            if (idle || int(k0) >= lim_last) continue;
            const bool masked = int(k0) + BK > lim_first;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                f32x16_t s = f32x16_t{}, dp = f32x16_t{};
#pragma unroll
                for (int f = 0; f < NF; ++f) {
                    const int at = (b * 32 + l32) * ROW + f * 32 + half * 16;
                    s = mfma_rows<T>(s, *reinterpret_cast<const uint4*>(lds_k[buf] + at), qf[f]);
                    dp = mfma_rows<T>(dp, *reinterpret_cast<const uint4*>(lds_v[buf] + at), dof[f]);
                }
                f32x16_t y;
                score_gradients<BIAS, CAP, CAREFUL>(a.capped, s, dp, y, nullptr, cc, uncap, slope2,
                                                    float(w.pos - int(k0) - b * 32 - 4 * half), dist[b], trow, masked,
                                                    w.lim - int(k0) - b * 32 - 4 * half, lse2, delta);
                if constexpr (TABLE) {
                    if (binned && live) add_bins(bins + threadIdx.x, COLS, a.buckets, dist[b], y);
                }
                if constexpr (CAP) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) y[r] *= s[r];
                }
                const AttnCols<T> p = to_operand<T>(y);
                const char* krows = lds_k[buf] + b * 32 * ROW;
#pragma unroll
                for (int d = 0; d < DB; ++d)
                    acc[d] = mfma_cols<T>(acc[d], load_cols<T, CAREFUL ? kClean : kRaw>(krows, ROW, d * 32, lane), p);
            }
        }
    };
    if constexpr (TABLE) lds_barrier();
    pass(std::false_type{});
    const bool bad = !idle && nonfinite(acc);
    if (__builtin_expect(NW == 1 ? __any(bad) : __syncthreads_or(bad), 0)) {
        if (NW > 1) lds_barrier();
        sk.load(a, kbase, a.ks, 1, begin, end);
        sv.load(a, vbase, a.vs, 1, begin, end);
        if constexpr (TABLE) {
#pragma unroll
            for (int b = 0; b < NB; ++b) next_dist[b] = load_dist(drow, begin + b * 32 + 4 * half, seg.dist_ld);
        }
        pass(std::true_type{});
    }
    if (__builtin_expect(a.part != nullptr, 0))  // a range of the keys: joined by k_attn_grad_join
        store_part<DB>(a.part, (task_id * uint64_t(a.kv_heads) + uint64_t(kv)) * (NW * 32) + uint64_t(wave * 32 + l32), acc, half, live);
    else
        store_rows<T, DB>(a.dq, grow * a.dqs + uint64_t(w.head) * dim, acc, a.scale, half, dim, live);
    if (!binned) return;
    // Each bucket's columns, by head of the group, in one fixed order.
    lds_barrier();
    float* to = a.dbias + ((a.first_part + task_id) * uint64_t(a.kv_heads) + uint64_t(kv)) * uint64_t(a.group * a.buckets);
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

// The pass over keys: a block of PAIRS pairs of waves, 32 keys a pair.  Of each tile of 64 packed query
// rows the first wave of a pair forms the weights and score gradients of rows 0 to 31, the second
// those of rows 32 to 63; both go through LDS, and then the first wave sums dv over the 64 rows, the second
// dk.  So a wave holds one gradient's sums instead of two (64 registers at 128 columns), and with V in LDS at
// bf16's 128 columns two waves a SIMD fit.  Four sequences of 4K, 16 x 128, capped: 960 us so, 1105 with V in
// registers and one wave a SIMD, 1380 with both gradients in a wave.  Vector instructions issue in 39 % of the
// cycles, matrix ones in 30 %, LDS works in 54 %: the waits between a tile's phases bound it.
template <class T, int D, int PAIRS>
struct KvLds {
    static constexpr int kRows = 64, kThreads = PAIRS * 128, kTile = kRows * lds_row<T, D>();
    static constexpr int kTurn = 32 * attn_turn_row<T>();
    static constexpr bool kKeep = sizeof(T) == 2 && D == 128;  // V in LDS, for its 32 registers
    static constexpr int kValues = kKeep ? PAIRS * 32 * lds_row<T, D>() : 16;
    static constexpr int kBytes = 2 * kTile + kRows * 7 * 4 + PAIRS * 4 * kTurn + kValues;
};

template <class T, int D, int PAIRS, int BIAS, bool CAP>
__global__ __launch_bounds__(PAIRS * 128, (sizeof(T) == 2 && (D < 128 || PAIRS > 1) ? (D < 64 ? 3 : 2) : 1)) void k_attn_bwd_kv(const AttnArgs a) {
    using L = KvLds<T, D, PAIRS>;
    constexpr int BQ = L::kRows, ROW = lds_row<T, D>(), NF = D * int(sizeof(T)) / 32, DB = D / 32,
                  PROW = attn_turn_row<T>();
    constexpr bool TABLE = BIAS == GATGPU_BIAS_TABLE;
    __shared__ __align__(16) char lds_q[L::kTile];
    __shared__ __align__(16) char lds_o[L::kTile];
    __shared__ __align__(16) char lds_v[L::kValues];
    __shared__ __align__(16) char lds_p[PAIRS][2][2][L::kTurn];  // weights, score gradients; of the tile's halves
    // Per packed row of a tile: log-sum in units of log2 (+inf: weighs nothing), delta, keys seen,
    // position, slope, first entry of its table, query
    __shared__ float r_lse[BQ], r_delta[BQ], r_slope[BQ];
    __shared__ int r_lim[BQ], r_pos[BQ], r_tab[BQ], r_query[BQ];
    extern __shared__ float table[];  // TABLE: [group][256]

    uint64_t task_id;
    int kv;
    if (!attn_task(a, task_id, kv)) return;
    const AttnTask task = a.tasks[task_id];
    const AttnSeg seg = a.segs[task.seg];
    const int tid = int(threadIdx.x), lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l32 = lane & 31,
              half = lane >> 5, pair = wave >> 1, role = wave & 1;
    const uint32_t key0 = task.at + uint32_t(pair) * 32, key = key0 + uint32_t(l32);
    const bool idle = key0 >= seg.k_len;
    const int dim = a.dim;
    const uint64_t grow = seg.k_begin + min(key, seg.k_len - 1);
    uint4 kf[NF], vf[L::kKeep ? 1 : NF];
    char* const own_v = lds_v + (L::kKeep ? (pair * 32 + l32) * ROW + half * 16 : 0);
    {
        const T* k = static_cast<const T*>(a.k) + grow * a.ks + uint64_t(kv) * dim;
        const T* v = static_cast<const T*>(a.v) + grow * a.vs + uint64_t(kv) * dim;
#pragma unroll
        for (int f = 0; f < NF; ++f) {
            const int at = (2 * f + half) * AttnType<T>::kPer;
            kf[f] = at < dim ? *reinterpret_cast<const uint4*>(k + at) : make_uint4(0, 0, 0, 0);
            const uint4 x = at < dim ? *reinterpret_cast<const uint4*>(v + at) : make_uint4(0, 0, 0, 0);
            if constexpr (L::kKeep) *reinterpret_cast<uint4*>(own_v + 32 * f) = x;  // (both waves of the pair: the same)
            else vf[f] = x;
        }
    }
    const T* qbase = static_cast<const T*>(a.q) + seg.q_begin * a.qs + uint64_t(kv) * uint64_t(a.group * dim);
    const T* obase = static_cast<const T*>(a.dout) + seg.q_begin * a.dos + uint64_t(kv) * uint64_t(a.group * dim);
    const uint32_t rows = seg.q_len * uint32_t(a.group), end = min(task.hi, rows);
    if constexpr (TABLE) fill_table(a, kv, table);
    const float cc = a.scale * kLog2e, uncap = CAP ? 1.0f / a.capped.out : 0.0f;

    f32x16_t acc[DB];
    AttnStage<T, D, PAIRS * 2, BQ> sq, so;
    sq.place(a, a.qs, a.group);
    so.place(a, a.dos, a.group);
    float n_lse = 0.0f, n_delta = 0.0f;
    const auto request = [&](uint32_t r0) __attribute__((always_inline)) {
        sq.load(a, qbase, a.qs, a.group, r0, end);
        so.load(a, obase, a.dos, a.group, r0, end);
        if (tid < BQ) {
            const uint32_t r = r0 + uint32_t(tid);
            n_lse = INFINITY;
            n_delta = 0.0f;
            if (r < end) {
                const uint32_t q = group_of(a, r);
                const uint64_t h = uint64_t(kv) * uint64_t(a.group) + (r - q * uint32_t(a.group));
                const float x = a.lse[(seg.q_begin + q) * uint64_t(a.heads) + h];
                n_lse = x == -INFINITY ? INFINITY : x * kLog2e;
                n_delta = a.delta[(seg.base + q) * uint64_t(a.heads) + h];
            }
        }
    };
    const auto pass = [&](auto careful) __attribute__((always_inline)) {
        constexpr bool CAREFUL = decltype(careful)::value;
#pragma unroll
        for (int d = 0; d < DB; ++d) acc[d] = f32x16_t{};
        if (task.lo < end) request(task.lo);
        for (uint32_t r0 = task.lo; r0 < end; r0 += BQ) {
            lds_barrier();
            sq.store(lds_q);
            so.store(lds_o);
            if (tid < BQ) {
                const AttnRow w = attn_row(a, seg, min(r0 + uint32_t(tid), rows - 1), kv);
                r_lse[tid] = n_lse;
                r_delta[tid] = n_delta;
                r_lim[tid] = w.lim;
                if (BIAS == GATGPU_BIAS_LINEAR) {
                    r_pos[tid] = w.pos;
                    r_slope[tid] = a.bias[w.head] * kLog2e;
                }
                if (TABLE) {
                    r_tab[tid] = w.local * 256;
                    r_query[tid] = w.query;
                }
            }
            lds_barrier();
            if (r0 + BQ < end) request(r0 + BQ);
            const int row = role * 32 + l32, lim = r_lim[row];
            const int lim_last = __builtin_amdgcn_readlane(lim, 31);
            // (Rows are in order of what they see: the tile's last row sees the most.)
            const int lim_tile = __builtin_amdgcn_readfirstlane(r_lim[63]);
            const int lim_half = __builtin_amdgcn_readfirstlane(r_lim[31]);
            if (!idle && int(key0) < lim_last) {
                const bool masked = int(key0) + 32 > __builtin_amdgcn_readlane(lim, 0);
                AttnDist dist{};
                if constexpr (TABLE)
                    dist = load_dist(a.dist + seg.dist + uint64_t(r_query[row]) * seg.dist_ld, key0 + 4 * half, seg.dist_ld);
                f32x16_t s = f32x16_t{}, dp = f32x16_t{};
#pragma unroll
                for (int f = 0; f < NF; ++f) {
                    const int at = row * ROW + f * 32 + half * 16;
                    s = mfma_rows<T>(s, kf[f], *reinterpret_cast<const uint4*>(lds_q + at));
                    uint4 value;
                    if constexpr (L::kKeep) value = *reinterpret_cast<const uint4*>(own_v + 32 * f);
                    else value = vf[f];
                    dp = mfma_rows<T>(dp, value, *reinterpret_cast<const uint4*>(lds_o + at));
                }
                f32x16_t y, p;
                score_gradients<BIAS, CAP, CAREFUL>(
                    a.capped, s, dp, y, &p, cc, uncap, BIAS == GATGPU_BIAS_LINEAR ? r_slope[row] : 0.0f,
                    BIAS == GATGPU_BIAS_LINEAR ? float(r_pos[row] - int(key0) - 4 * half) : 0.0f, dist,
                    table + (TABLE ? r_tab[row] : 0), masked, lim - int(key0) - 4 * half, r_lse[row],
                    r_delta[row]);
                if constexpr (CAP) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) y[r] *= s[r];
                }
                turn_store<T>(lds_p[pair][0][role], to_operand<T>(p), lane);
                turn_store<T>(lds_p[pair][1][role], to_operand<T>(y), lane);
            }
            lds_barrier();
            if (idle || int(key0) >= lim_tile) continue;
            // dv: dout and the weights; dk: Q and the score gradients.
            const char* cols = role ? lds_q : lds_o;
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                if (b == 0 && int(key0) >= lim_half) continue;
                const AttnCols<T> w = load_cols<T>(lds_p[pair][role][b], PROW, 0, lane);
                const char* c = cols + b * 32 * ROW;
#pragma unroll
                for (int d = 0; d < DB; ++d) {
                    if constexpr (CAREFUL) {
                        if (role) acc[d] = mfma_cols<T>(acc[d], load_cols<T, kClean>(c, ROW, d * 32, lane), w);
                        else acc[d] = mfma_cols_careful<T>(acc[d], c, ROW, d * 32, lane, w, nonzero_operand<T>(w));
                    } else {
                        acc[d] = mfma_cols<T>(acc[d], load_cols<T>(c, ROW, d * 32, lane), w);
                    }
                }
            }
            // (The barriers of the next tile keep the turned tiles until every wave has read them.)
        }
    };
    lds_barrier();
    pass(std::false_type{});
    const bool bad = !idle && nonfinite(acc);
    if (__builtin_expect(__syncthreads_or(bad), 0)) {
        lds_barrier();
        pass(std::true_type{});
    }
    const bool in = key < seg.k_len;
    if (__builtin_expect(a.part != nullptr, 0)) {  // a range of the rows: joined by k_attn_grad_join
        const uint64_t plane = (task_id * uint64_t(a.kv_heads) + uint64_t(kv)) * 2 + (role ? 0 : 1);
        store_part<DB>(a.part, plane * (PAIRS * 32) + uint64_t(pair * 32 + l32), acc, half, in);
    } else if (role) store_rows<T, DB>(a.dk, grow * a.dks + uint64_t(kv) * dim, acc, a.scale, half, dim, in);
    else store_rows<T, DB>(a.dv, grow * a.dvs + uint64_t(kv) * dim, acc, 1.0f, half, dim, in);
}

// LDS of a block, as the kernels declare it.
template <class T, int D, int NW>
constexpr size_t lds_q_pass() {
    return size_t(attn_buffers<T, NW>()) * 2 * attn_tile_rows<T, NW>() * lds_row<T, D>();
}
template <class T>
size_t backward_lds(int pass, int dim, int waves, int bias, int group, int buckets) {
    AttnArgs a;
    a.dim = dim;
    size_t bytes = 0;
    (void)attn_dispatch(a, waves, [&](auto d, auto nw, auto, auto) {
        constexpr int D = decltype(d)::value, NW = decltype(nw)::value;
        bytes = pass == kAttnBackwardKv ? size_t(KvLds<T, D, NW == 1 ? 1 : 2>::kBytes) : lds_q_pass<T, D, NW>();
        return hipSuccess;
    });
    if (bias == GATGPU_BIAS_TABLE) {
        bytes += size_t(group) * 1024;
        if (pass == kAttnBackwardQ) bytes += size_t(buckets) * size_t(waves) * 256;
    }
    return bytes;
}

template <class T>
hipError_t backward_q(const AttnArgs& a, int waves, hipStream_t s) {
    return attn_dispatch(a, waves, [&](auto d, auto nw, auto bias, auto cap) {
        constexpr int NW = decltype(nw)::value, BIAS = decltype(bias)::value;
        const size_t dyn = BIAS == GATGPU_BIAS_TABLE ? size_t(a.group) * 1024 + (a.dbias ? size_t(a.buckets) * NW * 256 : 0) : 0;
        k_attn_bwd_q<T, decltype(d)::value, NW, BIAS, decltype(cap)::value>
            <<<uint32_t(attn_blocks(a)), NW * 64, dyn, s>>>(a);
        return hipGetLastError();
    });
}
template <class T>
hipError_t backward_kv(const AttnArgs& a, int waves, hipStream_t s) {
    return attn_dispatch(a, waves, [&](auto d, auto nw, auto bias, auto cap) {
        constexpr int PAIRS = decltype(nw)::value == 1 ? 1 : 2, BIAS = decltype(bias)::value;
        const size_t dyn = BIAS == GATGPU_BIAS_TABLE ? size_t(a.group) * 1024 : 0;
        k_attn_bwd_kv<T, decltype(d)::value, PAIRS, BIAS, decltype(cap)::value>
            <<<uint32_t(attn_blocks(a)), PAIRS * 128, dyn, s>>>(a);
        return hipGetLastError();
    });
}

}  // namespace
}  // namespace gatgpu
