// Segment attention of short segments, forward (at most 64 keys) and backward (at most 128).
//
// All keys of a segment are on chip at once, so the softmax is taken in one step, and the
// backward pass forms everything in one go: 5 products a pair, delta = sum p dp from the
// weights themselves (out is not read), dk and dv summed in registers over the rows.
//
// Forward: a wave takes one segment and walks its key/value heads and, within each, the tiles
// of 32 packed query rows.  Backward: a block of a wave per 32 keys does, its waves adding up
// delta and dq through LDS.  The rows of the next step (tile or head) are requested before the
// current one is computed: a step is about as long as a trip to memory, and the bytes of few
// waves a SIMD keep the memory busy.
//
// 1500 segments of 9 to 60 rows, 8 x 32, bf16, table: forward 22 + 15 us (33 to 64 keys, up to 32), backward
// 63 + 33, of which the bias gradient's LDS sums take a third; the rows' bytes would take 35 in all.
//
// Row operands of the forward pass come straight from memory; what is contracted over its rows
// (V; backward K, Q, dout and the turned weights) passes through LDS.
#pragma once
#include "attention_tile.hpp"

namespace gatgpu {
namespace {

// Row operand of 32 rows: lane's row at p (null columns behind dim).
template <class T, int NF>
__device__ inline void load_row(uint4 (&f)[NF], const T* p, int half, int dim) {
    p += half * AttnType<T>::kPer;
    if (dim == 2 * NF * AttnType<T>::kPer) {
#pragma unroll
        for (int i = 0; i < NF; ++i) f[i] = *reinterpret_cast<const uint4*>(p + 2 * i * AttnType<T>::kPer);
    } else {
#pragma unroll
        for (int i = 0; i < NF; ++i) {
            const bool in = (2 * i + half) * AttnType<T>::kPer < dim;
            f[i] = in ? *reinterpret_cast<const uint4*>(p + 2 * i * AttnType<T>::kPer) : make_uint4(0, 0, 0, 0);
        }
    }
}
// The same to LDS, as rows.
template <class T, int D, int NF>
__device__ inline void store_row(char* rows, const uint4 (&f)[NF], int lane) {
    char* at = rows + (lane & 31) * lds_row<T, D>() + (lane >> 5) * 16;
#pragma unroll
    for (int i = 0; i < NF; ++i) *reinterpret_cast<uint4*>(at + 32 * i) = f[i];
}

// The biases of key/value head kv: of one query head a register a lane (its buckets), requested
// ahead; of several straight to the table.
__device__ inline float request_table(const AttnArgs& a, int kv, int lane) {
    return a.group == 1 ? a.bias[kv * a.buckets + min(lane, a.buckets - 1)] : 0.0f;
}
__device__ inline void spread_table(const AttnArgs& a, int kv, int lane, float entry, float* table) {
    if (a.group > 1) return fill_table(a, kv, table);
    entry = table_log2(entry);
    float4 v;
    v.x = __shfl(entry, min(4 * lane, a.buckets - 1));
    v.y = __shfl(entry, min(4 * lane + 1, a.buckets - 1));
    v.z = __shfl(entry, min(4 * lane + 2, a.buckets - 1));
    v.w = __shfl(entry, min(4 * lane + 3, a.buckets - 1));
    if (lane == 63) v.w = -INFINITY;  // GATGPU_HIDDEN
    *reinterpret_cast<float4*>(table + 4 * lane) = v;
}

// REST: as of k_attn_fwd.
template <class T, int D, int KB, int BIAS, bool CAP, bool REST>
__global__ __launch_bounds__(64, (D * int(sizeof(T)) * KB <= 128 ? 2 : 1)) void k_attn_small_fwd(const AttnArgs a) {
    constexpr int ROW = lds_row<T, D>(), NF = D * int(sizeof(T)) / 32, DB = D / 32;
    constexpr bool TABLE = BIAS == GATGPU_BIAS_TABLE;
    __shared__ __align__(16) char lds_v[KB * 32 * ROW];
    extern __shared__ __align__(16) float table[];  // TABLE: [group][256]

    const AttnTask task = a.tasks[blockIdx.x];
    const AttnSeg seg = a.segs[task.seg];
    const int lane = int(threadIdx.x), l32 = lane & 31, half = lane >> 5, dim = a.dim;
    const uint32_t rows = seg.q_len * uint32_t(a.group), tiles = (rows + 31) / 32;
    const float cc = a.scale * kLog2e;

    uint4 nk[KB][NF], nv[KB][NF], nq[NF];
    AttnDist nd[KB];
    float nt = 0.0f;
    const auto request_keys = [&](int kv) {
        if constexpr (TABLE) nt = request_table(a, kv, lane);
#pragma unroll
        for (int b = 0; b < KB; ++b) {
            const uint64_t row = seg.k_begin + min(uint32_t(32 * b + l32), seg.k_len - 1);
            load_row<T, NF>(nk[b], static_cast<const T*>(a.k) + row * a.ks + uint64_t(kv) * dim, half, dim);
            load_row<T, NF>(nv[b], static_cast<const T*>(a.v) + row * a.vs + uint64_t(kv) * dim, half, dim);
        }
    };
    const auto request_rows = [&](int kv, uint32_t tile) {
        const AttnRow w = attn_row(a, seg, min(tile * 32 + uint32_t(l32), rows - 1), kv);
        load_row<T, NF>(nq, static_cast<const T*>(a.q) + (seg.q_begin + uint64_t(w.query)) * a.qs + uint64_t(w.head) * dim,
                        half, dim);
        if constexpr (TABLE) {
            const uint8_t* drow = a.dist + seg.dist + uint64_t(w.query) * seg.dist_ld;
#pragma unroll
            for (int b = 0; b < KB; ++b) nd[b] = load_dist(drow, 32 * b + 4 * half, seg.dist_ld);
        }
    };
    request_keys(int(task.lo));
    request_rows(int(task.lo), 0);
    for (int kv = int(task.lo); kv < int(task.hi); ++kv) {
        uint4 kf[KB][NF];
        wave_sync();
        // (Keys behind the segment's end are copies of its last: their weights are 0.)
#pragma unroll
        for (int b = 0; b < KB; ++b) {
#pragma unroll
            for (int f = 0; f < NF; ++f) kf[b][f] = nk[b][f];
            store_row<T, D, NF>(lds_v + b * 32 * ROW, nv[b], lane);
        }
        if constexpr (TABLE) spread_table(a, kv, lane, nt, table);
        wave_sync();
        for (uint32_t tile = 0; tile < tiles; ++tile) {
            uint4 qf[NF];
#pragma unroll
            for (int f = 0; f < NF; ++f) qf[f] = nq[f];
            AttnDist dist[KB];
#pragma unroll
            for (int b = 0; b < KB; ++b) dist[b] = nd[b];
            if (tile + 1 < tiles) {
                request_rows(kv, tile + 1);
            } else if (kv + 1 < int(task.hi)) {
                request_keys(kv + 1);
                request_rows(kv + 1, 0);
            }
            const uint32_t r = tile * 32 + uint32_t(l32);
            const AttnRow w = attn_row(a, seg, min(r, rows - 1), kv);
            const float slope2 = BIAS == GATGPU_BIAS_LINEAR ? a.bias[w.head] * kLog2e : 0.0f;
            const float* trow = table + w.local * 256;
            const int lim_first = __builtin_amdgcn_readlane(w.lim, 0);
            f32x16_t acc[DB];
            float m, l;
            const auto pass = [&](auto careful) __attribute__((always_inline)) {
                constexpr bool CAREFUL = decltype(careful)::value;
                f32x16_t s[KB];
                float top = -INFINITY;
#pragma unroll
                for (int b = 0; b < KB; ++b) {
                    s[b] = f32x16_t{};
#pragma unroll
                    for (int f = 0; f < NF; ++f) s[b] = mfma_rows<T>(s[b], kf[b][f], qf[f]);
                    tile_scores<BIAS, CAP, CAREFUL>(a.capped, s[b], cc, 0.0f, slope2, float(w.pos - b * 32 - 4 * half), dist[b],
                                                    trow);
                    if (lim_first < 32 * b + 32) {
                        const int left = w.lim - 32 * b - 4 * half;
#pragma unroll
                        for (int e = 0; e < 16; ++e)
                            if (8 * (e / 4) + e % 4 >= left) s[b][e] = -INFINITY;
                    }
#pragma unroll
                    for (int e = 0; e < 16; e += 2) top = fmaxf(fmaxf(top, s[b][e]), s[b][e + 1]);
                }
                m = xor32_max(top);
                const float ref = m == -INFINITY ? 0.0f : m;
                l = 0.0f;
#pragma unroll
                for (int d = 0; d < DB; ++d) acc[d] = f32x16_t{};
#pragma unroll
                for (int b = 0; b < KB; ++b) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        s[b][e] = exp2_hw(s[b][e] - ref);
                        l += s[b][e];
                    }
                    const AttnCols<T> p = to_operand<T>(s[b]);
                    const char* vrows = lds_v + b * 32 * ROW;
#pragma unroll
                    for (int d = 0; d < DB; ++d) {
                        if constexpr (CAREFUL)
                            acc[d] = mfma_cols_careful<T>(acc[d], vrows, ROW, d * 32, lane, p, seen_operand<T>(s[b]));
                        else acc[d] = mfma_cols<T>(acc[d], load_cols<T>(vrows, ROW, d * 32, lane), p);
                    }
                    if constexpr (REST) {
                        AttnCols<T> lo, last;
                        rest_operands(s[b], p, lo, TABLE ? &last : nullptr);
#pragma unroll
                        for (int d = 0; d < DB; ++d) {
                            const AttnCols<T> v = load_cols<T, CAREFUL ? kClean : kRaw>(vrows, ROW, d * 32, lane);
                            acc[d] = mfma_cols<T>(acc[d], v, lo);
                            if constexpr (TABLE) acc[d] = mfma_cols<T>(acc[d], v, last);
                        }
                    }
                }
                l = xor32_add(l);
            };
            pass(std::false_type{});
            if (__builtin_expect(__any(nonfinite(acc)), 0)) pass(std::true_type{});
            store_out<T, DB>(a, seg, w, acc, m, l, half, r < rows);
        }
    }
}

// LDS of the backward pass, a block of NW waves with 32 keys each.  Rows of tiles carry 16 bytes
// behind them (32 cost a quarter of the blocks a CU for few conflicts).
template <class T, int D, int NW>
struct SmallLds {
    static constexpr int kRow = D * int(sizeof(T)) + 16;
    static constexpr int kSum = (D + 4) * 4;  // a row of a wave's share of dq
    static constexpr int kKeys = NW * 32 * kRow, kTile = 32 * kRow, kTurn = NW * 32 * attn_turn_row<T>(),
                         kDelta = 2 * NW * 32 * 4, kShare = NW == 1 ? 0 : NW * 32 * kSum;
    static constexpr int kBytes = 2 * kKeys + 2 * kTile + kTurn + kDelta + kShare;
    static constexpr int kCols = NW * 64 + 1;  // bias gradient: [buckets][kCols], a column a lane
    static size_t bytes(int bias, int group, int buckets, bool binned) {
        return size_t(kBytes) + (bias == GATGPU_BIAS_TABLE ? size_t(group) * 1024 + (binned ? size_t(buckets) * kCols * 4 : 0) : 0);
    }
};

// Orders the LDS traffic of a block; of one wave without a barrier.
template <int NW>
__device__ inline void block_sync() {
    if constexpr (NW == 1) wave_sync();
    else lds_barrier();
}

// Waves a SIMD that its registers are held to: those of 64 bf16 columns, or of 32 FP32 ones and several waves, do not fit
// half a SIMD's registers (1500 segments of up to 60 keys, 8 x 64 in bf16 with a table: 461 us with what did not fit in
// memory, 303 us so; 8 x 32 in FP32: 426, 362).  Those of 32 FP32 columns and one wave do, but for 26 with a table.
template <class T, int D, int NW>
constexpr int small_bwd_waves() {
    return D * int(sizeof(T)) <= 64 || (sizeof(T) == 4 && D == 32 && NW == 1) ? 2 : 1;
}

template <class T, int D, int NW, int BIAS, bool CAP>
__global__ __launch_bounds__(NW * 64, (small_bwd_waves<T, D, NW>())) void k_attn_small_bwd(const AttnArgs a) {
    using L = SmallLds<T, D, NW>;
    constexpr int ROW = L::kRow, NF = D * int(sizeof(T)) / 32, DB = D / 32, PROW = attn_turn_row<T>(), COLS = L::kCols;
    // Of a tile's rows one wave loads Q and dout; of two or four the even ones load Q, the odd ones dout,
    // PART of the row's NF parts of 32 bytes each.
    constexpr int PART = NW <= 2 ? NF : (NF + 1) / 2, LOADS = NW == 1 ? 2 * NF : PART;
    constexpr bool TABLE = BIAS == GATGPU_BIAS_TABLE;
    constexpr bool AHEAD = D * int(sizeof(T)) <= 128;  // the next head's keys are requested ahead
    extern __shared__ __align__(16) char lds[];
    char* const lds_k = lds;
    char* const lds_v = lds_k + L::kKeys;
    char* const lds_q = lds_v + L::kKeys;
    char* const lds_o = lds_q + L::kTile;
    char* const turns = lds_o + L::kTile;
    float* const lds_delta = reinterpret_cast<float*>(turns + L::kTurn);  // [2][NW][32]
    char* const share = turns + L::kTurn + L::kDelta;
    float* const table = reinterpret_cast<float*>(share + L::kShare);  // TABLE: [group][256], then its gradient
    float* const bins = table + a.group * 256;

    const AttnTask task = a.tasks[blockIdx.x];
    const AttnSeg seg = a.segs[task.seg];
    const int tid = int(threadIdx.x), lane = tid & 63, wave = NW == 1 ? 0 : __builtin_amdgcn_readfirstlane(tid >> 6),
              l32 = lane & 31, half = lane >> 5, dim = a.dim;
    const uint32_t rows = seg.q_len * uint32_t(a.group), tiles = (rows + 31) / 32;
    const uint32_t key0 = 32u * uint32_t(wave), key = key0 + uint32_t(l32);
    const bool idle = key0 >= seg.k_len, binned = TABLE && a.dbias;
    const float cc = a.scale * kLog2e, uncap = CAP ? 1.0f / a.capped.out : 0.0f;
    const uint64_t krow = seg.k_begin + min(key, seg.k_len - 1);
    char* const turn = turns + wave * 32 * PROW;
    char* const own_k = lds_k + wave * 32 * ROW;
    char* const own_v = lds_v + wave * 32 * ROW;

    uint4 nk[NF], nv[NF], nr[LOADS];
    const int first_part = NW == 4 ? wave / 2 * PART : 0;
    float nlse = 0.0f, nt = 0.0f;
    AttnDist nd{};
    const auto request_keys = [&](int kv) {
        if constexpr (TABLE) nt = request_table(a, kv, lane);
        load_row<T, NF>(nk, static_cast<const T*>(a.k) + krow * a.ks + uint64_t(kv) * dim, half, dim);
        load_row<T, NF>(nv, static_cast<const T*>(a.v) + krow * a.vs + uint64_t(kv) * dim, half, dim);
    };
    const auto request_rows = [&](int kv, uint32_t tile) {
        const uint32_t r = tile * 32 + uint32_t(l32);
        const AttnRow w = attn_row(a, seg, min(r, rows - 1), kv);
        const uint64_t g = seg.q_begin + uint64_t(w.query);
        const T* q = static_cast<const T*>(a.q) + g * a.qs + uint64_t(w.head) * dim + half * AttnType<T>::kPer;
        const T* o = static_cast<const T*>(a.dout) + g * a.dos + uint64_t(w.head) * dim + half * AttnType<T>::kPer;
        const T* p = wave & 1 ? o : q;
        // (Rows behind the last are 0 and weigh nothing.)
        const int there = r < rows ? dim - half * AttnType<T>::kPer : 0;
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int f = NW == 1 ? i % NF : first_part + i, c = 2 * f * AttnType<T>::kPer;
            nr[i] = c < there ? *reinterpret_cast<const uint4*>((NW > 1 ? p : i < NF ? q : o) + c) : make_uint4(0, 0, 0, 0);
        }
        nlse = r < rows ? a.lse[g * uint64_t(a.heads) + w.head] : -INFINITY;
        if constexpr (TABLE)
            nd = load_dist(a.dist + seg.dist + uint64_t(w.query) * seg.dist_ld, key0 + 4 * half, seg.dist_ld);
    };
    const auto from_lds = [&](const char* rows32, int i) {
        return *reinterpret_cast<const uint4*>(rows32 + l32 * ROW + half * 16 + 32 * i);
    };
    request_keys(int(task.lo));
    if (tiles) request_rows(int(task.lo), 0);
    for (int kv = int(task.lo); kv < int(task.hi); ++kv) {
        f32x16_t acc_k[DB], acc_v[DB];
        if (!AHEAD && kv > int(task.lo)) request_keys(kv);
        block_sync<NW>();
#pragma unroll
        for (int d = 0; d < DB; ++d) acc_k[d] = acc_v[d] = f32x16_t{};
#pragma unroll
        for (int f = 0; f < NF; ++f) {
            *reinterpret_cast<uint4*>(own_k + l32 * ROW + half * 16 + 32 * f) = nk[f];
            *reinterpret_cast<uint4*>(own_v + l32 * ROW + half * 16 + 32 * f) = nv[f];
        }
        if constexpr (TABLE) {
            if (wave == 0 || a.group > 1) spread_table(a, kv, lane, nt, table);
        }
        if (binned)
            for (int b = 0; b < a.buckets; ++b) bins[b * COLS + tid] = 0.0f;
        for (uint32_t tile = 0; tile < tiles; ++tile) {
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                const int f = NW == 1 ? i % NF : first_part + i;
                char* to = NW == 1 ? (i < NF ? lds_q : lds_o) : wave & 1 ? lds_o : lds_q;
                if (NF % PART == 0 || f < NF) *reinterpret_cast<uint4*>(to + l32 * ROW + half * 16 + 32 * f) = nr[i];
            }
            const float lse2 = nlse == -INFINITY ? INFINITY : nlse * kLog2e;
            const AttnDist dist = nd;
            block_sync<NW>();
            if (tile + 1 < tiles) {
                request_rows(kv, tile + 1);
            } else if (kv + 1 < int(task.hi)) {
                if (AHEAD) request_keys(kv + 1);
                request_rows(kv + 1, 0);
            }
            const uint32_t r = tile * 32 + uint32_t(l32);
            const AttnRow w = attn_row(a, seg, min(r, rows - 1), kv);
            const float slope2 = BIAS == GATGPU_BIAS_LINEAR ? a.bias[w.head] * kLog2e : 0.0f;
            const float* trow = table + w.local * 256;
            const int left = w.lim - int(key0) - 4 * half, lim_first = __builtin_amdgcn_readlane(w.lim, 0);
            const float gap = float(w.pos - int(key0) - 4 * half);
            f32x16_t s, y, p, acc_q[DB];
            float delta;
            // Weights p, dp (in y) and the rows' deltas, the same in every wave.  (s keeps the capped
            // scores for their slope.)
            const auto weights = [&](auto careful) {
                constexpr bool CAREFUL = decltype(careful)::value;
                s = y = f32x16_t{};
                if (!idle) {
#pragma unroll
                    for (int f = 0; f < NF; ++f) {
                        s = mfma_rows<T>(s, from_lds(own_k, f), from_lds(lds_q, f));
                        y = mfma_rows<T>(y, from_lds(own_v, f), from_lds(lds_o, f));
                    }
                }
                delta = 0.0f;
                if constexpr (!CAREFUL) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) delta = fmaf(s[e], 0.0f, delta);
                }
                if constexpr (CAP) cap_scores(a.capped, s, 0.0f);
                p = s;
                tile_scores<BIAS, false, CAREFUL>(a.capped, p, CAP ? 1.0f : cc, lse2, slope2, gap, dist, trow);
                if (lim_first < int(key0) + 32) {
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        if (8 * (e / 4) + e % 4 >= left) p[e] = -INFINITY;
                }
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    p[e] = exp2_hw(p[e]);
                    if (CAREFUL && p[e] == 0.0f) y[e] = 0.0f;
                    delta = fmaf(p[e], y[e], delta);
                }
                delta = xor32_add(delta);
                if (NW > 1) {
                    float* all = lds_delta + (CAREFUL ? NW * 32 : 0);
                    if (half == 0) all[wave * 32 + l32] = delta;
                    block_sync<NW>();
                    delta = 0.0f;
#pragma unroll
                    for (int v = 0; v < NW; ++v) delta += all[v * 32 + l32];
                }
            };
            weights(std::false_type{});
            // A NaN or an infinity in V or dout makes dp one and so the row's delta, whatever its weight.  One in K
            // or Q shows in the raw products only, since a mask puts -inf in a score's place: they are added to
            // delta, as 0 or NaN.  Then weights of 0 are kept out of everything.
            const bool careful = __any(delta * 0.0f != 0.0f);
            if (__builtin_expect(careful, 0)) weights(std::true_type{});
#pragma unroll
            for (int d = 0; d < DB; ++d) acc_q[d] = f32x16_t{};
            if (!idle) {
                turn_store<T>(turn, to_operand<T>(p), lane);
#pragma unroll
                for (int e = 0; e < 16; ++e) y[e] = p[e] * (y[e] - delta);
                if (__builtin_expect(careful, 0)) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        y[e] = p[e] == 0.0f ? 0.0f : y[e];
                        if (CAP) s[e] = p[e] == 0.0f ? 0.0f : s[e];  // (its slope)
                    }
                }
                if constexpr (TABLE) {
                    if (binned && r < rows) add_bins(bins + tid, COLS, a.buckets, dist, y);
                }
                if constexpr (CAP) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const float t = s[e] * uncap;
                        y[e] *= fmaf(-t, t, 1.0f);
                    }
                }
                wave_sync();
                const AttnCols<T> pc = load_cols<T>(turn, PROW, 0, lane), yo = to_operand<T>(y);
                wave_sync();
                turn_store<T>(turn, yo, lane);
                wave_sync();
                const AttnCols<T> yc = load_cols<T>(turn, PROW, 0, lane);
                if (__builtin_expect(!careful, 1)) {
#pragma unroll
                    for (int d = 0; d < DB; ++d) {
                        acc_v[d] = mfma_cols<T>(acc_v[d], load_cols<T>(lds_o, ROW, d * 32, lane), pc);
                        acc_q[d] = mfma_cols<T>(acc_q[d], load_cols<T>(own_k, ROW, d * 32, lane), yo);
                        acc_k[d] = mfma_cols<T>(acc_k[d], load_cols<T>(lds_q, ROW, d * 32, lane), yc);
                        if (DB > 1) __builtin_amdgcn_sched_barrier(0);
                    }
                } else {
#pragma unroll
                    for (int d = 0; d < DB; ++d) {
                        acc_v[d] = mfma_cols_careful<T>(acc_v[d], lds_o, ROW, d * 32, lane, pc, nonzero_operand<T>(pc));
                        acc_q[d] = mfma_cols<T>(acc_q[d], load_cols<T, kClean>(own_k, ROW, d * 32, lane), yo);
                        acc_k[d] = mfma_cols<T>(acc_k[d], load_cols<T, kClean>(lds_q, ROW, d * 32, lane), yc);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
            }
            if constexpr (NW == 1) {
                store_rows<T, DB>(a.dq, (seg.q_begin + uint64_t(w.query)) * a.dqs + uint64_t(w.head) * dim, acc_q, a.scale, half,
                                  dim, r < rows);
                wave_sync();
            } else {
                // The waves' shares of dq, added in order; 8 columns a thread at a time.
                float* mine = reinterpret_cast<float*>(share + (wave * 32 + l32) * L::kSum) + 4 * half;
#pragma unroll
                for (int d = 0; d < DB; ++d)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        *reinterpret_cast<float4*>(mine + d * 32 + 8 * i) =
                            make_float4(acc_q[d][4 * i], acc_q[d][4 * i + 1], acc_q[d][4 * i + 2], acc_q[d][4 * i + 3]);
                block_sync<NW>();
                for (int c = tid; c < 32 * D / 8; c += NW * 64) {
                    const uint32_t row = tile * 32 + uint32_t(c / (D / 8));
                    const int col = c % (D / 8) * 8;
                    if (row >= rows || col >= dim) continue;
                    float v[8] = {};
#pragma unroll
                    for (int q = 0; q < NW; ++q) {
                        const float* x = reinterpret_cast<const float*>(share + (q * 32 + c / (D / 8)) * L::kSum) + col;
#pragma unroll
                        for (int e = 0; e < 8; ++e) v[e] += x[e];
                    }
                    const uint32_t query = group_of(a, row);
                    const uint64_t to = (seg.q_begin + query) * a.dqs + uint64_t(kv * a.group) * uint64_t(dim) +
                                        (row - query * uint32_t(a.group)) * uint32_t(dim) + uint32_t(col);
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] *= a.scale;
                    if constexpr (sizeof(T) == 2) {
                        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.dq) + to) =
                            make_uint4(bf16x2(v[0], v[1]), bf16x2(v[2], v[3]), bf16x2(v[4], v[5]), bf16x2(v[6], v[7]));
                    } else {
                        *reinterpret_cast<float4*>(static_cast<float*>(a.dq) + to) = make_float4(v[0], v[1], v[2], v[3]);
                        *reinterpret_cast<float4*>(static_cast<float*>(a.dq) + to + 4) = make_float4(v[4], v[5], v[6], v[7]);
                    }
                }
            }
        }
        // Keys' gradients; then the head's bias gradient.
        store_rows<T, DB>(a.dk, krow * a.dks + uint64_t(kv) * dim, acc_k, a.scale, half, dim, key < seg.k_len);
        store_rows<T, DB>(a.dv, krow * a.dvs + uint64_t(kv) * dim, acc_v, 1.0f, half, dim, key < seg.k_len);
        if (binned) {
            // Two lanes a bucket, which add half of each wave's columns, those of one head of the group at a
            // time.  (With one head the reads are independent of each other and go out together.)
            block_sync<NW>();
            float* to = a.dbias + (uint64_t(task.at) * uint64_t(a.kv_heads) + uint64_t(kv)) * uint64_t(a.group * a.buckets);
            for (int b = wave * 32 + l32; b < (a.buckets + 31) / 32 * 32; b += NW * 32) {
                const float* row = bins + min(b, a.buckets - 1) * COLS + 32 * half;
                for (int g = 0; g < a.group; ++g) {
                    float sum = 0.0f;
                    if (a.group == 1) {
#pragma unroll
                        for (int v = 0; v < NW; ++v)
#pragma unroll
                            for (int i = 0; i < 32; ++i) sum += row[v * 64 + i];
                    } else {
#pragma unroll
                        for (int v = 0; v < NW; ++v)
                            for (int i = g; i < 32; i += a.group) sum += row[v * 64 + i];
                    }
                    sum = xor32_add(sum);
                    if (half == 0 && b < a.buckets) to[g * a.buckets + b] = sum;
                }
            }
        }
    }
}

// f(key blocks): 1 for segments of at most 32 keys.
template <class T>
hipError_t small_forward(const AttnArgs& a, int blocks, hipStream_t s) {
    return attn_dispatch(a, 1, [&](auto d, auto, auto bias, auto cap) {
        constexpr int D = decltype(d)::value, BIAS = decltype(bias)::value;
        constexpr bool CAP = decltype(cap)::value;
        if constexpr (attention_small_width<T>(D)) {
            const size_t dyn = BIAS == GATGPU_BIAS_TABLE ? size_t(a.group) * 1024 : 0;
            const auto launch = [&](auto kb, auto rest) {
                k_attn_small_fwd<T, D, decltype(kb)::value, BIAS, CAP, decltype(rest)::value><<<uint32_t(a.ntasks), 64, dyn, s>>>(a);
                return hipGetLastError();
            };
            constexpr std::integral_constant<int, 1> one{};
            if constexpr (sizeof(T) == 2) {
                constexpr std::integral_constant<int, 2> two{};
                if (blocks == 2) return a.rest ? launch(two, std::true_type{}) : launch(two, std::false_type{});
                if (a.rest) return launch(one, std::true_type{});
            }
            if (blocks == 1) return launch(one, std::false_type{});
            return hipErrorInvalidValue;
        } else {
            return hipErrorInvalidValue;
        }
    });
}
// f(waves): 1, 2 or 4, for segments of at most 32 keys a wave.
template <class T, class F>
hipError_t small_backward_with(const AttnArgs& a, int waves, F f) {
    return attn_dispatch(a, 1, [&](auto d, auto, auto bias, auto cap) {
        constexpr int D = decltype(d)::value;
        if constexpr (D * int(sizeof(T)) <= 256) {
            if (waves == 1) return f(d, std::integral_constant<int, 1>{}, bias, cap);
            if (waves == 2) return f(d, std::integral_constant<int, 2>{}, bias, cap);
            return f(d, std::integral_constant<int, 4>{}, bias, cap);
        } else {
            return hipErrorInvalidValue;
        }
    });
}
template <class T>
hipError_t small_backward(const AttnArgs& a, int waves, hipStream_t s) {
    return small_backward_with<T>(a, waves, [&](auto d, auto nw, auto bias, auto cap) {
        constexpr int D = decltype(d)::value, NW = decltype(nw)::value, BIAS = decltype(bias)::value;
        const size_t bytes = SmallLds<T, D, NW>::bytes(BIAS, a.group, a.buckets, a.dbias != nullptr);
        k_attn_small_bwd<T, D, NW, BIAS, decltype(cap)::value><<<uint32_t(a.ntasks), NW * 64, bytes, s>>>(a);
        return hipGetLastError();
    });
}
template <class T>
size_t small_backward_lds(int dim, int waves, int bias, int group, int buckets) {
    AttnArgs a;
    a.dim = dim;
    size_t bytes = ~size_t(0);
    (void)small_backward_with<T>(a, waves, [&](auto d, auto nw, auto, auto) {
        bytes = SmallLds<T, decltype(d)::value, decltype(nw)::value>::bytes(bias, group, buckets, true);
        return hipSuccess;
    });
    return bytes;
}

}  // namespace
}  // namespace gatgpu
