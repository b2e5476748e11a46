// Attention over a paged 8-bit cache (cache_attention.hpp says how operands lie).
//
// Few rows a request: bound by the cache's bytes, short calls by a launch and its chain of dependent reads.  The work, tiles
// of 64 keys times tiles of 16 rows over all requests, is cut into equal ranges for a fixed number of blocks a key/value
// head, since lengths are known on the device only: each block sums the requests' work to find its own range.  Its four
// waves take a request's row tiles side by side, so that keys come from memory once, and the key tiles of a row tile in turn,
// and join their sums in LDS.  What is cut between blocks leaves partial sums, which a second launch joins in the order of
// the keys.  Where tables are short, a block takes a row tile alone, and there is nothing to join.
//
// One token over 260001 keys, 32 heads on 8 of 128 columns, bf16 rows: 97 us, 5.5 TB/s, and 6.7 for the join; 48 tokens
// over 200 to 24000 keys: 80 us, 4.2 TB/s, and 5.7.
#include <algorithm>
#include <cmath>
#include <string>

#include "cache_attention.hpp"

namespace gatgpu {
namespace {

// Waves of a block: of ranges of the work, of a row tile alone, of a join.
constexpr int kWaves = 4, kAloneWaves = 8, kJoinWaves = 4;
constexpr uint32_t kSmallShare = 8;  // work of a worker, up to which none takes parts of two requests

// The queries of a wave's 16 rows as operands.
template <class T, int NB>
struct Queries {
    static constexpr int PARTS = QueryParts<T>::N;
    QueryParts<T> w[NB][2];
};
template <class T, int NB>
__device__ inline Queries<T, NB> load_queries(const CacheAttnArgs& a, const CacheRequest& rq, uint32_t packed, uint32_t head, int g) {
    Queries<T, NB> q;
    const bool there = packed < rq.rows * a.c.group;
    const T* const row = query_row<T>(a, rq, packed, head);
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const uint32_t col = uint32_t(64 * b + 16 * g + 8 * s);
            q.w[b][s] = load_query8(row, col, there && col < a.c.dim);
        }
    return q;
}

// A tile's bytes as they come: keys [operand][64 columns], values [16 columns], and the scales of the lane's 16 keys.
template <int NB>
struct Keys {
    uint4 w[4][NB];
};
template <int NB>
struct Values {
    uint4 w[4 * NB];
    float ks, vs;
    bool page;  // the lane's keys have one
};

// Pages of a tile's keys: of the lane's scores and values, and of the keys whose bytes it loads.
struct TilePages {
    uint32_t own, load;
};
__device__ inline uint32_t own_key(uint32_t tile, int lane) { return tile * kCacheTile + 16u * uint32_t(lane / 16); }
__device__ inline uint32_t loaded_key(uint32_t tile, int lane) { return tile * kCacheTile + 16u * uint32_t(lane % 16 / 4) + uint32_t(lane % 4); }
__device__ inline TilePages tile_pages(const CacheAttnArgs& a, const uint32_t* row, uint32_t keys, uint32_t tile, int lane) {
    const uint32_t own = block_of(a.c, keys, own_key(tile, lane)), load = block_of(a.c, keys, loaded_key(tile, lane) & ~15u);
    return {own == kNoPage ? own : row[own], load == kNoPage ? load : row[load]};
}
template <int NB>
__device__ inline void load_keys(const CacheAttnArgs& a, uint32_t page, uint32_t tile, uint32_t head, int lane, Keys<NB>& t) {
    const uint32_t g = uint32_t(lane / 16);
    const uint8_t* const k = a.k + key_byte(a.c, some_page(a.c, page), head, loaded_key(tile, lane)) + 16 * g;
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i)
#pragma unroll
        for (uint32_t b = 0; b < NB; ++b)
            t.w[i][b] = 64 * b + 16 * g < a.c.dim ? *reinterpret_cast<const uint4*>(k + i * 4 * a.c.dim + 64 * b) : make_uint4(0, 0, 0, 0);
}
template <int NB>
__device__ inline void load_values(const CacheAttnArgs& a, uint32_t page, uint32_t tile, uint32_t head, int lane, Values<NB>& t) {
    t.page = page < a.c.pages;
    const uint32_t own = some_page(a.c, page);
    t.ks = a.k_scale[uint64_t(own) * a.c.kv_heads + head];
    t.vs = a.v_scale[uint64_t(own) * a.c.kv_heads + head];
    const uint8_t* const v = a.v + value_byte(a.c, own, head, own_key(tile, lane), uint32_t(lane % 16));
#pragma unroll
    for (uint32_t d = 0; d < 4 * NB; ++d)
        t.w[d] = 16 * d < a.c.dim ? *reinterpret_cast<const uint4*>(v + (uint64_t(16 * d) << a.c.page_log)) : make_uint4(0, 0, 0, 0);
}

// A wave's running softmax: lane (n, g) has row n's reference, the weights' sum of its own keys, and its columns' sums.
template <int NB>
struct Running {
    f32x4_t o[4 * NB];
    float ref, sum;
    uint64_t far;  // lanes of rows whose reference is; all, where scales are far apart
    int first;     // exponent of the first page's values (the same in all lanes), kNoExponent before
};
constexpr int kNoExponent = 1000;

// Scores of a tile: keys [operand][register] by the lane's row.
struct Scores {
    f32x4_t s[4];
};
template <class T, int NB>
__device__ inline Scores scores(const Queries<T, NB>& q, const Keys<NB>& t) {
    Scores x;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f32x4_t s = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const uint4 lo = keys_operand(t.w[i][b].x, t.w[i][b].y), hi = keys_operand(t.w[i][b].z, t.w[i][b].w);
#pragma unroll
            for (int p = Queries<T, NB>::PARTS - 1; p >= 0; --p) {
                s = mfma_bf16(lo, q.w[b][0].w[p], s);
                s = mfma_bf16(hi, q.w[b][1].w[p], s);
            }
        }
        x.s[i] = s;
    }
    return x;
}
// The weights of a tile's keys as operands: fp16, and what their rounding took (FP32).
struct Weights {
    uint4 w[2], rest[2];
};
// seen: keys that the lane's row sees; whole: every row of the wave sees every key of the tile.
template <class T, int NB>
__device__ inline Weights weigh(const CacheAttnArgs& a, Running<NB>& run, Scores x, const Values<NB>& t, uint32_t tile, uint32_t seen, bool whole, int lane) {
    constexpr int PARTS = QueryParts<T>::N, APART = kCacheSpread<T> / 2;
    const int ev = scale_exponent(t.vs);
    const float by = score_factor(a.scale, t.ks);
    if (run.first == kNoExponent) {
        const uint64_t some = __ballot(t.page);
        if (some) run.first = __builtin_amdgcn_readlane(ev, __builtin_ctzll(some));
    }
    if (__ballot(t.page && uint32_t(ev - run.first + APART) > uint32_t(2 * APART))) run.far = ~uint64_t(0);
    if (!whole) {
        const uint32_t first = own_key(tile, lane), here = t.page && seen > first ? seen - first : 0;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (uint32_t(4 * i + r) >= here) x.s[i][r] = -INFINITY;
    }
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) top = fmaxf(top, x.s[i][r]);
    top = fmaf(top, by, float(ev));
    if (__any(top > run.ref + kCacheRoom)) {
        const float all = xor32_max(xor16_max(top));
        const bool up = all > run.ref + kCacheRoom;
        const float ref = up ? ceilf(all) - kCacheSet : run.ref, less = up ? __builtin_amdgcn_exp2f(run.ref - ref) : 1.0f;
        run.ref = ref;
        run.far |= __ballot(up && fabsf(ref) >= kCacheFar);
        run.sum *= less;
#pragma unroll
        for (int d = 0; d < 4 * NB; ++d) run.o[d] *= less;
    }
    const float shift = float(ev) - run.ref;  // (whole numbers: exact)
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            x.s[i][r] = __builtin_amdgcn_exp2f(fmaf(x.s[i][r], by, shift));
            sum += x.s[i][r];
        }
    run.sum = fmaf(sum, power_of_two(-ev), run.sum);
    Weights w;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        uint32_t u[4], l[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float v0 = x.s[2 * h + j / 2][j % 2 * 2], v1 = x.s[2 * h + j / 2][j % 2 * 2 + 1];
            u[j] = f16x2(v0, v1);
            if constexpr (PARTS > 1) {
                const f16x2_t up = __builtin_bit_cast(f16x2_t, u[j]);
                l[j] = f16x2(v0 - float(up[0]), v1 - float(up[1]));
            }
        }
        w.w[h] = make_uint4(u[0], u[1], u[2], u[3]);
        if constexpr (PARTS > 1) w.rest[h] = make_uint4(l[0], l[1], l[2], l[3]);
    }
    return w;
}
// A tile that some rows do not see whole: values of no token count as 0, and a NaN that some rows see counts as 0 and marks them.
template <int NB>
__device__ inline void clean(Running<NB>& run, Values<NB>& t, uint32_t tile, uint32_t keys, uint32_t seen, int lane) {
    const uint32_t first = own_key(tile, lane);
    const int valid = t.page && keys > first ? int(min(keys - first, 16u)) : 0;
    uint32_t nan = 0;
#pragma unroll
    for (int d = 0; d < 4 * NB; ++d) {
        t.w[d].x &= low_bytes(valid);
        t.w[d].y &= low_bytes(valid - 4);
        t.w[d].z &= low_bytes(valid - 8);
        t.w[d].w &= low_bytes(valid - 12);
        nan |= nan_bytes(t.w[d].x) | nan_bytes(t.w[d].y) | nan_bytes(t.w[d].z) | nan_bytes(t.w[d].w);
    }
    if (!__any(nan != 0)) return;
    const uint32_t here = t.page && seen > first ? seen - first : 0;
    uint32_t u[8];
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j) u[j] = (2 * j < here ? 0x3c00u : 0u) | (2 * j + 1 < here ? 0x3c000000u : 0u);
#pragma unroll
    for (int d = 0; d < 4 * NB; ++d) {
        uint32_t mark[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint32_t& c = (&t.w[d].x)[j];
            const uint32_t n = nan_bytes(c) >> 7;  // 1 at each NaN
            c &= ~(n * 0xffu);
            mark[j] = n * 0x38u;  // 1.0 in e4m3
        }
        f32x4_t count = {0.0f, 0.0f, 0.0f, 0.0f};
        count = mfma_f16(values_operand(mark[0], mark[1]), make_uint4(u[0], u[1], u[2], u[3]), count);
        count = mfma_f16(values_operand(mark[2], mark[3]), make_uint4(u[4], u[5], u[6], u[7]), count);
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (count[r] > 0.0f) run.o[d][r] = NAN;
    }
}
template <int PARTS, int NB>
__device__ inline void add_values(Running<NB>& run, const Weights& w, const Values<NB>& t) {
#pragma unroll
    for (int d = 0; d < 4 * NB; ++d) {
        const uint4 lo = values_operand(t.w[d].x, t.w[d].y), hi = values_operand(t.w[d].z, t.w[d].w);
        if constexpr (PARTS > 1) {
            run.o[d] = mfma_f16(lo, w.rest[0], run.o[d]);
            run.o[d] = mfma_f16(hi, w.rest[1], run.o[d]);
        }
        run.o[d] = mfma_f16(lo, w.w[0], run.o[d]);
        run.o[d] = mfma_f16(hi, w.w[1], run.o[d]);
    }
}

// A wave's share of tiles, every `per`-th from `tile` on, with a reference for each 16 keys (kCacheSpread).
template <class T, int NB>
__device__ inline void far_pass(const CacheAttnArgs& a, const uint32_t* row, const Queries<T, NB>& q, uint32_t keys, uint32_t seen, uint32_t tile, uint32_t stop,
                                      uint32_t per, uint32_t head, int lane, Running<NB>& run) {
#pragma unroll
    for (int d = 0; d < 4 * NB; ++d) run.o[d] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    run.ref = kCacheNoRef;
    run.sum = 0.0f;
    for (; tile < stop; tile += per) {
        const TilePages pages = tile_pages(a, row, keys, tile, lane);
        Keys<NB> k;
        Values<NB> v;
        load_keys<NB>(a, pages.load, tile, head, lane, k);
        load_values<NB>(a, pages.own, tile, head, lane, v);
        Scores x = scores<T, NB>(q, k);
        clean<NB>(run, v, tile, keys, seen, lane);
        const float by = score_factor(a.scale, v.ks);
        const uint32_t first = own_key(tile, lane), here = v.page && seen > first ? seen - first : 0;
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                x.s[i][r] = uint32_t(4 * i + r) < here ? far_score(x.s[i][r], by) : -INFINITY;
                top = fmaxf(top, x.s[i][r]);
            }
        const float own = far_reference(top), ref = fmaxf(run.ref, xor32_max(xor16_max(own)));
        const int less = shift_of(run.ref, ref), up = shift_of(own, ref) - int(kCacheUp), to = up + scale_exponent(v.vs);
        run.ref = ref;
        run.sum = shifted(run.sum, less);
#pragma unroll
        for (int d = 0; d < 4 * NB; ++d) run.o[d] = shifted_all(run.o[d], less);
        float sum = 0.0f;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            uint32_t u[4], l[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float p0 = far_weight(x.s[2 * h + j / 2][j % 2 * 2], own), p1 = far_weight(x.s[2 * h + j / 2][j % 2 * 2 + 1], own);
                sum += p0 + p1;
                u[j] = f16x2(p0, p1);
                const f16x2_t hi = __builtin_bit_cast(f16x2_t, u[j]);
                l[j] = f16x2(p0 - float(hi[0]), p1 - float(hi[1]));
            }
            for (int g = 0; g < 4; ++g) {  // (the lanes' keys of one page at a time)
                const uint32_t keep = lane / 16 == g ? 0xffffffffu : 0u;
                const uint4 w = make_uint4(u[0] & keep, u[1] & keep, u[2] & keep, u[3] & keep), rest = make_uint4(l[0] & keep, l[1] & keep, l[2] & keep, l[3] & keep);
                const int theirs = __shfl(to, 16 * g + lane % 16);
#pragma unroll
                for (int d = 0; d < 4 * NB; ++d) {
                    const uint4 c = h ? values_operand(v.w[d].z, v.w[d].w) : values_operand(v.w[d].x, v.w[d].y);
                    run.o[d] += shifted_all(mfma_f16(c, w, mfma_f16(c, rest, f32x4_t{0.0f, 0.0f, 0.0f, 0.0f})), theirs);
                }
            }
        }
        run.sum += shifted(sum, up);
    }
    run.sum = xor32_add(xor16_add(run.sum));
}

// Row tiles that a block takes side by side, as a power of two (at most 4, the most of a request here), and the work of a
// request.  (64 requests of 4096 keys with 32 packed rows, 32 heads on 8 of 128 columns: 118 us, one row tile after another 189.)
__device__ inline uint32_t together(uint32_t rows) { return rows > 2 ? 2 : rows > 1 ? 1 : 0; }
__device__ inline uint64_t work_of(const CacheAttnArgs& a, const CacheRequest& q) {
    const uint32_t rows = row_tiles(a.c, q);
    return rows ? uint64_t(key_tiles(q)) << together(rows) : 0;
}

// Sums of the waves: [wave][columns / 16][lane] columns, [wave][row] references and weights.
template <int NB, int WAVES>
struct JoinLds {
    f32x4_t o[WAVES][4 * NB][kWave];
    float ref[WAVES][kCacheRows], sum[WAVES][kCacheRows];
};

// Parts of a small call's request.
__device__ inline uint32_t parts_of(uint64_t work, uint64_t share) { return uint32_t(work + share - 1) / uint32_t(share); }
// Inclusive sums over a block's threads; `total`: of all of them.
template <int WAVES>
__device__ inline uint64_t sums_upto(uint64_t x, uint64_t& total) {
    __shared__ uint64_t s_sum[WAVES];
    const int lane = int(threadIdx.x) % kWave, wave = int(threadIdx.x) / kWave;
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) {
        const uint64_t p = __shfl_up(x, d);
        if (lane >= d) x += p;
    }
    __syncthreads();  // (the sums of the call before have been read)
    if (lane == kWave - 1) s_sum[wave] = x;
    __syncthreads();
    total = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        if (w < wave) x += s_sum[w];
        total += s_sum[w];
    }
    return x;
}

// Two waves a SIMD hide their requests behind each other.  (Three, with 168 registers each, keep a part of them in memory:
// 142 us against 96 for one token over 260K, 32 heads of 128 on 8.)
template <class T, int NB, bool ALONE>
__global__ __launch_bounds__((ALONE ? kAloneWaves : kWaves) * kWave, 2) void k_cache_attention(const CacheAttnArgs a) {
    constexpr int PARTS = Queries<T, NB>::PARTS, WAVES = ALONE ? kAloneWaves : kWaves;
    __shared__ JoinLds<NB, WAVES> join;
    __shared__ uint64_t s_start, s_at, s_end;
    __shared__ uint32_t s_request;
    bool apart = false;  // each worker's work is of one request
    const int tid = int(threadIdx.x), lane = tid % kWave, wave = tid / kWave, n = lane % 16, g = lane / 16;
    const uint32_t head = blockIdx.x, worker = blockIdx.y, block = worker * a.c.kv_heads + head;
    uint64_t at = 0, end = 0, base = 0, share = 1;  // the worker's work, and that before its request
    uint32_t request = worker;
    if constexpr (!ALONE) {
        const uint32_t per = (a.c.requests + (WAVES * kWave) - 1) / (WAVES * kWave), from = min(a.c.requests, uint32_t(tid) * per), to = min(a.c.requests, from + per);
        uint64_t own = 0;
        for (uint32_t r = from; r < to; ++r) own += work_of(a, request_of(a, r));
        uint64_t total;
        const uint64_t upto = sums_upto<WAVES>(own, total);
        const uint64_t each = total / a.c.requests;  // (a worker takes one short request, not several in turn)
        share = max(min(max(each, uint64_t(1)), uint64_t(a.least)), (total + a.workers - 1) / a.workers);
        apart = gridDim.y > a.workers && total <= uint64_t(kSmallShare) * a.workers;
        uint64_t mine = own, upto_mine = upto, all = total, place = worker;  // the place among all of what is shared out
        if (apart) {
            mine = 0;
            for (uint32_t r = from; r < to; ++r) mine += parts_of(work_of(a, request_of(a, r)), share);
            upto_mine = sums_upto<WAVES>(mine, all);
        } else {
            place = worker < a.workers ? uint64_t(worker) * share : total;
        }
        if (place < all && place >= upto_mine - mine && place < upto_mine) {  // one thread's requests hold it
            uint64_t sum = upto - own, before = upto_mine - mine;
            for (uint32_t r = from; r < to; ++r) {
                const uint64_t work = work_of(a, request_of(a, r)), places = apart ? parts_of(work, share) : work;
                if (place < before + places) {
                    s_request = r;
                    s_start = sum;
                    s_at = apart ? sum + (place - before) * share : place;
                    s_end = apart ? min(sum + work, s_at + share) : min(total, place + share);
                    break;
                }
                sum += work;
                before += places;
            }
        }
        __syncthreads();
        if (place < all) {
            request = s_request;
            base = s_start;
            at = s_at;
            end = s_end;
        }
        if (at >= end) {
            if (tid == 0) a.meta[block] = make_uint4(0, 0, 0, 0);
            return;
        }
    }
    uint4 meta = make_uint4(0, 0, 0, 0);
    while (request < a.c.requests) {
        const CacheRequest rq = request_of(a, request);
        const uint32_t tiles = key_tiles(rq), rows = row_tiles(a.c, rq);
        if constexpr (ALONE) {
            if (end || blockIdx.z >= rows) return;
            end = tiles;
        }
        if (at >= end) break;
        // Waves side by side take the request's row tiles, those of one row tile its key tiles in turn.
        const uint32_t log = ALONE ? 0 : together(rows), per = uint32_t(WAVES) >> log, member = uniform(uint32_t(wave)) % per, group = uniform(uint32_t(wave)) / per;
        const uint64_t work = ALONE ? tiles : work_of(a, rq), in = at - base, here = min(end - at, work - in);
        if (in >= work) {  // the next request
            base += work;
            ++request;
            continue;
        }
        const uint32_t up = (1u << log) - 1, lo = uint32_t((in + up) >> log), hi = index_min(tiles, (in + here + up) >> log);
        const uint32_t row_tile = ALONE ? blockIdx.z : group;
        const uint32_t packed = row_tile * kCacheRows + uint32_t(n);
        const bool there = packed < rq.rows * a.c.group;
        const uint32_t seen = there ? cache_seen(rq, packed / a.c.group) : 0;
        // Rows of a tile stand in the order of their positions.
        const uint32_t last = min(rq.rows * a.c.group, (row_tile + 1) * kCacheRows) - 1;
        const uint32_t least = cache_seen(rq, row_tile * kCacheRows / a.c.group), most = row_tile < rows ? cache_seen(rq, last / a.c.group) : 0;
        const uint32_t* const row = a.table + uint64_t(request) * a.ld;
        const Queries<T, NB> q = load_queries<T, NB>(a, rq, packed, head, g);
        Running<NB> run;
#pragma unroll
        for (int d = 0; d < 4 * NB; ++d) run.o[d] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
        run.ref = kCacheNoRef;
        run.sum = 0.0f;
        run.far = 0;
        run.first = kNoExponent;
        const uint32_t stop = most ? min(hi, (most - 1) / kCacheTile + 1) : 0;
        uint32_t tile = lo + member;
        if (tile < stop) {
            // A tile's keys are requested when the scores of the one before are formed, its values when those are added.
            TilePages pages = tile_pages(a, row, rq.keys, tile, lane);
            Keys<NB> k;
            Values<NB> v;
            load_keys<NB>(a, pages.load, tile, head, lane, k);
            load_values<NB>(a, pages.own, tile, head, lane, v);
            pages = tile_pages(a, row, rq.keys, tile + per, lane);
            while (true) {
                const Scores x = scores<T, NB>(q, k);
                __builtin_amdgcn_sched_barrier(0);
                const uint32_t next = tile + per;
                if (next < stop) load_keys<NB>(a, pages.load, next, head, lane, k);
                const bool whole = tile < least / kCacheTile && __all(v.page);  // every row sees every key
                const Weights w = weigh<T, NB>(a, run, x, v, tile, seen, whole, lane);
                if (!whole) clean<NB>(run, v, tile, rq.keys, seen, lane);
                add_values<PARTS, NB>(run, w, v);
                __builtin_amdgcn_sched_barrier(0);
                if (next >= stop) break;
                load_values<NB>(a, pages.own, next, head, lane, v);
                pages = tile_pages(a, row, rq.keys, next + per, lane);
                tile = next;
            }
        }
        run.sum = xor32_add(xor16_add(run.sum));
        // The sums of a row tile's waves to one: each of them joins its share of the columns.
        const int shift = weighed(run.ref, run.sum);
        if (lane < 16) {
            join.ref[wave][n] = run.ref;
            join.sum[wave][n] = run.sum;
        }
#pragma unroll
        for (int d = 0; d < 4 * NB; ++d) join.o[wave][d][lane] = shifted_all(run.o[d], shift);
        if (run.far) {
            const bool mine = run.far >> lane & 1;
            far_pass<T, NB>(a, row, q, rq.keys, seen, lo + member, stop, per, head, lane, run);
            if (mine && lane < 16) {
                join.ref[wave][n] = run.ref;
                join.sum[wave][n] = run.sum;
            }
#pragma unroll
            for (int d = 0; d < 4 * NB; ++d)
                if (mine) join.o[wave][d][lane] = run.o[d];
        }
        __syncthreads();
        const uint32_t first = group * per;
        float ref = join.ref[first][n], sum = 0.0f;
        int less[WAVES];
#pragma unroll
        for (uint32_t w = 1; w < uint32_t(WAVES); ++w)
            if (w < per) ref = fmaxf(ref, join.ref[first + w][n]);
#pragma unroll
        for (uint32_t w = 0; w < uint32_t(WAVES); ++w) {
            if (w >= per) break;
            less[w] = shift_of(join.ref[first + w][n], ref);
            sum += shifted(join.sum[first + w][n], less[w]);
        }
        const bool cut = lo > 0 || hi < tiles;
        const uint64_t piece = (uint64_t(block) * 2 + (lo > 0 ? 0 : 1)) * a.row_tiles + row_tile;
        for (uint32_t db = row_tile < rows ? member : 4 * NB; db < 4 * NB; db += per) {
            f32x4_t o = shifted_all(join.o[first][db][lane], less[0]);
#pragma unroll
            for (uint32_t w = 1; w < uint32_t(WAVES); ++w)
                if (w < per) o += shifted_all(join.o[first + w][db][lane], less[w]);
            if (cut) *reinterpret_cast<f32x4_t*>(a.part + ((piece * (4 * NB) + uint64_t(db)) * kWave + uint64_t(lane)) * 4) = o;
            else store4<T>(a, rq, packed, head, uint32_t(16 * db + 4 * g), o, sum);
        }
        if (member == 0 && row_tile < rows && lane < 16) {
            if (cut) {
                a.stat[piece * 32 + uint64_t(n)] = ref;
                a.stat[piece * 32 + 16 + uint64_t(n)] = sum;
            } else {
                store_lse(a, rq, packed, head, ref, sum);
            }
        }
        if (lo == 0 && hi < tiles) meta = make_uint4(request, 0, apart ? parts_of(work, share) : uint32_t((base + work - 1) / share) - worker + 1, 0);
        at += here;
        __syncthreads();
    }
    if (!ALONE && tid == 0) a.meta[block] = meta;
}

// The pieces of the request that begins in a worker and ends in another: 16 columns of a row tile a block, its waves a quarter
// of the pieces each.
template <class T, int NB>
__global__ __launch_bounds__(kJoinWaves * kWave) void k_cache_join(const CacheAttnArgs a) {
    __shared__ f32x4_t s_o[kJoinWaves][kWave];
    __shared__ float s_ref[kJoinWaves][kCacheRows], s_sum[kJoinWaves][kCacheRows];
    const int tid = int(threadIdx.x), lane = tid % kWave, wave = tid / kWave, n = lane % 16, g = lane / 16;
    const uint32_t block = blockIdx.x, db = blockIdx.y, row_tile = blockIdx.z;
    const uint4 meta = a.meta[block];
    if (!meta.z) return;
    const uint32_t head = block % a.c.kv_heads;
    const CacheRequest rq = request_of(a, meta.x);
    if (row_tile >= row_tiles(a.c, rq)) return;
    const auto piece_of = [&](uint32_t p) { return ((uint64_t(block) + uint64_t(p) * uint64_t(a.c.kv_heads)) * 2 + (p ? 0 : 1)) * a.row_tiles + row_tile; };
    f32x4_t o = {0.0f, 0.0f, 0.0f, 0.0f};
    float ref = kCacheNoRef, sum = 0.0f;
#pragma unroll 4
    for (uint32_t p = uint32_t(wave); p < meta.z; p += kJoinWaves) ref = fmaxf(ref, a.stat[piece_of(p) * 32 + uint64_t(n)]);
#pragma unroll 4
    for (uint32_t p = uint32_t(wave); p < meta.z; p += kJoinWaves) {
        const uint64_t piece = piece_of(p);
        const f32x4_t x = *reinterpret_cast<const f32x4_t*>(a.part + ((piece * (4 * NB) + db) * kWave + uint64_t(lane)) * 4);
        const int less = shift_of(a.stat[piece * 32 + uint64_t(n)], ref);
        o += shifted_all(x, less);
        sum += shifted(a.stat[piece * 32 + 16 + uint64_t(n)], less);
    }
    s_o[wave][lane] = o;
    if (lane < 16) {
        s_ref[wave][n] = ref;
        s_sum[wave][n] = sum;
    }
    __syncthreads();
    if (wave) return;
    float top = s_ref[0][n];
#pragma unroll
    for (int w = 1; w < kJoinWaves; ++w) top = fmaxf(top, s_ref[w][n]);
    o = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    sum = 0.0f;
#pragma unroll
    for (int w = 0; w < kJoinWaves; ++w) {
        const int less = shift_of(s_ref[w][n], top);
        o += shifted_all(s_o[w][lane], less);
        sum += shifted(s_sum[w][n], less);
    }
    const uint32_t packed = row_tile * kCacheRows + uint32_t(n);
    store4<T>(a, rq, packed, head, 16 * db + 4 * uint32_t(g), o, sum);
    if (db == 0 && lane < 16) store_lse(a, rq, packed, head, top, sum);
}

// Blocks a key/value head: two a unit in all.
uint32_t cache_workers(const gatgpu_ctx* c, int kv_heads) { return uint32_t(std::max(1, 2 * c->cus / kv_heads)); }

// With those that calls of little work and few requests take besides, where none takes parts of two requests.  Measured with
// one row of 32 heads on 8 of 128 columns, bf16, 64 workers a head, parts of two against that: 4 requests of 300 keys 17.0 and
// 13.0 us, 16 17.4 and 13.8, 64 17.7 and 21.7.
uint32_t workers_most(uint32_t workers, const CacheSizes& c) { return workers + (c.requests <= workers / 4 ? c.requests : 0); }

template <class T, int NB>
hipError_t launch(const CacheAttnArgs& a, hipStream_t s) {
    if (!a.workers) {
        k_cache_attention<T, NB, true><<<dim3(a.c.kv_heads, a.c.requests, a.row_tiles), kAloneWaves * kWave, 0, s>>>(a);
        return hipGetLastError();
    }
    k_cache_attention<T, NB, false><<<dim3(a.c.kv_heads, workers_most(a.workers, a.c)), kWaves * kWave, 0, s>>>(a);
    if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    k_cache_join<T, NB><<<dim3(a.c.kv_heads * workers_most(a.workers, a.c), uint32_t(a.c.dim / 16), a.row_tiles), kJoinWaves * kWave, 0, s>>>(a);
    return hipGetLastError();
}

uint64_t pad256(uint64_t b) { return (b + 255) / 256 * 256; }
struct Workspace {
    uint64_t part, stat, meta;
};
// Row tiles of a request, at most.
uint32_t rows_of(const CacheSizes& s, uint32_t tile) { return uint32_t((std::min<uint64_t>(s.most, s.rows) * s.group + tile - 1) / tile); }
Workspace workspace_of(const gatgpu_ctx* c, const CacheSizes& s) {
    const uint64_t blocks = uint64_t(workers_most(cache_workers(c, int(s.kv_heads)), s)) * s.kv_heads, nb = s.dim > 64 ? 2 : 1;
    const uint64_t pieces = blocks * 2 * rows_of(s, kCacheRows);
    return {pad256(pieces * 4 * nb * kWave * 16), pad256(pieces * 32 * 4), pad256(blocks * 16)};
}
CacheSizes sizes_of(const gatgpu_cache* cache, const gatgpu_cache_attention_io* io) {
    CacheSizes c;
    c.rows = io->rows;
    c.requests = io->requests;
    c.most = io->most;
    c.blocks = io->blocks;
    c.pages = cache->pages;
    while ((1u << c.page_log) < cache->page) ++c.page_log;
    c.heads = uint32_t(io->heads);
    c.kv_heads = uint32_t(cache->kv_heads);
    c.group = uint32_t(io->heads / cache->kv_heads);
    c.dim = uint32_t(cache->dim);
    return c;
}
// Whether requests have more rows than the four tiles of 16 that a block takes side by side.  Measured with 32 heads on 8 of
// 128 columns, those against the tiles of 128 and more: bf16, 32 requests of 4000 keys with 32 packed rows each 67 and 118 us,
// with 64 118 and 128; 64 of 600 keys with 64 45 and 48; FP32, 32 of 4000 with 64 134 and 228, 64 of 600 with 64 54 and 89.
// With 128 rows in tiles of 16, which would read the keys twice: bf16 204 and 130, FP32 250 and 236.
bool in_chunks(const CacheSizes& c) { return uint64_t(c.most) * c.group > 4 * kCacheRows; }
// A block a row tile, nothing to join, where no request has more than 16 tiles of keys (many rows: 8) and the blocks are few.
// Measured with 32 heads on 8 of 128 columns, bf16, ranges of the work against that.  One row each: 16 requests of 300 keys
// 13.8 and 7.4 us, of 1024 19 and 12; one of 2048 13 and 16; 64 of 1024 29 and 27.  8 rows, two tiles: 64 of 300 22 and 32.
// 50 rows: 4 of 300 30 and 20, of 1024 30 and 43; 35 of 512 60 and 55, of 1024 80 and 90.
bool block_a_tile(const gatgpu_ctx* ctx, const CacheSizes& c, uint32_t row_tiles, bool chunks) {
    const uint64_t tiles = chunks ? 8 : 16, blocks = uint64_t(ctx->cus) * (chunks ? 4 : 2);
    return uint64_t(c.blocks) << c.page_log <= tiles * kCacheTile && uint64_t(c.requests) * row_tiles * c.kv_heads <= blocks;
}
uint64_t workspace_bytes(const gatgpu_ctx* c, const CacheSizes& s, bool bf16) {
    const Workspace w = workspace_of(c, s);
    return in_chunks(s) ? chunk_plan(c->cus, s, bf16).bytes : w.part + w.stat + w.meta;
}

}  // namespace
}  // namespace gatgpu

namespace {

using namespace gatgpu;

int check_sizes(gatgpu_ctx* c, const gatgpu_cache* cache, const gatgpu_cache_attention_io* io) {
    if (!io) return fail(c, GATGPU_EINVAL, "null arrays");
    if (io->precision != GATGPU_FP32 && io->precision != GATGPU_BF16) return fail(c, GATGPU_EINVAL, "bad precision");
    if (io->heads < 1 || io->heads > 64 || io->heads % cache->kv_heads) return fail(c, GATGPU_EINVAL, "heads must be 1 to 64 and a multiple of kv_heads");
    if (io->rows >= (uint64_t(1) << 31) / uint64_t(io->heads)) return fail(c, GATGPU_EOVERFLOW, "rows * heads must be below 2^31");
    if (io->requests > (1u << 20)) return fail(c, GATGPU_EOVERFLOW, "more than 2^20 requests");
    if (uint64_t(io->blocks) * cache->page >= (uint64_t(1) << 32)) return fail(c, GATGPU_EOVERFLOW, "blocks * page must be below 2^32");
    if (io->table_stride < io->blocks || io->table_stride > (uint64_t(1) << 40)) return fail(c, GATGPU_EINVAL, "table has a bad row stride");
    return GATGPU_OK;
}
int check_rows(gatgpu_ctx* c, const gatgpu_cache* cache, const gatgpu_cache_attention_io* io, const char* name, const void* p, uint64_t stride) {
    if (!p) return fail(c, GATGPU_EINVAL, std::string("null ") + name);
    const uint64_t size = io->precision == GATGPU_BF16 ? 2 : 4;
    if (stride < uint64_t(io->heads) * uint64_t(cache->dim) || stride > (uint64_t(1) << 44))
        return fail(c, GATGPU_EINVAL, std::string(name) + " has a bad row stride");
    if (reinterpret_cast<uintptr_t>(p) % 16 || stride * size % 16) return fail(c, GATGPU_EINVAL, std::string(name) + " and its stride must be 16-byte aligned");
    return check_device_array(c, p, name);
}
int check_words(gatgpu_ctx* c, const char* name, const void* p) {
    if (!p) return fail(c, GATGPU_EINVAL, std::string("null ") + name);
    if (reinterpret_cast<uintptr_t>(p) % 4) return fail(c, GATGPU_EINVAL, std::string(name) + " must be 4-byte aligned");
    return check_device_array(c, p, name);
}

}  // namespace

extern "C" {

int gatgpu_cache_attention_workspace(gatgpu_ctx* c, const gatgpu_cache* cache, const gatgpu_cache_attention_io* io, uint64_t* bytes) {
    if (!c) return fail(nullptr, GATGPU_EINVAL, "null context");
    if (!bytes) return fail(c, GATGPU_EINVAL, "null output");
    if (int r = check_cache(c, cache, false)) return r;
    if (int r = check_sizes(c, cache, io)) return r;
    *bytes = workspace_bytes(c, sizes_of(cache, io), io->precision == GATGPU_BF16);
    return GATGPU_OK;
}

int gatgpu_cache_attention(gatgpu_ctx* c, const gatgpu_cache* cache, const gatgpu_cache_attention_io* io, void* ws, uint64_t bytes) {
    if (!c) return fail(nullptr, GATGPU_EINVAL, "null context");
    DeviceGuard on(c->device);
    if (!on.ok) return fail(c, GATGPU_EDEVICE, "cannot select the context's device");
    if (int r = check_cache(c, cache, true)) return r;
    if (int r = check_sizes(c, cache, io)) return r;
    if (!(io->scale > 0.0f) || !std::isfinite(io->scale)) return fail(c, GATGPU_EINVAL, "scale must be positive and finite");
    if (!io->rows || !io->requests || !io->most) return GATGPU_OK;
    if (int r = check_rows(c, cache, io, "q", io->q, io->q_stride)) return r;
    if (int r = check_rows(c, cache, io, "out", io->out, io->out_stride)) return r;
    if (int r = check_words(c, "q_begin", io->q_begin)) return r;
    if (int r = check_words(c, "k_len", io->k_len)) return r;
    if (io->blocks)
        if (int r = check_words(c, "table", io->table)) return r;
    if (io->lse)
        if (int r = check_words(c, "lse", io->lse)) return r;
    CacheAttnArgs a;
    a.c = sizes_of(cache, io);
    const uint64_t need = workspace_bytes(c, a.c, io->precision == GATGPU_BF16);
    if (bytes < need) return fail(c, GATGPU_EINVAL, "workspace of " + std::to_string(bytes) + " bytes, " + std::to_string(need) + " needed");
    if (!ws || reinterpret_cast<uintptr_t>(ws) % 16) return fail(c, GATGPU_EINVAL, "workspace must be 16-byte aligned device memory");
    if (int r = check_device_array(c, ws, "workspace")) return r;
    a.scale = io->scale * 1.44269504088896341f;
    a.ld = io->table_stride;
    a.qs = io->q_stride;
    a.os = io->out_stride;
    a.q = io->q;
    a.out = io->out;
    a.lse = io->lse;
    a.q_begin = io->q_begin;
    a.k_len = io->k_len;
    a.table = io->table;
    a.k = cache->k;
    a.v = cache->v;
    a.k_scale = cache->k_scale;
    a.v_scale = cache->v_scale;
    const bool bf16 = io->precision == GATGPU_BF16, wide = cache->dim > 64, chunks = in_chunks(a.c);
    a.row_tiles = rows_of(a.c, chunks ? chunk_rows(a.c, bf16) : kCacheRows);
    const bool alone = block_a_tile(c, a.c, a.row_tiles, chunks);
    if (chunks) {
        const ChunkPlan plan = chunk_plan(c->cus, a.c, bf16);
        a.workers = alone ? 0 : plan.workers;
        a.least = 4;  // (2 and 8 instead: 16 requests of 50 rows over 1024 keys, 8 heads on 2, 44 and 37 us, 36 with 4; one 22 and 33, 25 with 4)
        HIPCHECK(c, launch_cache_chunk(a, bf16, plan, ws, c->stream));
        return GATGPU_OK;
    }
    a.workers = alone ? 0 : cache_workers(c, cache->kv_heads);
    a.least = 4;  // (a tile a wave; 2 and 8 instead: one row over 4096 keys 13.8 and 14.5 us, 13.1 with 4)
    const Workspace w = workspace_of(c, a.c);
    a.part = static_cast<float*>(ws);
    a.stat = reinterpret_cast<float*>(static_cast<char*>(ws) + w.part);
    a.meta = reinterpret_cast<uint4*>(static_cast<char*>(ws) + w.part + w.stat);
    HIPCHECK(c, bf16 ? (wide ? launch<uint16_t, 2>(a, c->stream) : launch<uint16_t, 1>(a, c->stream))
                     : (wide ? launch<float, 2>(a, c->stream) : launch<float, 1>(a, c->stream)));
    return GATGPU_OK;
}

}  // extern "C"
