// Attention over a paged 8-bit cache, many rows a request: chunks of prompts.
//
// Bound by matrix and vector instructions (4 products of 64 x 32 x dim a step and wave, an exponential a pair).  A block of
// four or eight waves takes 128 or 256 packed rows, 32 a wave, on v_mfma_f32_32x32x16.  Its threads request a tile of 64 keys
// two steps ahead, turn its bytes to bf16 keys and fp16 values once for all waves, and leave them in one of two LDS buffers
// while the other is worked on; one barrier a step.
//   S^T = K Q^T: lane (n = lane % 32, h = lane / 32) gets row n's scores of LDS rows 8 i + 4 h + r (register 4 i + r), and LDS
//   row m of 32 holds key 16 (m / 16) + 8 (m / 4 % 2) + 4 (m / 8 % 2) + m % 4, so that registers 8 s ... 8 s + 7 are keys
//   16 s + 8 h ... + 7: the second product's operand as they stand.
//
// Work is cut into equal ranges of (row tile, key tile) for as many blocks as run at once, since lengths are known on the
// device only: a first launch of one block forms the sums over the tiles, and a last one joins the tiles that a range's end
// cuts.  Where tables are short, a block takes a row tile alone, in one launch.
//
// 6 requests of 324 to 1649 rows over up to 10392 keys, 16 heads on 4 of 128 columns, bf16: 252 to 260 us, 656 to
// 676 TFLOP/s, the whole call; under a profiler the kernel alone 261 to 275 (vector instructions 47 % of the cycles, matrix pipes
// 35 %, one behind the other in a wave), sums 5.2, join 18.
#include <algorithm>
#include <type_traits>

#include "cache_attention.hpp"

namespace gatgpu {
namespace {

constexpr int kScan = 1024;
constexpr uint32_t kWaveRows = 32;  // packed rows of a wave
typedef float f32x16_t __attribute__((ext_vector_type(16)));

struct ChunkArgs {
    CacheAttnArgs a;
    uint32_t tiles = 0;          // at most
    uint32_t tile_rows = 0;      // packed rows of a block
    uint32_t* begin = nullptr;   // [requests + 1] first row tile of each request
    uint32_t* request = nullptr; // [tiles]
    uint64_t* upto = nullptr;    // [tiles + 1] key tiles of the row tiles before each
};

__device__ inline uint32_t chunk_tiles(const ChunkArgs& p, const CacheRequest& q) { return (q.rows * p.a.c.group + p.tile_rows - 1) / p.tile_rows; }
// Key tiles that the rows of row tile t see (one, if none).
__device__ inline uint32_t tiles_seen(const ChunkArgs& p, const CacheRequest& q, uint32_t t) {
    const uint32_t last = min(q.rows * p.a.c.group, (t + 1) * p.tile_rows) - 1, n = cache_seen(q, last / p.a.c.group);
    return n ? (n - 1) / kCacheTile + 1 : 1;
}
__device__ inline uint64_t scan_sums(uint64_t x, uint64_t& total) {
    __shared__ uint64_t wave_total[kScan / kWave];
    const int lane = int(threadIdx.x) % kWave, wave = int(threadIdx.x) / kWave;
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) {
        const uint64_t p = __shfl_up(x, d);
        if (lane >= d) x += p;
    }
    __syncthreads();
    if (lane == kWave - 1) wave_total[wave] = x;
    __syncthreads();
    total = 0;
    for (int w = 0; w < kScan / kWave; ++w) {
        if (w < wave) x += wave_total[w];
        total += wave_total[w];
    }
    return x;
}
__global__ __launch_bounds__(kScan) void k_cache_plan(const ChunkArgs p) {
    const CacheAttnArgs& a = p.a;
    const uint32_t tid = threadIdx.x;
    uint64_t total, before = 0;
    for (uint32_t first = 0; first < a.c.requests; first += kScan) {
        const uint32_t r = first + tid;
        const uint64_t n = r < a.c.requests ? chunk_tiles(p, request_of(a, r)) : 0, sum = scan_sums(n, total);
        if (r < a.c.requests) p.begin[r] = index_min(before + sum - n, p.tiles);
        before += total;
    }
    const uint32_t tiles = index_min(before, p.tiles);  // (never more, for rows in order)
    if (tid == 0) {
        p.begin[a.c.requests] = tiles;
        p.upto[0] = 0;
    }
    __syncthreads();
    before = 0;
    for (uint32_t first = 0; first < tiles; first += kScan) {
        const uint32_t t = first + tid;
        uint64_t n = 0;
        if (t < tiles) {
            uint32_t lo = 0, hi = a.c.requests - 1;  // the last request that begins at or before t
            while (lo < hi) {
                const uint32_t mid = (lo + hi + 1) / 2;
                if (p.begin[mid] <= t) lo = mid;
                else hi = mid - 1;
            }
            p.request[t] = lo;
            const CacheRequest q = request_of(a, lo);
            const uint32_t own = t - p.begin[lo];
            n = own < chunk_tiles(p, q) ? tiles_seen(p, q, own) : 0;
        }
        const uint64_t sum = scan_sums(n, total);
        if (t < tiles) p.upto[t + 1] = before + sum;
        before += total;
    }
}

// A block's tiles of keys and values: [buffer][row][64 columns of NB], [buffer][column][64 keys]; pieces of 16 bytes.
template <int NB>
struct ChunkLds {
    uint4 k[2][kCacheTile][8 * NB];
    uint4 v[2][64 * NB][8];
    float scale[2][4][2];  // of each 16 keys: what a score is multiplied by, and the values' exponent; without a page: -1
    uint16_t bad[2][64 * NB][4];  // which of each 16 keys' values are NaN (they stand as 0 in v)
    uint32_t nan[4];       // the values of tile i (of a piece), in place i % 4, hold one
    uint32_t far;          // some row is formed again
};

// What a thread requests of a tile, in 16 bytes: of N keys each 16 columns, and of N columns each 16 keys.
template <int N>
struct Bytes {
    uint4 k[N], v[N];
    float ks;      // what the 16 keys' scores are multiplied by, and their values' exponent (of the first threads)
    int vs;
    int tokens;    // among the 16 keys of the values
};
// What a row crosses its pieces' indices with, of PIECES of them a row: 16 neighbouring lanes then meet the 16 pieces of 256
// bytes, all banks of a cycle, both as they write (pieces of a row or of a few) and as they read (a piece of 16 rows).
template <int PIECES>
__device__ inline uint32_t turned(uint32_t row) {
    return PIECES == 16 ? row % 16 : row / 2 % 8;
}
template <int N>
struct Pages {
    uint32_t k[N], v;
};
__device__ inline f32x16_t mfma32_bf16(uint4 a, uint4 b, f32x16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}
__device__ inline f32x16_t mfma32_f16(uint4 a, uint4 b, f32x16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
}
// What a block works on at a time: key tiles lo to hi of a row tile.
struct Piece {
    uint32_t head, request, row_tile, lo, hi;
    bool cut;        // there are others of the row tile
    uint64_t place;  // where the first wave's sums go then
};
// One piece: the rows' sums over its tiles, to the output, or where others are to be joined to them.  `far` becomes the lanes of rows
// that are to be formed again; FAR: of those, with a reference for each 16 keys (kCacheSpread), else of all others.
template <class T, int NB, int WAVES, bool FAR>
__device__ inline __attribute__((always_inline)) void chunk_piece(const ChunkArgs& p, ChunkLds<NB>& lds, const CacheRequest& rq, const Piece& w, uint64_t& far) {
    constexpr int PARTS = QueryParts<T>::N, PIECES = 4 * NB;  // 16-byte pieces of a key's bytes
    constexpr int THREADS = WAVES * kWave, N = NB * 256 > THREADS ? NB * 256 / THREADS : 1;  // pieces of keys (of values) a thread
    constexpr uint32_t ROWS = WAVES * kWaveRows, KEYS = THREADS / PIECES, COLS = THREADS / 4;  // keys and columns of a pass
    const CacheAttnArgs& a = p.a;
    const int tid = int(threadIdx.x), lane = tid % kWave, wave = tid / kWave, n = lane % 32, h = lane / 32;
    const uint32_t head = w.head, lo = w.lo, hi = w.hi;
    // What this thread brings of a tile: keys k_key + 32 i, columns 16 k_piece; columns v_col + 64 i, keys 16 v_group.
    const uint32_t k_key = uint32_t(tid) / PIECES, k_piece = uint32_t(tid) % PIECES, v_group = uint32_t(tid) % 4, v_col = uint32_t(tid) / 4;
    const bool brings = THREADS <= NB * 256 || tid < NB * 256;
    const uint32_t packed = w.row_tile * ROWS + uint32_t(wave) * kWaveRows + uint32_t(n), rows = rq.rows * a.c.group;
    const uint32_t seen = packed < rows ? cache_seen(rq, packed / a.c.group) : 0;
    // Rows of a wave stand in the order of their positions; a wave without rows sees nothing.
    const uint32_t first_row = w.row_tile * ROWS + uniform(uint32_t(wave)) * kWaveRows;
    const uint32_t least = first_row < rows ? cache_seen(rq, first_row / a.c.group) : 0;
    const uint32_t most = first_row < rows ? cache_seen(rq, (min(rows, first_row + kWaveRows) - 1) / a.c.group) : 0;
    const uint32_t* const table = a.table + uint64_t(w.request) * a.ld;

    // Where this thread's bytes lie in a page, but for the tile's place in it (pages of 64 tokens and more).
    const uint32_t in_page = (1u << a.c.page_log) - 1, all_seen = cache_seen(rq, w.row_tile * ROWS / a.c.group);  // by every row
    const uint64_t page_bytes = (uint64_t(a.c.kv_heads) << a.c.page_log) * a.c.dim;
    uint32_t k_at[N], v_at[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        k_at[i] = uint32_t(key_byte(a.c, 0, head, k_key + uint32_t(i) * KEYS)) + 16 * k_piece;
        v_at[i] = uint32_t(value_byte(a.c, 0, head, 16 * v_group, v_col + COLS * uint32_t(i)));
    }
    int low = kMostScale, high = kLeastScale;  // of the exponents of the values' scales
    const auto load_pages = [&](uint32_t tile) {
        Pages<N> g;
        const uint32_t first = tile * kCacheTile;
        const auto page_of = [&](uint32_t key) {
            const uint32_t block = block_of(a.c, rq.keys, key);
            return block == kNoPage ? block : table[block];
        };
#pragma unroll
        for (int i = 0; i < N; ++i) g.k[i] = page_of(first + (k_key + uint32_t(i) * KEYS) / 16 * 16);
        g.v = page_of(first + 16 * v_group);
        return g;
    };
    const auto load_bytes = [&](uint32_t tile, const Pages<N>& g) {
        Bytes<N> x;
        if (tid < 4) {
            const uint64_t place = uint64_t(some_page(a.c, g.v)) * a.c.kv_heads + head;
            x.ks = g.v < a.c.pages ? score_factor(a.scale, a.k_scale[place]) : -1.0f;
            x.vs = scale_exponent(a.v_scale[place]);
        }
        const uint32_t place = tile * kCacheTile & in_page;
        const uint8_t* const v = a.v + place + some_page(a.c, g.v) * page_bytes;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint8_t* const k = a.k + place * a.c.dim + some_page(a.c, g.k[i]) * page_bytes;
            x.k[i] = brings && 16 * k_piece < a.c.dim ? *reinterpret_cast<const uint4*>(k + k_at[i]) : make_uint4(0, 0, 0, 0);
            x.v[i] = brings && v_col + COLS * uint32_t(i) < a.c.dim ? *reinterpret_cast<const uint4*>(v + v_at[i]) : make_uint4(0, 0, 0, 0);
        }
        x.tokens = g.v < a.c.pages ? int(min(rq.keys - (tile * kCacheTile + 16 * v_group), 16u)) : 0;
        return x;
    };
    const auto put = [&](uint32_t tile, Bytes<N>& x) {
        if (!brings) return;
        const uint32_t buffer = (tile - lo) % 2;
        if (tid < 4) {
            lds.scale[buffer][tid][0] = x.ks;
            lds.scale[buffer][tid][1] = __int_as_float(x.vs);
        }
        if (x.tokens < 16) {  // values of no token count as 0
#pragma unroll
            for (int i = 0; i < N; ++i) {
                x.v[i].x &= low_bytes(x.tokens);
                x.v[i].y &= low_bytes(x.tokens - 4);
                x.v[i].z &= low_bytes(x.tokens - 8);
                x.v[i].w &= low_bytes(x.tokens - 12);
            }
        }
        if (tile >= all_seen / kCacheTile) {  // some rows do not see all of it: its NaNs stand as 0, and are marked
#pragma unroll
            for (int i = 0; i < N; ++i) {
                uint4& v = x.v[i];
                const uint32_t w[4] = {nan_bytes(v.x) >> 7, nan_bytes(v.y) >> 7, nan_bytes(v.z) >> 7, nan_bytes(v.w) >> 7};  // 1 in each byte
                uint32_t bits = 0;
#pragma unroll
                for (int k = 0; k < 4; ++k) bits |= ((w[k] | w[k] >> 7 | w[k] >> 14 | w[k] >> 21) & 15u) << (4 * k);
                v = make_uint4(v.x & ~(w[0] * 0xffu), v.y & ~(w[1] * 0xffu), v.z & ~(w[2] * 0xffu), v.w & ~(w[3] * 0xffu));
                lds.bad[buffer][v_col + COLS * uint32_t(i)][v_group] = uint16_t(bits);
                if (bits) lds.nan[(tile - lo) % 4] = 1;  // (every writer writes the same)
            }
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint32_t key = k_key + uint32_t(i) * KEYS;
            const uint32_t m = key / 32 * 32 + key / 16 % 2 * 16 + key / 4 % 2 * 8 + key / 8 % 2 * 4 + key % 4;
            lds.k[buffer][m][(2 * k_piece) ^ turned<8 * NB>(m)] = keys_operand(x.k[i].x, x.k[i].y);
            lds.k[buffer][m][(2 * k_piece + 1) ^ turned<8 * NB>(m)] = keys_operand(x.k[i].z, x.k[i].w);
            const uint32_t col = v_col + COLS * uint32_t(i);
            lds.v[buffer][col][(2 * v_group) ^ turned<8>(col)] = values_operand(x.v[i].x, x.v[i].y);
            lds.v[buffer][col][(2 * v_group + 1) ^ turned<8>(col)] = values_operand(x.v[i].z, x.v[i].w);
        }
    };

    QueryParts<T> q[4 * NB];
    f32x16_t o[2 * NB];
    float ref = kCacheNoRef, sum = 0.0f;
    Pages<N> pages = load_pages(lo);
    Bytes<N> bytes = load_bytes(lo, pages);
    pages = load_pages(lo + 1);
    const T* const row = query_row<T>(a, rq, packed, head);
#pragma unroll
    for (int s = 0; s < 4 * NB; ++s) {
        const uint32_t col = uint32_t(16 * s + 8 * h);
        q[s] = load_query8(row, col, packed < rows && col < a.c.dim);
    }
#pragma unroll
    for (int d = 0; d < 2 * NB; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[d][r] = 0.0f;
    if (tid < 4) lds.nan[tid] = 0;
    __syncthreads();
    put(lo, bytes);
    if (lo + 1 < hi) {
        bytes = load_bytes(lo + 1, pages);
        pages = load_pages(lo + 2);
    }
    __syncthreads();
    for (uint32_t tile = lo; tile < hi; ++tile) {
        const uint32_t buffer = (tile - lo) % 2;
        if (tid == 0) lds.nan[(tile - lo + 2) % 4] = 0;  // (read two barriers ago, set again behind the next one)
        if (tile + 1 < hi) {
            put(tile + 1, bytes);
            if (tile + 2 < hi) {
                bytes = load_bytes(tile + 2, pages);
                pages = load_pages(tile + 3);
            }
        }
        if (tile * kCacheTile < most) {
            // Of the tile's four 16 keys: scales, and whether they have a page.  The same in all lanes.
            float by[4];
            int ev[4];
            uint32_t held = 0;
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const uint32_t factor = uniform(__float_as_uint(lds.scale[buffer][g][0]));
                by[g] = __uint_as_float(factor & 0x7fffffffu);
                ev[g] = int(uniform(__float_as_uint(lds.scale[buffer][g][1])));
                if (!(factor >> 31)) {
                    held |= 1u << g;
                    low = min(low, ev[g]);
                    high = max(high, ev[g]);
                }
            }
            f32x16_t s[2];
#pragma unroll
            for (int r = 0; r < 16; ++r) s[0][r] = s[1][r] = 0.0f;
            // Two chains of products; their keys are read a step ahead.
            uint4 keys[2][2];
            const auto read_keys = [&](int c) {
#pragma unroll
                for (int k = 0; k < 2; ++k) keys[c % 2][k] = lds.k[buffer][32 * k + n][uint32_t(2 * c + h) ^ turned<8 * NB>(uint32_t(n))];
            };
            read_keys(0);
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int c = 0; c < 4 * NB; ++c) {
                if (c + 1 < 4 * NB) read_keys(c + 1);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int part = PARTS - 1; part >= 0; --part)
#pragma unroll
                    for (int k = 0; k < 2; ++k) s[k] = mfma32_bf16(keys[c % 2][k], q[c].w[part], s[k]);
            }
            __builtin_amdgcn_s_setprio(0);
            uint4 values[2][2 * NB];  // of 16 keys, for the second product: the first ones are there when their weights are
            const auto read_values = [&](int g) {
#pragma unroll
                for (int d = 0; d < 2 * NB; ++d) values[g % 2][d] = lds.v[buffer][32 * d + n][uint32_t(2 * g + h) ^ turned<8>(uint32_t(n))];
            };
            if (!FAR) read_values(0);
            __builtin_amdgcn_sched_barrier(0);
            const bool whole = tile < least / kCacheTile && held == 15;
            if (!whole) {
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const int g = 2 * k + r / 8;
                        if (!(held >> g & 1) || tile * kCacheTile + uint32_t(16 * g + 8 * h + r % 8) >= seen) s[k][r] = -INFINITY;
                    }
            }
            int far_up[4];  // FAR: by what the sums of each 16 keys' weights are shifted
            float far_ref[4];
            if constexpr (FAR) {
                float to = ref;
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    float top = -INFINITY;
#pragma unroll
                    for (int r = 0; r < 8; ++r) {
                        const float x = far_score(s[g / 2][8 * (g % 2) + r], by[g]);
                        s[g / 2][8 * (g % 2) + r] = x;
                        top = fmaxf(top, x);
                    }
                    far_ref[g] = far_reference(xor32_max(top));
                    to = fmaxf(to, far_ref[g]);
                }
                const int less = shift_of(ref, to);
                ref = to;
                sum = shifted(sum, less);
#pragma unroll
                for (int d = 0; d < 2 * NB; ++d) o[d] = shifted_all(o[d], less);
#pragma unroll
                for (int g = 0; g < 4; ++g) far_up[g] = shift_of(far_ref[g], ref) - int(kCacheUp);
            } else {
                float top = -INFINITY;
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    float t = s[g / 2][8 * (g % 2)];
#pragma unroll
                    for (int r = 1; r < 8; ++r) t = fmaxf(t, s[g / 2][8 * (g % 2) + r]);
                    top = fmaxf(top, fmaf(t, by[g], float(ev[g])));
                }
                if (__any(top > ref + kCacheRoom)) {
                    const float both = xor32_max(top);
                    const bool up = both > ref + kCacheRoom;
                    const float to = up ? ceilf(both) - kCacheSet : ref, less = up ? __builtin_amdgcn_exp2f(ref - to) : 1.0f;
                    ref = to;
                    far |= __ballot(up && fabsf(to) >= kCacheFar);
                    sum *= less;
#pragma unroll
                    for (int d = 0; d < 2 * NB; ++d)
#pragma unroll
                        for (int r = 0; r < 16; ++r) o[d][r] *= less;
                }
            }
            uint4 w[4], rest[4];
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const float shift = float(ev[g]) - ref;  // (whole numbers: exact)
                float x[8], of = 0.0f;
#pragma unroll
                for (int r = 0; r < 8; ++r) {
                    if constexpr (FAR) x[r] = far_weight(s[g / 2][8 * (g % 2) + r], far_ref[g]);
                    else x[r] = __builtin_amdgcn_exp2f(fmaf(s[g / 2][8 * (g % 2) + r], by[g], shift));
                    of += x[r];
                }
                uint32_t u[4], l[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    u[j] = f16x2(x[2 * j], x[2 * j + 1]);
                    if constexpr (PARTS > 1) {
                        const f16x2_t up = __builtin_bit_cast(f16x2_t, u[j]);
                        l[j] = f16x2(x[2 * j] - float(up[0]), x[2 * j + 1] - float(up[1]));
                    }
                }
                sum = FAR ? sum + shifted(of, far_up[g]) : fmaf(of, power_of_two(-ev[g]), sum);
                w[g] = make_uint4(u[0], u[1], u[2], u[3]);
                if constexpr (PARTS > 1) rest[g] = make_uint4(l[0], l[1], l[2], l[3]);
            }
            if (tile >= all_seen / kCacheTile && lds.nan[(tile - lo) % 4]) {  // NaNs mark the rows that see them
#pragma unroll
                for (int d = 0; d < 2 * NB; ++d)
#pragma unroll 1
                    for (int g = 0; g < 4; ++g) {
                        const uint32_t bits = uint32_t(lds.bad[buffer][32 * d + n][g]) >> (8 * h);
                        uint32_t x[4], u[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const uint32_t key = tile * kCacheTile + uint32_t(16 * g + 8 * h + 2 * j);
                            x[j] = (bits >> (2 * j) & 1u ? 0x3c00u : 0u) | (bits >> (2 * j + 1) & 1u ? 0x3c000000u : 0u);
                            u[j] = (key < seen ? 0x3c00u : 0u) | (key + 1 < seen ? 0x3c000000u : 0u);
                        }
                        f32x16_t count;
#pragma unroll
                        for (int r = 0; r < 16; ++r) count[r] = 0.0f;
                        count = mfma32_f16(make_uint4(x[0], x[1], x[2], x[3]), make_uint4(u[0], u[1], u[2], u[3]), count);
#pragma unroll
                        for (int r = 0; r < 16; ++r)
                            if (count[r] > 0.0f) o[d][r] = NAN;
                    }
            }
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                if (FAR) read_values(g);
                else if (g + 1 < 4) read_values(g + 1);
                __builtin_amdgcn_sched_barrier(0);
                if constexpr (FAR) {
#pragma unroll
                    for (int d = 0; d < 2 * NB; ++d) {
                        f32x16_t t;
#pragma unroll
                        for (int r = 0; r < 16; ++r) t[r] = 0.0f;
                        if constexpr (PARTS > 1) t = mfma32_f16(values[g % 2][d], rest[g], t);
                        o[d] += shifted_all(mfma32_f16(values[g % 2][d], w[g], t), far_up[g] + ev[g]);
                    }
                    continue;
                }
#pragma unroll
                for (int part = 0; part < (PARTS > 1 ? 2 : 1); ++part)
#pragma unroll
                    for (int d = 0; d < 2 * NB; ++d) o[d] = mfma32_f16(values[g % 2][d], PARTS > 1 && part == 0 ? rest[g] : w[g], o[d]);
            }
            __builtin_amdgcn_s_setprio(0);
        }
        __syncthreads();
    }
    sum = xor32_add(sum);
    if (!FAR && high - low > kCacheSpread<T>) far = ~uint64_t(0);
    // A lane's row; both halves of a row are of one mind.
    if ((far >> lane & 1) != uint64_t(FAR)) return;
    const int shift = w.cut ? weighed(ref, sum) : 0;
    const uint64_t piece = w.place + uint64_t(wave);
#pragma unroll
    for (int d = 0; d < 2 * NB; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const f32x4_t x = {o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]};
            if (w.cut) *reinterpret_cast<f32x4_t*>(a.part + ((piece * (8 * NB) + uint64_t(4 * d + i)) * kWave + uint64_t(lane)) * 4) = shifted_all(x, shift);
            else store4<T>(a, rq, packed, head, uint32_t(32 * d + 8 * i + 4 * h), x, sum);
        }
    if (lane < 32) {
        if (w.cut) {
            a.stat[piece * 64 + uint64_t(n)] = ref;
            a.stat[piece * 64 + 32 + uint64_t(n)] = sum;
        } else {
            store_lse(a, rq, packed, head, ref, sum);
        }
    }
}
// ALONE: a block a row tile; else each worker's range of the work.
template <class T, int NB, int WAVES, bool ALONE>
__global__ __launch_bounds__(WAVES * kWave, sizeof(T) == 2 ? 2 : 1) void k_cache_chunk(const ChunkArgs p) {
    __shared__ ChunkLds<NB> lds;
    const CacheAttnArgs& a = p.a;
    const int tid = int(threadIdx.x), lane = tid % kWave;
    const uint32_t head = blockIdx.x, worker = blockIdx.y, block = worker * a.c.kv_heads + head;
    const auto upto = read_only(p.upto);
    uint64_t at = 0, end = 1, share = 1;
    uint32_t tile_at = worker;
    if constexpr (!ALONE) {
        const uint32_t tiles = read_only(p.begin)[a.c.requests];
        const uint64_t total = tiles ? upto[tiles] : 0;
        const uint64_t each = tiles ? total / tiles : 0;  // (a worker takes one short tile, not several in turn)
        share = max(min(max(each, uint64_t(1)), uint64_t(a.least)), (total + a.workers - 1) / a.workers);
        at = min(total, uint64_t(worker) * share);
        end = min(total, at + share);
        if (at < end) tile_at = uniform(last_at_most(p.upto, tiles, at, lane));
    }
    uint4 meta = make_uint4(0, 0, 0, 0);
    for (; at < end; ++tile_at) {
        uint64_t base = 0, next_base;
        uint32_t request = worker, row_tile = blockIdx.z;
        if constexpr (!ALONE) {
            base = upto[tile_at];
            next_base = upto[tile_at + 1];
            if (at >= next_base) continue;  // (a tile of no work)
            request = read_only(p.request)[tile_at];
            row_tile = tile_at - read_only(p.begin)[request];
        }
        const CacheRequest rq = request_of(a, request);
        if constexpr (ALONE) {
            if (row_tile >= chunk_tiles(p, rq)) return;
            next_base = end = tiles_seen(p, rq, row_tile);
        }
        const uint32_t all = uint32_t(next_base - base), lo = uint32_t(at - base), hi = index_min(all, lo + (end - at));
        const Piece w = {head, request, row_tile, lo, hi, lo > 0 || hi < all, (uint64_t(block) * 2 + (lo > 0 ? 0 : 1)) * WAVES};
        uint64_t far = 0;
        if (tid == 0) lds.far = 0;
        chunk_piece<T, NB, WAVES, false>(p, lds, rq, w, far);
        if (far) lds.far = 1;  // (every writer writes the same)
        __syncthreads();
        if (lds.far) chunk_piece<T, NB, WAVES, true>(p, lds, rq, w, far);
        if (lo == 0 && hi < all) meta = make_uint4(request, row_tile, uint32_t((next_base - 1) / share) - worker + 1, 0);
        at += hi - lo;
        __syncthreads();
    }
    if (!ALONE && tid == 0) a.meta[block] = meta;
}

// The pieces of the row tile that begins in a worker and ends in another: a wave its 32 rows, four columns of each lane a block.
template <class T, int NB, int WAVES>
__global__ __launch_bounds__(WAVES * kWave) void k_cache_chunk_join(const ChunkArgs p) {
    const CacheAttnArgs& a = p.a;
    const uint4 meta = a.meta[blockIdx.x];
    if (!meta.z) return;
    const int lane = int(threadIdx.x) % kWave, wave = int(threadIdx.x) / kWave, n = lane % 32, h = lane / 32;
    const uint32_t head = blockIdx.x % a.c.kv_heads, which = blockIdx.y;
    f32x4_t o = {0.0f, 0.0f, 0.0f, 0.0f};
    float ref = kCacheNoRef, sum = 0.0f;
    for (uint32_t i = 0; i < meta.z; ++i) {
        const uint64_t piece = ((uint64_t(blockIdx.x) + uint64_t(i) * a.c.kv_heads) * 2 + (i ? 0 : 1)) * WAVES + uint64_t(wave);
        const f32x4_t x = *reinterpret_cast<const f32x4_t*>(a.part + ((piece * (8 * NB) + which) * kWave + uint64_t(lane)) * 4);
        const float r = a.stat[piece * 64 + uint64_t(n)], s = a.stat[piece * 64 + 32 + uint64_t(n)];
        const float top = fmaxf(ref, r);
        const int less = shift_of(ref, top), more = shift_of(r, top);
        o = shifted_all(o, less) + shifted_all(x, more);
        sum = shifted(sum, less) + shifted(s, more);
        ref = top;
    }
    const CacheRequest rq = request_of(a, meta.x);
    const uint32_t packed = meta.y * (WAVES * kWaveRows) + uint32_t(wave) * kWaveRows + uint32_t(n);
    store4<T>(a, rq, packed, head, which / 4 * 32 + which % 4 * 8 + 4 * uint32_t(h), o, sum);
    if (which == 0 && lane < 32) store_lse(a, rq, packed, head, ref, sum);
}

uint64_t pad256(uint64_t b) { return (b + 255) / 256 * 256; }

template <class T, int NB, int WAVES>
hipError_t launch(const ChunkArgs& p, hipStream_t s) {
    if (!p.a.workers) {
        k_cache_chunk<T, NB, WAVES, true><<<dim3(p.a.c.kv_heads, p.a.c.requests, p.a.row_tiles), WAVES * kWave, 0, s>>>(p);
        return hipGetLastError();
    }
    const uint32_t blocks = p.a.workers * p.a.c.kv_heads;
    k_cache_plan<<<1, kScan, 0, s>>>(p);
    if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    k_cache_chunk<T, NB, WAVES, false><<<dim3(p.a.c.kv_heads, p.a.workers), WAVES * kWave, 0, s>>>(p);
    if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    k_cache_chunk_join<T, NB, WAVES><<<dim3(blocks, 8 * NB), WAVES * kWave, 0, s>>>(p);
    return hipGetLastError();
}
// Waves a block: eight where requests may fill them, since a tile is then brought and turned for twice the rows (FP32's
// products need twice the registers, and leave room for four).  Measured with 16 requests of 4000 keys, 32 heads on 8 of 128
// columns, bf16, four waves against eight: 128 packed rows each 80 and 96 us, 160 114 and 105, 256 117 and 108, 384 162 and
// 172, 512 197 and 179, 1024 369 and 321.
int waves_of(const CacheSizes& c, bool bf16) { return bf16 && uint64_t(c.most) * c.group > 4 * kWaveRows ? 8 : 4; }

}  // namespace

uint32_t chunk_rows(const CacheSizes& c, bool bf16) { return uint32_t(waves_of(c, bf16)) * kWaveRows; }

ChunkPlan chunk_plan(int cus, const CacheSizes& c, bool bf16) {
    ChunkPlan p;
    const uint32_t tile = chunk_rows(c, bf16);
    p.tiles = uint32_t(c.rows * c.group / tile + c.requests);  // a request's last tile may be part full
    p.workers = uint32_t(std::max(1, (bf16 && waves_of(c, bf16) == 4 ? 2 : 1) * cus / int(c.kv_heads)));
    const uint64_t blocks = uint64_t(p.workers) * c.kv_heads, nb = c.dim > 64 ? 2 : 1;
    uint64_t at = 0;
    const auto take = [&](uint64_t bytes) {
        const uint64_t here = at;
        at += pad256(bytes);
        return here;
    };
    p.begin = take((uint64_t(c.requests) + 1) * 4);
    p.request = take(uint64_t(p.tiles) * 4);
    p.upto = take((uint64_t(p.tiles) + 1) * 8);
    p.part = take(blocks * 2 * tile * 64 * nb * 4);
    p.stat = take(blocks * 2 * tile * 8);
    p.meta = take(blocks * 16);
    p.bytes = at;
    return p;
}

hipError_t launch_cache_chunk(const CacheAttnArgs& args, bool bf16, const ChunkPlan& plan, void* workspace, hipStream_t s) {
    ChunkArgs p;
    p.a = args;
    char* const ws = static_cast<char*>(workspace);
    p.tiles = plan.tiles;
    const int waves = waves_of(args.c, bf16);
    p.tile_rows = chunk_rows(args.c, bf16);
    p.begin = reinterpret_cast<uint32_t*>(ws + plan.begin);
    p.request = reinterpret_cast<uint32_t*>(ws + plan.request);
    p.upto = reinterpret_cast<uint64_t*>(ws + plan.upto);
    p.a.part = reinterpret_cast<float*>(ws + plan.part);
    p.a.stat = reinterpret_cast<float*>(ws + plan.stat);
    p.a.meta = reinterpret_cast<uint4*>(ws + plan.meta);
    const bool wide = args.c.dim > 64;
    const auto as = [&](auto w) {
        constexpr int W = decltype(w)::value;
        return wide ? launch<uint16_t, 2, W>(p, s) : launch<uint16_t, 1, W>(p, s);
    };
    if (bf16) return waves == 8 ? as(std::integral_constant<int, 8>{}) : as(std::integral_constant<int, 4>{});
    return wide ? launch<float, 2, 4>(p, s) : launch<float, 1, 4>(p, s);
}

}  // namespace gatgpu
