// Keys and values of new tokens into the pages of an 8-bit cache.
//
//   e = max(e of the page if tokens stay, least e with max |x| <= 448 2^e over the page's new tokens)
//   byte = e4m3(x 2^-e);  a byte that stays becomes e4m3(byte 2^(old e - e))
//
// Bound by bytes: rows read once (two or four bytes a value), one byte a value written.  A block takes the new tokens of
// one page and key/value head, reads their keys and values into registers, finds the largest magnitudes and rounds
// them from there (what registers do not hold, beyond 16 KB of each, is read again).  Values are turned in LDS,
// since a page holds them by column: the attention's second product then takes its operands straight from memory.
//
// 24 prompts of 54 thousand tokens, 8 heads of 128, bf16: 77 us, 4.3 TB/s; 96 requests of one token 6.1 us, a launch and a chain
// of reads (slots, scale, row), then a byte of a line for each of a value's columns.
#include <algorithm>
#include <string>

#include "cache.hpp"

namespace gatgpu {
namespace {

constexpr int kThreads = 256;
constexpr uint32_t kShort = 4;  // tokens of a page that a wave takes by itself
constexpr int kMaxPage = 256, kMaxDim = 128, kTurnPad = 4;

struct AppendArgs {
    uint64_t rows = 0;
    uint32_t chunk = 1;  // rows among which a block looks for the first tokens of pages
    uint32_t page = 0, slots = 0;
    int kv_heads = 0, dim = 0;
    const void* x[2] = {};  // rows of keys and of values
    uint64_t xs[2] = {};
    const uint32_t* slot = nullptr;
    uint8_t* cache[2] = {};
    float* scale[2] = {};
};

constexpr uint32_t kInfinity = 0x7f800000u;
// The least exponent e with m <= 448 2^e = 1.75 2^(8 + e), in the scales' range; m: bits of a finite magnitude.
__device__ inline int exponent_for(uint32_t m) {
    const int e = int(m >> 23) - 127 - 8 + ((m & 0x7fffffu) > 0x600000u ? 1 : 0);
    return e < kLeastScale ? kLeastScale : e > kMostScale ? kMostScale : e;
}
// Four values (bits) to e4m3 bytes.
__device__ inline uint32_t round4(const uint32_t (&u)[4], float by) {
    float x[4];
    uint32_t bad = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[i] = __builtin_amdgcn_fmed3f(__uint_as_float(u[i]) * by, -448.0f, 448.0f);
        if ((u[i] & kInfinity) == kInfinity) bad |= 0x7fu << (8 * i);
    }
    uint32_t w = uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false));
    w = uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], int(w), true));
    return w | bad;
}
// Four bytes of a page whose scale grows.
__device__ inline uint32_t round_again(uint32_t w, float by) {
    uint32_t u[4];
    u[0] = __float_as_uint(__builtin_amdgcn_cvt_f32_fp8(int(w), 0));
    u[1] = __float_as_uint(__builtin_amdgcn_cvt_f32_fp8(int(w), 1));
    u[2] = __float_as_uint(__builtin_amdgcn_cvt_f32_fp8(int(w), 2));
    u[3] = __float_as_uint(__builtin_amdgcn_cvt_f32_fp8(int(w), 3));
    return round4(u, by);
}

// 16 bytes of four neighbouring tokens' rows, zeros behind the last token.
struct Quad {
    uint4 row[4];
};
template <class T>
__device__ inline void widen(uint4 w, uint32_t (&u)[16 / sizeof(T)]) {
    const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 2) {
            u[2 * i] = v[i] << 16;
            u[2 * i + 1] = v[i] & 0xffff0000u;
        } else {
            u[i] = v[i];
        }
    }
}
// The largest magnitude among a quad's values, as FP32 bits, which order as magnitudes do; NaN and infinities beyond kInfinity.
template <class T>
__device__ inline uint32_t largest(const Quad& q) {
    uint32_t top = 0;
    if constexpr (sizeof(T) == 2) {
        typedef unsigned short u16x2_t __attribute__((ext_vector_type(2)));
        u16x2_t m = {0, 0};
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2_t, (&q.row[i].x)[k] & 0x7fff7fffu));
        top = uint32_t(max(m[0], m[1])) << 16;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k) top = max(top, (&q.row[i].x)[k] & 0x7fffffffu);
    }
    return top;
}
// The same among the finite ones.
template <class T>
__device__ inline uint32_t largest_finite(const Quad& q) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t u[16 / sizeof(T)];
        widen<T>(q.row[i], u);
#pragma unroll
        for (int k = 0; k < int(16 / sizeof(T)); ++k) top = max(top, (u[k] & kInfinity) == kInfinity ? 0u : u[k] & 0x7fffffffu);
    }
    return top;
}
__device__ inline void block_max(uint32_t (&x)[2], uint32_t (*words)[kThreads / kWave]) {
#pragma unroll
    for (int d = kWave / 2; d; d /= 2) {
        x[0] = max(x[0], uint32_t(__shfl_xor(int(x[0]), d)));
        x[1] = max(x[1], uint32_t(__shfl_xor(int(x[1]), d)));
    }
    __syncthreads();
    if (threadIdx.x % kWave == 0) {
        words[0][threadIdx.x / kWave] = x[0];
        words[1][threadIdx.x / kWave] = x[1];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) x[i] = max(max(words[i][0], words[i][1]), max(words[i][2], words[i][3]));
}

// Where the new tokens of a page go, for one head and side.
template <class T>
struct Run {
    const T* x;       // the first one's row
    uint64_t stride;  // from row to row
    uint8_t* to;      // the page's bytes
    float* scale;
    uint32_t off;     // tokens before them
};
template <class T>
__device__ inline Run<T> run_at(const AppendArgs& a, uint64_t row, uint32_t slot, int head, int side) {
    Run<T> r;
    const uint64_t place = uint64_t(slot / a.page) * uint64_t(a.kv_heads) + uint64_t(head);
    r.x = static_cast<const T*>(a.x[side]) + row * a.xs[side] + uint64_t(head) * uint64_t(a.dim);
    r.stride = a.xs[side];
    r.to = a.cache[side] + place * a.page * uint64_t(a.dim);
    r.scale = a.scale[side] + place;
    r.off = slot % a.page;
    return r;
}
// Piece i of four neighbouring tokens' rows: i / per fours, i % per pieces of 16 bytes.
template <class T>
__device__ inline Quad load_quad(const Run<T>& r, uint32_t tokens, uint32_t per, uint32_t i) {
    constexpr uint32_t N = 16 / sizeof(T);
    Quad q;
    const uint32_t t = i / per * 4;
    const T* const p = r.x + uint64_t(t) * r.stride + uint64_t(i % per) * N;
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k) q.row[k] = t + k < tokens ? *reinterpret_cast<const uint4*>(p + k * r.stride) : make_uint4(0, 0, 0, 0);
    return q;
}
// Bytes of the tokens that stay, from exponent `had` to e, by `threads` threads.
__device__ inline void grow(uint8_t* to, uint32_t off, uint32_t page, uint32_t dim, int had, int e, int side, uint32_t thread, uint32_t threads) {
    const float by = power_of_two(had - e < -126 ? -126 : had - e);
    if (side == 0) {
        uint32_t* const w = reinterpret_cast<uint32_t*>(to);
        for (uint32_t i = thread; i < off * dim / 4; i += threads) w[i] = round_again(w[i], by);
    } else {
        const uint32_t words = (off + 3) / 4;
        for (uint32_t i = thread; i < words * dim; i += threads) {
            const uint32_t at = i % words * 4;
            uint32_t* const w = reinterpret_cast<uint32_t*>(to + uint64_t(i / words) * page + at);
            const uint32_t stay = off - at >= 4 ? 0xffffffffu : (1u << (8 * (off - at))) - 1;
            *w = (round_again(*w, by) & stay) | (*w & ~stay);
        }
    }
}
// A piece's tokens t ... t + 3 as keys: N columns of a token side by side.
template <class T>
__device__ inline void put_keys(uint8_t* to, uint32_t dim, uint32_t tokens, uint32_t t, const uint32_t (&u)[4][16 / sizeof(T)], float by) {
    constexpr int N = 16 / int(sizeof(T));
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k) {
        if (t + k >= tokens) break;
        uint32_t w[N / 4];
#pragma unroll
        for (int c = 0; c < N / 4; ++c) {
            const uint32_t v[4] = {u[k][4 * c], u[k][4 * c + 1], u[k][4 * c + 2], u[k][4 * c + 3]};
            w[c] = round4(v, by);
        }
        uint32_t* const p = reinterpret_cast<uint32_t*>(to + uint64_t(k) * dim);
        if constexpr (N == 8) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
        else *p = w[0];
    }
}

// A page's few tokens, by a wave: a lane a piece of the rows.
template <class T>
__device__ inline void append_short(const AppendArgs& a, uint64_t row, uint32_t tokens, int head, int side) {
    constexpr int N = 16 / int(sizeof(T));
    const uint32_t lane = threadIdx.x % kWave, per = uint32_t(a.dim) / N, page = a.page;
    const Run<T> r = run_at<T>(a, row, a.slot[row], head, side);
    const float scale = *r.scale;
    Quad q{};
    if (lane < per) q = load_quad(r, tokens, per, lane);
    uint32_t top = largest<T>(q);
#pragma unroll
    for (int d = kWave / 2; d; d /= 2) top = max(top, uint32_t(__shfl_xor(int(top), d)));
    if (top >= kInfinity) {  // NaN and infinities leave the scale alone
        top = largest_finite<T>(q);
#pragma unroll
        for (int d = kWave / 2; d; d /= 2) top = max(top, uint32_t(__shfl_xor(int(top), d)));
    }
    const int had = r.off ? scale_exponent(scale) : kLeastScale, e = max(exponent_for(top), had);
    if (r.off && e > had) {
        grow(r.to, r.off, page, uint32_t(a.dim), had, e, side, lane, kWave);
        __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "workgroup");  // (words that hold new tokens too are written before these)
    }
    if (lane == 0) *r.scale = power_of_two(e);
    if (lane >= per) return;
    const float by = power_of_two(-e);
    uint32_t u[4][N];
#pragma unroll
    for (int k = 0; k < 4; ++k) widen<T>(q.row[k], u[k]);
    if (side == 0) {
        put_keys<T>(r.to + uint64_t(r.off) * uint64_t(a.dim) + lane * N, uint32_t(a.dim), tokens, 0, u, by);
    } else {
#pragma unroll
        for (uint32_t c = 0; c < uint32_t(N); ++c) {
            const uint32_t v[4] = {u[0][c], u[1][c], u[2][c], u[3][c]}, w = round4(v, by);
            uint8_t* const p = r.to + uint64_t(lane * N + c) * page + r.off;
            for (uint32_t k = 0; k < tokens; ++k) p[k] = uint8_t(w >> (8 * k));
        }
    }
}

// Bits 0 to 63 of a 128-bit word from bit `at` on.
struct Bits128 {
    uint64_t lo, hi;
    __device__ uint64_t from(uint32_t at) const { return at ? lo >> at | hi << (64 - at) : lo; }
};

// A block looks for the first tokens of pages among `chunk` rows, and sees 128.  A page's few tokens (a request's new one)
// are a wave's, others the block's, keys and values at once: a thread takes 16 bytes of four neighbouring tokens of each, a
// row's bytes lie in neighbouring lanes, and four tokens' values of a column make one word of the page's column.
template <class T>
__global__ __launch_bounds__(kThreads, 4) void k_cache_append(const AppendArgs a) {
    constexpr int N = 16 / int(sizeof(T));  // values of 16 bytes
    extern __shared__ uint32_t turn[];      // values: [dim][page + kTurnPad] bytes
    __shared__ uint32_t s_word[2][kThreads / kWave];
    __shared__ uint64_t s_starts;
    __shared__ Bits128 s_goes_on;
    const int tid = int(threadIdx.x), lane = tid % kWave, wave = tid / kWave;
    const int head = int(blockIdx.y);
    const uint64_t first = uint64_t(blockIdx.x) * a.chunk;
    const uint32_t page = a.page, dim = uint32_t(a.dim), turn_row = (page + kTurnPad) / 4, per = dim / N;  // words, 16-byte pieces a token
    if (wave < 2) {
        const uint64_t row = first + uint64_t(tid);
        bool there = false, goes_on = false;  // goes on: the token after that of the row before, in its page
        if (row < a.rows) {
            const uint32_t s = a.slot[row], before = row ? a.slot[row - 1] : GATGPU_NO_PAGE;
            there = s < a.slots;
            goes_on = there && row && s % page && before + 1 == s;
        }
        const uint64_t on = __ballot(goes_on), starts = __ballot(there && !goes_on && uint32_t(tid) < a.chunk);
        if (lane == 0) {
            if (wave == 0) {
                s_starts = starts;
                s_goes_on.lo = on;
            } else {
                s_goes_on.hi = on;
            }
        }
    }
    __syncthreads();
    uint32_t number = 0;
    uint64_t longer = 0;
    for (uint64_t left = s_starts; left; left &= left - 1) {
        const uint32_t at = uint32_t(__builtin_ctzll(left));
        const uint64_t on = s_goes_on.from(at) >> 1;
        const uint32_t tokens = ~on ? 1 + uint32_t(__builtin_ctzll(~on)) : 64;
        if (tokens > kShort) {
            longer |= left & (~left + 1);
        } else {
            for (int side = 0; side < 2; ++side)
                if (int(number++ % (kThreads / kWave)) == wave) append_short<T>(a, first + at, tokens, head, side);
        }
    }
    for (uint64_t left = longer; left; left &= left - 1) {
        const uint32_t at = uint32_t(__builtin_ctzll(left));
        const uint64_t row = first + at, on = s_goes_on.from(at) >> 1;
        const uint32_t slot = a.slot[row], off = slot % page;
        const Run<T> runs[2] = {run_at<T>(a, row, slot, head, 0), run_at<T>(a, row, slot, head, 1)};
        const float scale[2] = {*runs[0].scale, *runs[1].scale};
        uint32_t tokens = uint32_t(__builtin_ctzll(~on)) + 1;  // (63 bits of `on` are seen)
        if (!(~on << 1)) {  // 64 tokens are seen, and there may be more: rows as long as their slots go on
            const bool more = row + uint64_t(tid) < a.rows && off + uint32_t(tid) < page && a.slot[row + uint64_t(tid)] == slot + uint32_t(tid);
            const uint64_t some = __ballot(more);
            __syncthreads();
            if (lane == 0) s_word[0][wave] = ~some ? uint32_t(__builtin_ctzll(~some)) : uint32_t(kWave);
            __syncthreads();
            tokens = 0;
            for (int w = 0; w < kThreads / kWave; ++w) {
                tokens += s_word[0][w];
                if (s_word[0][w] < uint32_t(kWave)) break;
            }
        }
        const uint32_t quads = (tokens + 3) / 4 * per;
        Quad held[2] = {};  // the thread's first ones; more than 256 of them are read again
        uint32_t top[2];
        if (uint32_t(tid) < quads) {
            held[0] = load_quad(runs[0], tokens, per, uint32_t(tid));
            held[1] = load_quad(runs[1], tokens, per, uint32_t(tid));
        }
#pragma unroll
        for (int side = 0; side < 2; ++side) {
            top[side] = largest<T>(held[side]);
            for (uint32_t i = uint32_t(tid) + kThreads; i < quads; i += kThreads) top[side] = max(top[side], largest<T>(load_quad(runs[side], tokens, per, i)));
        }
        block_max(top, s_word);
        if (max(top[0], top[1]) >= kInfinity) {  // NaN and infinities leave the scale alone
#pragma unroll
            for (int side = 0; side < 2; ++side) {
                top[side] = largest_finite<T>(held[side]);
                for (uint32_t i = uint32_t(tid) + kThreads; i < quads; i += kThreads)
                    top[side] = max(top[side], largest_finite<T>(load_quad(runs[side], tokens, per, i)));
            }
            block_max(top, s_word);
        }
        int e[2];
        bool grows = false;
#pragma unroll
        for (int side = 0; side < 2; ++side) {
            const int had = off ? scale_exponent(scale[side]) : kLeastScale;
            e[side] = max(exponent_for(top[side]), had);
            if (off && e[side] > had) {
                grow(runs[side].to, off, page, dim, had, e[side], side, uint32_t(tid), kThreads);
                grows = true;
            }
        }
        if (grows) __syncthreads();  // (words that hold new tokens too are written before these)
        const float by[2] = {power_of_two(-e[0]), power_of_two(-e[1])};
        const auto put = [&](int side, uint32_t i, const Quad& q) {
            const uint32_t t = i / per * 4, col = i % per * N;
            uint32_t u[4][N];
#pragma unroll
            for (int k = 0; k < 4; ++k) widen<T>(q.row[k], u[k]);
            if (side == 0) {
                put_keys<T>(runs[0].to + uint64_t(off + t) * dim + col, dim, tokens, t, u, by[0]);
            } else {
#pragma unroll
                for (int c = 0; c < N; ++c) {
                    const uint32_t v[4] = {u[0][c], u[1][c], u[2][c], u[3][c]};
                    turn[(col + uint32_t(c)) * turn_row + t / 4] = round4(v, by[1]);
                }
            }
        };
#pragma unroll
        for (int side = 1; side >= 0; --side) {
            if (uint32_t(tid) < quads) put(side, uint32_t(tid), held[side]);
            for (uint32_t i = uint32_t(tid) + kThreads; i < quads; i += kThreads) put(side, i, load_quad(runs[side], tokens, per, i));
        }
        __syncthreads();  // (the scales have been read by all, too)
        if (tid < 2) *(tid ? runs[1].scale : runs[0].scale) = power_of_two(tid ? e[1] : e[0]);
        if (tokens == page) {
            const uint32_t pieces = page / 16;
            for (uint32_t i = uint32_t(tid); i < pieces * dim; i += kThreads) {
                const uint32_t* const w = turn + i / pieces * turn_row + i % pieces * 4;
                *reinterpret_cast<uint4*>(runs[1].to + uint64_t(i) * 16) = make_uint4(w[0], w[1], w[2], w[3]);
            }
        } else {
            const uint8_t* const bytes = reinterpret_cast<const uint8_t*>(turn);
            for (uint32_t i = uint32_t(tid); i < tokens * dim; i += kThreads) {
                const uint32_t col = i / tokens, of = i % tokens;
                runs[1].to[uint64_t(col) * page + off + of] = bytes[col * turn_row * 4 + of];
            }
        }
        __syncthreads();
    }
}

}  // namespace

int check_cache(gatgpu_ctx* c, const gatgpu_cache* cache, bool arrays) {
    if (!cache) return fail(c, GATGPU_EINVAL, "null cache");
    if (cache->page < 16 || cache->page > uint32_t(kMaxPage) || (cache->page & (cache->page - 1)))
        return fail(c, GATGPU_EINVAL, "page must be 16, 32, 64, 128 or 256");
    if (!cache->pages) return fail(c, GATGPU_EINVAL, "a cache has at least one page");
    if (uint64_t(cache->pages) * cache->page >= (uint64_t(1) << 32)) return fail(c, GATGPU_EOVERFLOW, "pages * page must be below 2^32");
    if (cache->kv_heads < 1 || cache->kv_heads > 64) return fail(c, GATGPU_EINVAL, "kv_heads must be 1 to 64");
    if (cache->dim < 16 || cache->dim > kMaxDim || cache->dim % 16) return fail(c, GATGPU_EINVAL, "dim must be a multiple of 16, at most 128");
    if (!arrays) return GATGPU_OK;
    const void* const p[4] = {cache->k, cache->v, cache->k_scale, cache->v_scale};
    const char* const name[4] = {"k of the cache", "v of the cache", "k_scale", "v_scale"};
    for (int i = 0; i < 4; ++i) {
        if (!p[i]) return fail(c, GATGPU_EINVAL, std::string("null ") + name[i]);
        if (reinterpret_cast<uintptr_t>(p[i]) % 16) return fail(c, GATGPU_EINVAL, std::string(name[i]) + " must be 16-byte aligned");
        if (int r = check_device_array(c, p[i], name[i])) return r;
    }
    return GATGPU_OK;
}

}  // namespace gatgpu

namespace {

using namespace gatgpu;

int check_rows(gatgpu_ctx* c, const gatgpu_cache* cache, const gatgpu_append_io* io, const char* name, const void* p, uint64_t stride) {
    if (!p) return fail(c, GATGPU_EINVAL, std::string("null ") + name);
    const uint64_t size = io->precision == GATGPU_BF16 ? 2 : 4;
    if (stride < uint64_t(cache->kv_heads) * uint64_t(cache->dim) || stride > (uint64_t(1) << 44))
        return fail(c, GATGPU_EINVAL, std::string(name) + " has a bad row stride");
    if (reinterpret_cast<uintptr_t>(p) % 16 || stride * size % 16) return fail(c, GATGPU_EINVAL, std::string(name) + " and its stride must be 16-byte aligned");
    return check_device_array(c, p, name);
}

}  // namespace

extern "C" int gatgpu_cache_append(gatgpu_ctx* c, const gatgpu_cache* cache, const gatgpu_append_io* io) {
    if (!c) return fail(nullptr, GATGPU_EINVAL, "null context");
    DeviceGuard on(c->device);
    if (!on.ok) return fail(c, GATGPU_EDEVICE, "cannot select the context's device");
    if (int r = check_cache(c, cache, true)) return r;
    if (!io) return fail(c, GATGPU_EINVAL, "null arrays");
    if (io->precision != GATGPU_FP32 && io->precision != GATGPU_BF16) return fail(c, GATGPU_EINVAL, "bad precision");
    if (io->rows >= (uint64_t(1) << 27)) return fail(c, GATGPU_EOVERFLOW, "more than 2^27 - 1 rows");  // (2^21 blocks: a block takes 64 of so many rows)
    if (!io->rows) return GATGPU_OK;
    if (int r = check_rows(c, cache, io, "k", io->k, io->k_stride)) return r;
    if (int r = check_rows(c, cache, io, "v", io->v, io->v_stride)) return r;
    if (!io->slot) return fail(c, GATGPU_EINVAL, "null slot");
    if (reinterpret_cast<uintptr_t>(io->slot) % 4) return fail(c, GATGPU_EINVAL, "slot must be 4-byte aligned");
    if (int r = check_device_array(c, io->slot, "slot")) return r;
    AppendArgs a;
    a.rows = io->rows;
    a.page = cache->page;
    a.slots = cache->pages * cache->page;
    a.kv_heads = cache->kv_heads;
    a.dim = cache->dim;
    a.x[0] = io->k;
    a.x[1] = io->v;
    a.xs[0] = io->k_stride;
    a.xs[1] = io->v_stride;
    a.slot = io->slot;
    a.cache[0] = cache->k;
    a.cache[1] = cache->v;
    a.scale[0] = cache->k_scale;
    a.scale[1] = cache->v_scale;
    // Rows of a block: as many as leave four blocks a unit, from two (a token of each request: a wave its keys, one its values)
    // to the 64 that one mask holds, since the length of a page's run is not known here and a block without one is not free.
    // By 2, by 16 and by 64, 8 heads of 128, bf16: 96 requests of a token 5.7, 21 and 74 us, 1000 21, 27 and 79; 4 prompts of
    // 1000 tokens 37, 11 and 12; 100 of 64 176, 30 and 12.
    const uint64_t rows_a_block = io->rows * uint64_t(cache->kv_heads) / uint64_t(4 * c->cus);
    a.chunk = uint32_t(std::min<uint64_t>(std::max<uint64_t>(rows_a_block, 2), 64));
    const dim3 grid(uint32_t((io->rows + a.chunk - 1) / a.chunk), uint32_t(cache->kv_heads));
    const size_t lds = size_t(cache->dim) * (cache->page + kTurnPad);
    if (io->precision == GATGPU_BF16) k_cache_append<uint16_t><<<grid, kThreads, lds, c->stream>>>(a);
    else k_cache_append<float><<<grid, kThreads, lds, c->stream>>>(a);
    HIPCHECK(c, hipGetLastError());
    return GATGPU_OK;
}
