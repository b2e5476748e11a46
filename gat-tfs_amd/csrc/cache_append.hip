// Keys and values of new tokens into the pages of an 8-bit cache.
//
//   e = max(e of the page if tokens stay, least e with max |x| <= 448 2^e over the page's new tokens)
//   byte = e4m3(x 2^-e);  a byte that stays becomes e4m3(byte 2^(old e - e))
//
// Bound by bytes: rows read once (two or four bytes a value), one byte a value written.  A block takes the new tokens of
// one page, key/value head and side (keys or values), reads them into registers, finds their largest magnitude and
// rounds them from there (what registers do not hold, of pages of 256 tokens, is read again).  Values are turned in LDS,
// since a page holds them by column: the attention's second product then takes its operands straight from memory.
#include <algorithm>
#include <string>

#include "cache.hpp"

namespace gatgpu {
namespace {

constexpr int kThreads = 256, kHeld = 8;  // 16-byte chunks of rows that a thread keeps
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

// Magnitude of a finite value as bits, which order as the values do; 0 of NaN and infinities.
__device__ inline uint32_t magnitude(uint32_t u) {
    u &= 0x7fffffffu;
    return u >= 0x7f800000u ? 0 : u;
}
// The least exponent e with m <= 448 2^e = 1.75 2^(8 + e), in the scales' range.
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
        x[i] = fminf(fmaxf(__uint_as_float(u[i]) * by, -448.0f), 448.0f);
        if ((u[i] & 0x7f800000u) == 0x7f800000u) bad |= 0x7fu << (8 * i);
    }
    uint32_t w = uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false));
    w = uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], int(w), true));
    return bad ? w | bad : w;
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
// 16 bytes of a row as FP32 bits.
template <class T>
struct Bits {
    uint32_t u[16 / sizeof(T)];
};
template <class T>
__device__ inline Bits<T> widen(uint4 w) {
    const uint32_t v[4] = {w.x, w.y, w.z, w.w};
    Bits<T> b;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 2) {
            b.u[2 * i] = v[i] << 16;
            b.u[2 * i + 1] = v[i] & 0xffff0000u;
        } else {
            b.u[i] = v[i];
        }
    }
    return b;
}

template <class T>
__global__ __launch_bounds__(kThreads) void k_cache_append(const AppendArgs a) {
    constexpr int N = 16 / int(sizeof(T));  // values a chunk
    extern __shared__ uint8_t turn[];       // values: [dim][page + kTurnPad]
    __shared__ uint32_t s_word[kThreads / kWave];
    __shared__ uint64_t s_starts;
    const int tid = int(threadIdx.x), lane = tid % kWave, wave = tid / kWave;
    const int head = int(blockIdx.y), side = int(blockIdx.z);
    const uint64_t first = uint64_t(blockIdx.x) * a.chunk;
    const uint32_t page = a.page;
    if (wave == 0) {
        const uint64_t row = first + uint64_t(lane);
        bool start = false;
        if (uint32_t(lane) < a.chunk && row < a.rows) {
            const uint32_t s = a.slot[row];
            start = s < a.slots && (row == 0 || s % page == 0 || a.slot[row - 1] + 1 != s);
        }
        const uint64_t some = __ballot(start);
        if (lane == 0) s_starts = some;
    }
    __syncthreads();
    for (uint64_t starts = s_starts; starts; starts &= starts - 1) {
        const uint64_t row = first + uint64_t(__builtin_ctzll(starts));
        const uint32_t slot = a.slot[row], off = slot % page;
        // Tokens of this page: rows as long as their slots go on.
        const bool more = row + uint64_t(tid) < a.rows && off + uint32_t(tid) < page && a.slot[row + uint64_t(tid)] == slot + uint32_t(tid);
        const uint64_t on = __ballot(more);
        if (lane == 0) s_word[wave] = ~on ? uint32_t(__builtin_ctzll(~on)) : uint32_t(kWave);
        __syncthreads();
        uint32_t tokens = 0;
        for (int w = 0; w < kThreads / kWave; ++w) {
            tokens += s_word[w];
            if (s_word[w] < uint32_t(kWave)) break;
        }
        __syncthreads();
        const uint32_t per = uint32_t(a.dim) / N, chunks = tokens * per;  // chunks a token, and in all
        const T* const x = static_cast<const T*>(a.x[side]) + row * a.xs[side] + uint64_t(head) * uint64_t(a.dim);
        const auto load = [&](uint32_t i) { return *reinterpret_cast<const uint4*>(x + uint64_t(i / per) * a.xs[side] + uint64_t(i % per) * N); };
        uint4 held[kHeld];
        uint32_t top = 0;
        const auto see = [&](uint4 w) {
            const Bits<T> b = widen<T>(w);
#pragma unroll
            for (int j = 0; j < N; ++j) top = max(top, magnitude(b.u[j]));
        };
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
            const uint32_t at = uint32_t(tid + i * kThreads);
            held[i] = at < chunks ? load(at) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < kHeld; ++i) see(held[i]);
        for (uint32_t at = uint32_t(tid + kHeld * kThreads); at < chunks; at += kThreads) see(load(at));
#pragma unroll
        for (int d = kWave / 2; d; d /= 2) top = max(top, uint32_t(__shfl_xor(int(top), d)));
        if (lane == 0) s_word[wave] = top;
        __syncthreads();
        top = max(max(s_word[0], s_word[1]), max(s_word[2], s_word[3]));
        const uint64_t place = uint64_t(slot / page) * uint64_t(a.kv_heads) + uint64_t(head);
        uint8_t* const to = a.cache[side] + place * page * uint64_t(a.dim);
        const int had = off ? scale_exponent(a.scale[side][place]) : kLeastScale;
        const int e = max(exponent_for(top), had);
        if (off && e > had) {  // the page's scale grows under the tokens that stay
            const float by = power_of_two(had - e < -126 ? -126 : had - e);
            if (side == 0) {
                uint32_t* const w = reinterpret_cast<uint32_t*>(to);
                for (uint32_t i = uint32_t(tid); i < off * uint32_t(a.dim) / 4; i += kThreads) w[i] = round_again(w[i], by);
            } else {
                const uint32_t words = (off + 3) / 4;
                for (uint32_t i = uint32_t(tid); i < words * uint32_t(a.dim); i += kThreads) {
                    const uint32_t at = i % words * 4;
                    uint32_t* const w = reinterpret_cast<uint32_t*>(to + uint64_t(i / words) * page + at);
                    const uint32_t stay = off - at >= 4 ? 0xffffffffu : (1u << (8 * (off - at))) - 1;
                    *w = (round_again(*w, by) & stay) | (*w & ~stay);
                }
            }
        }
        __syncthreads();  // (the scale has been read, and the words of tokens that stay are written)
        if (tid == 0) a.scale[side][place] = power_of_two(e);
        const float by = power_of_two(-e);
        const auto put = [&](uint32_t at, uint4 w) {
            const Bits<T> b = widen<T>(w);
            const uint32_t token = at / per, col = at % per * N;
            uint32_t q[N / 4];
#pragma unroll
            for (int i = 0; i < N / 4; ++i) {
                const uint32_t u[4] = {b.u[4 * i], b.u[4 * i + 1], b.u[4 * i + 2], b.u[4 * i + 3]};
                q[i] = round4(u, by);
            }
            if (side == 0) {
                uint8_t* const p = to + uint64_t(off + token) * uint64_t(a.dim) + col;
                if constexpr (N == 8) *reinterpret_cast<uint2*>(p) = make_uint2(q[0], q[1]);
                else *reinterpret_cast<uint32_t*>(p) = q[0];
            } else {
#pragma unroll
                for (int j = 0; j < N; ++j) turn[(col + uint32_t(j)) * (page + kTurnPad) + token] = uint8_t(q[j / 4] >> (8 * (j % 4)));
            }
        };
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
            const uint32_t at = uint32_t(tid + i * kThreads);
            if (at < chunks) put(at, held[i]);
        }
        for (uint32_t at = uint32_t(tid + kHeld * kThreads); at < chunks; at += kThreads) put(at, load(at));
        __syncthreads();
        if (side == 0) continue;
        if (tokens == page) {
            for (uint32_t i = uint32_t(tid); i < page / 16 * uint32_t(a.dim); i += kThreads) {
                const uint32_t col = i / (page / 16), at = i % (page / 16) * 16;
                const uint32_t* const w = reinterpret_cast<const uint32_t*>(turn + col * (page + kTurnPad) + at);
                *reinterpret_cast<uint4*>(to + uint64_t(col) * page + at) = make_uint4(w[0], w[1], w[2], w[3]);
            }
        } else {
            for (uint32_t i = uint32_t(tid); i < tokens * uint32_t(a.dim); i += kThreads) {
                const uint32_t col = i / tokens, at = i % tokens;
                to[uint64_t(col) * page + off + at] = turn[col * (page + kTurnPad) + at];
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
    if (io->rows >= (uint64_t(1) << 27)) return fail(c, GATGPU_EOVERFLOW, "more than 2^27 - 1 rows");  // (of a launch: 16 threads a row)
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
    // A block a row where most rows are their page's first (a token of each request), else 16 rows: prompts, in which at
    // most one or two of them are.
    a.chunk = io->rows <= 2048 ? 1 : 16;
    const dim3 grid(uint32_t((io->rows + a.chunk - 1) / a.chunk), uint32_t(cache->kv_heads), 2);
    const size_t lds = size_t(cache->dim) * (cache->page + kTurnPad);
    if (io->precision == GATGPU_BF16) k_cache_append<uint16_t><<<grid, kThreads, lds, c->stream>>>(a);
    else k_cache_append<float><<<grid, kThreads, lds, c->stream>>>(a);
    HIPCHECK(c, hipGetLastError());
    return GATGPU_OK;
}
