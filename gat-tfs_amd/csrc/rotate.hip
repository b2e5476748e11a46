// Norms and rotation of queries and keys, forward and backward.
//
//   r = 1 / sqrt(mean(x^2) + eps),  n = x r,  t = n gamma          (without a norm: t = x)
//   y_i = t_i c_i + t_p s_i, p the other column of i's pair, s_i = -sin for the first of a pair, sin for the second
//   dt_i = dy_i c_i - dy_p s_i,  dgamma = sum dt n,  g = dt gamma,  dx = r (g - n mean(g n))
//
// Bound by bytes: a head's vector is read once into TPV lanes of 16 bytes each, and written once.  The other column of
// a pair half a rotation away comes by a second read of the same lines, which the first has just brought.  A row's angles are formed once a block, a thread an angle, in 64
// bits: position * freq in turns, of which the whole ones go before what is left is rounded to 32 bits, so that far
// positions keep an angle's error of 2^-23.  Groups of lanes then take the row's heads in turn with their columns' sines
// in registers.  The backward pass gives each block a fixed set of rows and keeps its columns' sums for gamma in
// registers over them; blocks leave one partial row each, added in one fixed order.
//
// 20011 rows of 20 heads of 128, bf16: forward 42 us, 4.9 TB/s of the 2 rows, backward 80 us, 3.9 TB/s of 3, the partial
// rows' sums 4.6.  7 rows of 16 heads of 64: 3.7 us, a launch.
#include <algorithm>
#include <cmath>
#include <string>
#include <type_traits>

#include "context.hpp"
#include "norm.hpp"

namespace gatgpu {
namespace {

constexpr int kBlock = 256;
// A vector whose mean square (with eps) lies beyond these is multiplied by a power of two and its squares are formed again, so
// that they stay among FP32's normal numbers: n is the same, and dx's factor takes the power.
constexpr float kLeastSquare = 0x1p-100f, kMostSquare = 0x1p120f, kEnlarge = 0x1p96f, kReduce = 0x1p-80f;

struct RotateArgs {
    uint64_t rows = 0;
    int heads = 0, kv_heads = 0, dim = 0, norm = 0, half = 0, neighbours = 0;
    int gpt = 0;  // groups of lanes a row
    float eps = 0.0f;
    // Vectors of the queries and of the keys
    const void *x[2] = {}, *dy[2] = {};
    void* y[2] = {};  // forward: q_out, k_out; backward: dq, dk
    uint64_t xs[2] = {}, dys[2] = {}, ys[2] = {};
    const float* gamma[2] = {};
    const uint32_t* position = nullptr;
    const double* freq = nullptr;
    float* part = nullptr;  // [blocks][2][dim], or null
};

template <class T>
struct Chunk {
    static constexpr int N = 16 / int(sizeof(T));
    float x[N];
};
template <class T>
__device__ inline Chunk<T> widen(uint4 w) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
    Chunk<T> c;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 2) {
            c.x[2 * i] = __uint_as_float(u[i] << 16);
            c.x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
        } else {
            c.x[i] = __uint_as_float(u[i]);
        }
    }
    return c;
}
template <class T>
__device__ inline uint4 load16(const T* p) {
    return *reinterpret_cast<const uint4*>(p);
}
// Bits of a NaN may change, nothing else does beside the rounding to nearest even.
template <class T>
__device__ inline void store_chunk(T* p, const Chunk<T>& c) {
    if constexpr (sizeof(T) == 2)
        *reinterpret_cast<uint4*>(p) = make_uint4(bf16x2(c.x[0], c.x[1]), bf16x2(c.x[2], c.x[3]), bf16x2(c.x[4], c.x[5]), bf16x2(c.x[6], c.x[7]));
    else
        *reinterpret_cast<float4*>(p) = make_float4(c.x[0], c.x[1], c.x[2], c.x[3]);
}
template <class T>
__device__ inline float load_one(const T* p) {
    if constexpr (sizeof(T) == 2) return bf16_widen(*p);
    else return *p;
}
template <int CTRL>
__device__ inline float add_dpp(float x) {
    return x + __uint_as_float(uint32_t(__builtin_amdgcn_mov_dpp(int(__float_as_uint(x)), CTRL, 0xf, 0xf, true)));
}
// Sum over groups of TPV lanes, in each of them: within quads by quad permutes, then of mirrored halves of 8 and 16 lanes
// (whose lanes are equal by then), then as the row halves swap.
template <int TPV>
__device__ inline float group_sum(float x) {
    if (TPV > 1) x = add_dpp<0xb1>(x);
    if (TPV > 2) x = add_dpp<0x4e>(x);
    if (TPV > 4) x = add_dpp<0x141>(x);
    if (TPV > 8) x = add_dpp<0x140>(x);
    if (TPV > 16) x = xor16_add(x);
    if (TPV > 32) x = xor32_add(x);
    return x;
}
// 1 / sqrt(x), x among FP32's normal numbers: the hardware's, and one step of Newton's method on it.
__device__ inline float inverse_root(float x) {
    const float r = __builtin_amdgcn_rsqf(x), h = 0.5f * x * r;
    return x < INFINITY ? fmaf(r, fmaf(-h, r, 0.5f), r) : r;
}

// A vector's place.
template <class T>
struct Vector {
    const T* x;   // what is rotated: the row, or backward the gradient's
    const T* n;   // backward: the row itself
    T* to;
    int which;    // 0 queries, 1 keys
};
template <class T, bool BACK>
__device__ inline Vector<T> vector_at(const RotateArgs& a, uint64_t row, int v) {
    Vector<T> p;
    p.which = v >= a.heads;
    const uint64_t at = uint64_t(p.which ? v - a.heads : v) * uint64_t(a.dim);
    const T* const x = static_cast<const T*>(a.x[p.which]) + row * a.xs[p.which] + at;
    p.to = static_cast<T*>(a.y[p.which]) + row * a.ys[p.which] + at;
    p.n = x;
    p.x = BACK ? static_cast<const T*>(a.dy[p.which]) + row * a.dys[p.which] + at : x;
    return p;
}
// A lane's 16 bytes of a vector as they come: its columns, those of its pairs' other ones (0 where there are none or they
// stand in the same chunk), and backward the row's.
struct Raw {
    uint4 own, other, n;
};
// The other columns of a chunk: kSame: in the chunk itself; kChunk: half a rotation away, a chunk for a chunk; both where
// a chunk turns as a whole or not at all.  kAny: any.
enum { kSame = 0, kChunk = 1, kAny = 2 };
template <class T, bool BACK, int PAIRS>
__device__ inline Raw fetch(const RotateArgs& a, const Vector<T>& p, int col) {
    Raw r;
    r.own = load16(p.x + col);
    r.other = r.n = make_uint4(0, 0, 0, 0);
    if (PAIRS == kChunk && col < 2 * a.half) r.other = load16(p.x + (col < a.half ? col + a.half : col - a.half));
    if (BACK && a.norm) r.n = load16(p.n + col);
    return r;
}
// The other column of column i, or i.
__device__ inline int partner_of(const RotateArgs& a, int i) {
    if (i >= 2 * a.half) return i;
    return a.neighbours ? i ^ 1 : i < a.half ? i + a.half : i - a.half;
}
template <class T, int PAIRS>
__device__ inline Chunk<T> partners(const RotateArgs& a, const Vector<T>& p, const Chunk<T>& own, uint4 other, int col) {
    if (PAIRS == kChunk) return widen<T>(other);
    Chunk<T> c;
#pragma unroll
    for (int j = 0; j < Chunk<T>::N; ++j) {
        if (PAIRS == kSame) c.x[j] = col < 2 * a.half ? own.x[j ^ 1] : 0.0f;
        else c.x[j] = col + j < 2 * a.half ? load_one(p.x + partner_of(a, col + j)) : 0.0f;
    }
    return c;
}
// A lane's factors of its columns and of their pairs' other ones (forward with gamma in them), and gamma.
template <class T>
struct Factors {
    Chunk<T> own, other, gamma;
};
// gamma: of the vector's kind, turn: of its row, both in LDS.
template <class T, bool BACK, int PAIRS>
__device__ inline void load_factors(const RotateArgs& a, const float* gamma, const float2* turn, int col, Factors<T>& f) {
    constexpr int N = Chunk<T>::N;
    float c[N], s[N], theirs[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
        f.gamma.x[j] = theirs[j] = gamma[col + j];
        c[j] = 1.0f;
        s[j] = 0.0f;
    }
    if (PAIRS == kAny) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int i = col + j;
            if (i < 2 * a.half) {
                const bool second = a.neighbours ? i & 1 : i >= a.half;
                const float2 w = turn[a.neighbours ? i / 2 : second ? i - a.half : i];
                c[j] = w.x;
                s[j] = second != BACK ? w.y : -w.y;
                theirs[j] = gamma[partner_of(a, i)];
            }
        }
    } else if (col < 2 * a.half) {
        const bool late = PAIRS == kChunk && col >= a.half;
        const float2* const at = turn + (PAIRS == kSame ? col / 2 : late ? col - a.half : col);
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const float2 w = at[PAIRS == kSame ? j / 2 : j];
            c[j] = w.x;
            s[j] = (PAIRS == kSame ? bool(j & 1) : late) != BACK ? w.y : -w.y;
            if (!BACK) theirs[j] = PAIRS == kSame ? f.gamma.x[j ^ 1] : gamma[(late ? col - a.half : col + a.half) + j];
        }
    }
#pragma unroll
    for (int j = 0; j < N; ++j) {
        f.own.x[j] = BACK ? c[j] : c[j] * f.gamma.x[j];
        f.other.x[j] = BACK ? s[j] : s[j] * theirs[j];
    }
}

// Rows at once: a group of TPV lanes takes heads g % gpt, g % gpt + gpt, ... of row g / gpt, each vector's bytes requested
// while the one before is worked on, across the rows that the block takes in turn; the next rows' angles are formed
// meanwhile, in the other of two buffers.
template <class T, int TPV, bool BACK, int PAIRS>
__global__ __launch_bounds__(kBlock, BACK ? 3 : 4) void k_rotate(const RotateArgs a) {
    constexpr int N = Chunk<T>::N, G = kBlock / TPV;
    constexpr int ANGLES = (G * TPV * N / 2 + kBlock - 1) / kBlock;  // of a thread, at most
    extern __shared__ float lds[];
    float* const gamma = lds;                                         // [2][dim]
    float2* const turn = reinterpret_cast<float2*>(lds + 2 * a.dim);  // [2][rows at once][half]
    const int tid = int(threadIdx.x), g = tid / TPV, col = tid % TPV * N, mine = g / a.gpt, start = g % a.gpt;
    const int at_once = G / a.gpt, vectors = a.heads + a.kv_heads, angles = at_once * a.half;
    const uint64_t stride = uint64_t(gridDim.x) * uint64_t(at_once);
    const bool there = col < a.dim, any = start < vectors;
    const float per = 1.0f / float(a.dim);
    const int step = a.gpt * a.dim;
    uint64_t first = uint64_t(blockIdx.x) * uint64_t(at_once);

    double freq[ANGLES];  // turns a position
    uint32_t position[ANGLES];
    const auto load_positions = [&](uint64_t from) {
#pragma unroll
        for (int k = 0; k < ANGLES; ++k) {
            const int i = tid + k * kBlock;
            position[k] = 0;
            if (i < angles && from + uint64_t(i / a.half) < a.rows) position[k] = a.position[from + uint64_t(i / a.half)];
        }
    };
    const auto form_angles = [&](float2* to) {
#pragma unroll
        for (int k = 0; k < ANGLES; ++k) {
            const int i = tid + k * kBlock;
            if (i >= angles) break;
            const double t = double(position[k]) * freq[k], part = t - rint(t);
            // Of a turn: as an FP32 number, and what that lacks, by which the sine and cosine turn on.
            const float f = float(part), less = float(part - double(f)) * 6.28318530717958648f;
            float s, c;
            sincospif(2.0f * f, &s, &c);
            to[i] = make_float2(fmaf(-less, s, c), fmaf(less, c, s));
        }
    };
    const auto fetch_first = [&](uint64_t row, Vector<T>& at) {
        Raw r{};
        if (any && row < a.rows) {
            at = vector_at<T, BACK>(a, row, start);
            if (there) r = fetch<T, BACK, PAIRS>(a, at, col);
        }
        return r;
    };
    for (int i = tid; i < 2 * a.dim; i += kBlock) {
        const float* const from = a.norm ? a.gamma[i >= a.dim] : nullptr;
        gamma[i] = from ? from[i >= a.dim ? i - a.dim : i] : 1.0f;
    }
    Vector<T> now{};
    Raw raw = fetch_first(first + uint64_t(mine), now);
    if (a.half) {
        load_positions(first);
#pragma unroll
        for (int k = 0; k < ANGLES; ++k) {
            const int i = tid + k * kBlock;
            freq[k] = i < angles ? a.freq[i % a.half] * 0.15915494309189533577 : 0.0;  // 1 / (2 pi)
        }
        form_angles(turn);
        load_positions(first + stride);
    } else {
        __syncthreads();
    }
    Chunk<T> sum[2];
#pragma unroll
    for (int j = 0; j < N; ++j) sum[0].x[j] = sum[1].x[j] = 0.0f;
    for (int buffer = 0; first < a.rows; first += stride, buffer ^= 1) {
        if (a.half) {
            __syncthreads();
            if (first + stride < a.rows) {
                form_angles(turn + (buffer ^ 1) * angles);
                load_positions(first + 2 * stride);
            }
        }
        const uint64_t row = first + uint64_t(mine);
        if (row >= a.rows || !any) continue;
        Factors<T> f;
        int held = -1;  // whose factors f are
        for (int v = start; v < vectors; v += a.gpt) {
            Vector<T> next = now;
            Raw ahead{};
            if (v + a.gpt < vectors) {
                if ((v + a.gpt >= a.heads) == (v >= a.heads)) {
                    next.x += step;
                    next.n += step;
                    next.to += step;
                } else {
                    next = vector_at<T, BACK>(a, row, v + a.gpt);
                }
                if (there) ahead = fetch<T, BACK, PAIRS>(a, next, col);
            } else {
                ahead = fetch_first(row + stride, next);
            }
            if (held != now.which && there) {
                load_factors<T, BACK, PAIRS>(a, gamma + now.which * a.dim, turn + buffer * angles + mine * a.half, col, f);
                held = now.which;
            }
            Chunk<T> own = widen<T>(raw.own), other{}, out;
            if (there) other = partners<T, PAIRS>(a, now, own, raw.other, col);
            float r = 1.0f, up = 1.0f;
            Chunk<T> in = BACK ? widen<T>(raw.n) : own;
            if (a.norm) {
                const auto mean_square = [&](float eps) {
                    float sq = 0.0f;
#pragma unroll
                    for (int j = 0; j < N; ++j) sq = fmaf(in.x[j], in.x[j], sq);
                    return fmaf(group_sum<TPV>(sq), per, eps);
                };
                float mean = mean_square(a.eps);
                if (!(mean >= kLeastSquare && mean <= kMostSquare)) {  // (all lanes of the vector)
                    up = mean < 1.0f ? kEnlarge : kReduce;
#pragma unroll
                    for (int j = 0; j < N; ++j) {
                        in.x[j] *= up;
                        if (!BACK) {
                            own.x[j] *= up;
                            other.x[j] *= up;
                        }
                    }
                    mean = mean_square(a.eps * up * up);
                }
                r = inverse_root(mean);
            }
#pragma unroll
            for (int j = 0; j < N; ++j) {
                out.x[j] = fmaf(own.x[j], f.own.x[j], other.x[j] * f.other.x[j]);  // backward: dt
                if (!BACK) out.x[j] *= r;
            }
            if constexpr (BACK) {
                if (a.norm) {
                    float dot = 0.0f;
                    Chunk<T> n;
#pragma unroll
                    for (int j = 0; j < N; ++j) {
                        n.x[j] = in.x[j] * r;
                        const float add = there ? out.x[j] * n.x[j] : 0.0f;
                        sum[0].x[j] += now.which ? 0.0f : add;
                        sum[1].x[j] += now.which ? add : 0.0f;
                        out.x[j] = there ? out.x[j] * f.gamma.x[j] : 0.0f;
                        dot = fmaf(out.x[j], n.x[j], dot);
                    }
                    dot = group_sum<TPV>(dot) * per;
#pragma unroll
                    for (int j = 0; j < N; ++j) out.x[j] = r * fmaf(-n.x[j], dot, out.x[j]);
                    if (up != 1.0f) {
#pragma unroll
                        for (int j = 0; j < N; ++j) out.x[j] *= up;
                    }
                }
            }
            if (there) store_chunk(now.to + col, out);
            now = next;
            raw = ahead;
        }
    }
    if constexpr (BACK) {
        if (!a.part) return;
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            __syncthreads();
#pragma unroll
            for (int j = 0; j < N; ++j) lds[tid * N + j] = sum[which].x[j];  // [group][TPV * N]
            __syncthreads();
            for (int i = tid; i < a.dim; i += kBlock) {
                float total = 0.0f;
                for (int k = 0; k < G; ++k) total += lds[k * TPV * N + i];
                a.part[(uint64_t(blockIdx.x) * 2 + uint64_t(which)) * uint64_t(a.dim) + uint64_t(i)] = total;
            }
        }
    }
}

// Lanes a vector, a power of two.
int lanes(int dim, bool bf16) {
    int n = 1;
    while (n * (bf16 ? 8 : 4) < dim) n *= 2;
    return n;
}
struct RotateShape {
    int gpt;
    uint32_t blocks;
};
// Groups a row: as few as leave a unit four blocks, since a row's angles are read by each of its groups.
RotateShape rotate_shape(uint64_t rows, int vectors, int dim, bool bf16, int cus, bool back) {
    const int groups = kBlock / lanes(dim, bf16);
    int gpt = 1;
    while (gpt < groups && gpt < vectors && ((rows * uint64_t(gpt) + uint64_t(groups) - 1) / uint64_t(groups) < uint64_t(4 * cus) || gpt * 8 < vectors)) gpt *= 2;
    const uint64_t at_once = uint64_t(groups / gpt), blocks = std::max<uint64_t>(1, (rows + at_once - 1) / at_once);
    return {gpt, uint32_t(std::min<uint64_t>(blocks, uint64_t(back ? 3 : 4) * uint64_t(cus)))};
}

template <class T, bool BACK, int PAIRS>
hipError_t launch_pairs(RotateArgs a, int cus, hipStream_t st) {
    const int tpv = lanes(a.dim, sizeof(T) == 2);
    const RotateShape sh = rotate_shape(a.rows, a.heads + a.kv_heads, a.dim, sizeof(T) == 2, cus, BACK);
    a.gpt = sh.gpt;
    const size_t turns = size_t(a.dim) * 8 + 2 * size_t(kBlock / tpv / sh.gpt) * size_t(a.half) * 8, sums = BACK && a.part ? size_t(kBlock) * Chunk<T>::N * 4 : 0;
    const size_t bytes = std::max(turns, sums);
    const auto as = [&](auto n) {
        if (tpv == n) k_rotate<T, decltype(n)::value, BACK, PAIRS><<<sh.blocks, kBlock, bytes, st>>>(a);
    };
    as(std::integral_constant<int, 2>{});
    as(std::integral_constant<int, 4>{});
    as(std::integral_constant<int, 8>{});
    as(std::integral_constant<int, 16>{});
    as(std::integral_constant<int, 32>{});
    if constexpr (sizeof(T) == 2) as(std::integral_constant<int, 1>{});
    else as(std::integral_constant<int, 64>{});
    return hipGetLastError();
}
template <class T, bool BACK>
hipError_t launch(const RotateArgs& a, int cus, hipStream_t st) {
    constexpr int N = Chunk<T>::N;
    if (!a.half || (a.neighbours && 2 * a.half % N == 0)) return launch_pairs<T, BACK, kSame>(a, cus, st);
    return !a.neighbours && a.half % N == 0 ? launch_pairs<T, BACK, kChunk>(a, cus, st) : launch_pairs<T, BACK, kAny>(a, cus, st);
}

}  // namespace
}  // namespace gatgpu

namespace {

using namespace gatgpu;

int check_rows(gatgpu_ctx* c, const gatgpu_rotate_io* io, const char* name, const void* p, uint64_t stride, int heads) {
    if (!p) return fail(c, GATGPU_EINVAL, std::string("null ") + name);
    const uint64_t size = io->precision == GATGPU_BF16 ? 2 : 4;
    if (stride < uint64_t(heads) * uint64_t(io->dim) || stride > (uint64_t(1) << 44)) return fail(c, GATGPU_EINVAL, std::string(name) + " has a bad row stride");
    if (reinterpret_cast<uintptr_t>(p) % 16 || stride * size % 16) return fail(c, GATGPU_EINVAL, std::string(name) + " and its stride must be 16-byte aligned");
    return check_device_array(c, p, name);
}
int check_array(gatgpu_ctx* c, const char* name, const void* p, uintptr_t size) {
    if (!p) return fail(c, GATGPU_EINVAL, std::string("null ") + name);
    if (reinterpret_cast<uintptr_t>(p) % size) return fail(c, GATGPU_EINVAL, std::string(name) + " is not aligned to its elements");
    return check_device_array(c, p, name);
}
int check_shape(gatgpu_ctx* c, const gatgpu_rotate_io* io) {
    if (!io) return fail(c, GATGPU_EINVAL, "null arrays");
    if (io->precision != GATGPU_FP32 && io->precision != GATGPU_BF16) return fail(c, GATGPU_EINVAL, "bad precision");
    if (io->heads < 1 || io->heads > 1024 || io->kv_heads < 0 || io->kv_heads > 1024) return fail(c, GATGPU_EINVAL, "heads must be 1 to 1024, kv_heads 0 to 1024");
    if (io->dim < 8 || io->dim > 256 || io->dim % 8) return fail(c, GATGPU_EINVAL, "dim must be a multiple of 8, at most 256");
    if (io->rot < 0 || io->rot > io->dim || io->rot % 2) return fail(c, GATGPU_EINVAL, "rot must be even, 0 to dim");
    if (io->pairs != GATGPU_PAIRS_HALVES && io->pairs != GATGPU_PAIRS_NEIGHBOURS) return fail(c, GATGPU_EINVAL, "bad pairs");
    if (!(io->eps >= 0.0f) || !std::isfinite(io->eps)) return fail(c, GATGPU_EINVAL, "eps must be finite and not negative");
    if (io->rows >= (uint64_t(1) << 31)) return fail(c, GATGPU_EOVERFLOW, "more than 2^31 - 1 rows");
    return GATGPU_OK;
}
// What both directions read.
int check_inputs(gatgpu_ctx* c, const gatgpu_rotate_io* io) {
    if (io->norm) {
        if (io->gamma_q)
            if (int r = check_array(c, "gamma_q", io->gamma_q, 4)) return r;
        if (io->gamma_k)
            if (int r = check_array(c, "gamma_k", io->gamma_k, 4)) return r;
    }
    if (!io->rows) return GATGPU_OK;
    if (io->rot) {
        if (int r = check_array(c, "position", io->position, 4)) return r;
        if (int r = check_array(c, "freq", io->freq, 8)) return r;
    }
    return GATGPU_OK;
}
RotateArgs make_args(const gatgpu_rotate_io* io) {
    RotateArgs a;
    a.rows = io->rows;
    a.heads = io->heads;
    a.kv_heads = io->kv_heads;
    a.dim = io->dim;
    a.norm = io->norm != 0;
    a.half = io->rot / 2;
    a.neighbours = io->pairs == GATGPU_PAIRS_NEIGHBOURS;
    a.eps = io->eps;
    a.x[0] = io->q;
    a.x[1] = io->k;
    a.xs[0] = io->q_stride;
    a.xs[1] = io->k_stride;
    a.gamma[0] = io->gamma_q;
    a.gamma[1] = io->gamma_k;
    a.position = io->position;
    a.freq = io->freq;
    return a;
}
uint64_t backward_bytes(const gatgpu_ctx* c, const gatgpu_rotate_io* io) {
    const RotateShape sh = rotate_shape(io->rows, io->heads + io->kv_heads, io->dim, io->precision == GATGPU_BF16, c->cus, true);
    return uint64_t(sh.blocks) * 2 * uint64_t(io->dim) * 4;
}

}  // namespace

extern "C" {

int gatgpu_rotate_forward(gatgpu_ctx* c, const gatgpu_rotate_io* io) {
    if (!c) return fail(nullptr, GATGPU_EINVAL, "null context");
    DeviceGuard on(c->device);
    if (!on.ok) return fail(c, GATGPU_EDEVICE, "cannot select the context's device");
    if (int r = check_shape(c, io)) return r;
    if (int r = check_inputs(c, io)) return r;
    if (!io->rows) return GATGPU_OK;
    if (int r = check_rows(c, io, "q", io->q, io->q_stride, io->heads)) return r;
    if (int r = check_rows(c, io, "q_out", io->q_out, io->q_out_stride, io->heads)) return r;
    if (io->kv_heads) {
        if (int r = check_rows(c, io, "k", io->k, io->k_stride, io->kv_heads)) return r;
        if (int r = check_rows(c, io, "k_out", io->k_out, io->k_out_stride, io->kv_heads)) return r;
    }
    RotateArgs a = make_args(io);
    a.y[0] = io->q_out;
    a.y[1] = io->k_out;
    a.ys[0] = io->q_out_stride;
    a.ys[1] = io->k_out_stride;
    HIPCHECK(c, (io->precision == GATGPU_BF16 ? launch<uint16_t, false> : launch<float, false>)(a, c->cus, c->stream));
    return GATGPU_OK;
}

int gatgpu_rotate_workspace(gatgpu_ctx* c, const gatgpu_rotate_io* io, uint64_t* bytes) {
    if (!c) return fail(nullptr, GATGPU_EINVAL, "null context");
    if (!bytes) return fail(c, GATGPU_EINVAL, "null output");
    if (int r = check_shape(c, io)) return r;
    *bytes = backward_bytes(c, io);
    return GATGPU_OK;
}

int gatgpu_rotate_backward(gatgpu_ctx* c, const gatgpu_rotate_io* io, void* ws, uint64_t bytes) {
    if (!c) return fail(nullptr, GATGPU_EINVAL, "null context");
    DeviceGuard on(c->device);
    if (!on.ok) return fail(c, GATGPU_EDEVICE, "cannot select the context's device");
    if (int r = check_shape(c, io)) return r;
    if (int r = check_inputs(c, io)) return r;
    RotateArgs a = make_args(io);
    if (io->rows) {
        const auto three = [&](const char* x, const void* px, uint64_t sx, const char* y, const void* py, uint64_t sy, const char* d, const void* pd, uint64_t sd, int heads) {
            if (io->norm)
                if (int r = check_rows(c, io, x, px, sx, heads)) return r;
            if (int r = check_rows(c, io, y, py, sy, heads)) return r;
            return check_rows(c, io, d, pd, sd, heads);
        };
        if (int r = three("q", io->q, io->q_stride, "dq_out", io->dq_out, io->dq_out_stride, "dq", io->dq, io->dq_stride, io->heads)) return r;
        if (io->kv_heads)
            if (int r = three("k", io->k, io->k_stride, "dk_out", io->dk_out, io->dk_out_stride, "dk", io->dk, io->dk_stride, io->kv_heads)) return r;
    }
    a.dy[0] = io->dq_out;
    a.dy[1] = io->dk_out;
    a.dys[0] = io->dq_out_stride;
    a.dys[1] = io->dk_out_stride;
    a.y[0] = io->dq;
    a.y[1] = io->dk;
    a.ys[0] = io->dq_stride;
    a.ys[1] = io->dk_stride;
    if (io->dgamma_q || io->dgamma_k) {
        if (!io->norm) return fail(c, GATGPU_EINVAL, "dgamma without a norm");
        if (io->dgamma_q)
            if (int r = check_array(c, "dgamma_q", io->dgamma_q, 4)) return r;
        if (io->dgamma_k)
            if (int r = check_array(c, "dgamma_k", io->dgamma_k, 4)) return r;
        const uint64_t need = backward_bytes(c, io);
        if (bytes < need) return fail(c, GATGPU_EINVAL, "workspace of " + std::to_string(bytes) + " bytes, " + std::to_string(need) + " needed");
        if (!ws || reinterpret_cast<uintptr_t>(ws) % 16) return fail(c, GATGPU_EINVAL, "workspace must be 16-byte aligned device memory");
        if (int r = check_device_array(c, ws, "workspace")) return r;
        a.part = static_cast<float*>(ws);
    }
    if (!io->rows && !a.part) return GATGPU_OK;
    if (!io->rows) a.half = 0;  // (zeros to dgamma: no positions, which may be null)
    HIPCHECK(c, (io->precision == GATGPU_BF16 ? launch<uint16_t, true> : launch<float, true>)(a, c->cus, c->stream));
    if (a.part) {
        const uint32_t blocks = uint32_t(backward_bytes(c, io) / (2 * uint64_t(io->dim) * 4));
        HIPCHECK(c, launch_column_sums(a.part, blocks, uint32_t(io->dim), io->dgamma_q, io->dgamma_k, c->stream));
    }
    return GATGPU_OK;
}

}  // extern "C"
