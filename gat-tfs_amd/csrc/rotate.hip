// Norms and rotation of queries and keys, forward and backward.
//
//   r = 1 / sqrt(mean(x^2) + eps),  n = x r,  t = n gamma          (without a norm: t = x)
//   y_i = t_i c_i + t_p s_i, p the other column of i's pair, s_i = -sin for the first of a pair, sin for the second
//   dt_i = dy_i c_i - dy_p s_i,  dgamma = sum dt n,  g = dt gamma,  dx = r (g - n mean(g n))
//
// Bound by bytes: a head's vector is read once into TPV lanes of 16 bytes each, and written once.  The other column of
// a pair half a rotation away comes by a second read of the same lines, which the first has just brought (a lane
// exchange would take one LDS permute an element).  A row's angles are formed once a block, a thread an angle, in 64
// bits: position * freq in turns, of which the whole ones go before what is left is rounded to 32 bits, so that far
// positions keep an angle's error of 2^-23.  Groups of lanes then take the row's heads in turn with their columns' sines
// in registers.  The backward pass gives each block a fixed set of rows and keeps its columns' sums for gamma in
// registers over them; blocks leave one partial row each, added in one fixed order.
#include <algorithm>
#include <cmath>
#include <string>
#include <type_traits>

#include "context.hpp"
#include "norm.hpp"

namespace gatgpu {
namespace {

constexpr int kBlock = 256;

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
__device__ inline Chunk<T> load_chunk(const T* p) {
    const uint4 w = *reinterpret_cast<const uint4*>(p);
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
template <int TPV>
__device__ inline float group_sum(float x) {
#pragma unroll
    for (int d = TPV / 2; d; d /= 2) x += __shfl_xor(x, d);
    return x;
}

// The other columns of a chunk's pairs.
template <class T>
__device__ inline Chunk<T> load_partners(const RotateArgs& a, const T* row, int col, const Chunk<T>& own) {
    constexpr int N = Chunk<T>::N;
    Chunk<T> p = own;
    if (!a.half) return p;
    if (a.neighbours) {
#pragma unroll
        for (int j = 0; j < N; ++j) p.x[j] = own.x[j ^ 1];
    } else if (a.half % N == 0) {
        if (col < 2 * a.half) p = load_chunk(row + (col < a.half ? col + a.half : col - a.half));
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int i = col + j;
            if (i < 2 * a.half) p.x[j] = load_one(row + (i < a.half ? i + a.half : i - a.half));
        }
    }
    return p;
}
template <class T>
__device__ inline void load_gamma(const RotateArgs& a, const float* gamma, int col, bool partners, Chunk<T>& own, Chunk<T>& other) {
    constexpr int N = Chunk<T>::N;
#pragma unroll
    for (int j = 0; j < N; ++j) {
        own.x[j] = gamma ? gamma[col + j] : 1.0f;
        other.x[j] = 1.0f;
        if (partners && gamma) {
            const int i = col + j, p = a.neighbours ? i ^ 1 : i < a.half ? i + a.half : i - a.half;
            other.x[j] = i < 2 * a.half ? gamma[p] : 0.0f;
        }
    }
}

// T rows of the block's turn at a time; group g of TPV lanes takes heads g % gpt, g % gpt + gpt, ... of row g / gpt.
template <class T, int TPV, bool BACK>
__global__ __launch_bounds__(kBlock) void k_rotate(const RotateArgs a) {
    constexpr int N = Chunk<T>::N, G = kBlock / TPV;
    extern __shared__ float lds[];
    float2* const turn = reinterpret_cast<float2*>(lds);  // [rows at once][half]
    const int tid = int(threadIdx.x), g = tid / TPV, col = tid % TPV * N;
    const int at_once = G / a.gpt, vectors = a.heads + a.kv_heads;
    const bool there = col < a.dim;
    Chunk<T> sum[2];
#pragma unroll
    for (int j = 0; j < N; ++j) sum[0].x[j] = sum[1].x[j] = 0.0f;
    for (uint64_t first = uint64_t(blockIdx.x) * at_once; first < a.rows; first += uint64_t(gridDim.x) * at_once) {
        if (a.half) {
            __syncthreads();
            for (int i = tid; i < at_once * a.half; i += kBlock) {
                const uint64_t row = first + uint64_t(i / a.half);
                if (row < a.rows) {
                    const double t = double(a.position[row]) * a.freq[i % a.half] * 0.15915494309189533577;  // 1 / (2 pi)
                    float s, c;
                    sincospif(2.0f * float(t - rint(t)), &s, &c);
                    turn[i] = make_float2(c, BACK ? -s : s);
                }
            }
            __syncthreads();
        }
        const uint64_t row = first + uint64_t(g / a.gpt);
        if (row >= a.rows) continue;
        Chunk<T> c, s;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int i = col + j;
            c.x[j] = 1.0f;
            s.x[j] = 0.0f;
            if (i < 2 * a.half) {
                const bool second = a.neighbours ? i & 1 : i >= a.half;
                const float2 w = turn[g / a.gpt * a.half + (a.neighbours ? i / 2 : second ? i - a.half : i)];
                c.x[j] = w.x;
                s.x[j] = second ? w.y : -w.y;
            }
        }
        Chunk<T> own, other;
        int held = -1;  // whose gamma own and other are
        for (int v = g % a.gpt; v < vectors; v += a.gpt) {
            const int which = v >= a.heads;
            const uint64_t at = uint64_t(which ? v - a.heads : v) * uint64_t(a.dim);
            const T* const x = static_cast<const T*>(a.x[which]) + row * a.xs[which] + at;
            T* const y = static_cast<T*>(a.y[which]) + row * a.ys[which] + at;
            Chunk<T> in{}, pair{}, out{};
            if (there && (!BACK || a.norm)) in = load_chunk(x + col);
            if constexpr (BACK) {
                const T* const dy = static_cast<const T*>(a.dy[which]) + row * a.dys[which] + at;
                if (there) {
                    out = load_chunk(dy + col);
                    pair = load_partners(a, dy, col, out);
                }
            } else if (there) {
                pair = load_partners(a, x, col, in);
            }
            if (a.norm && held != which && there) {
                load_gamma(a, a.gamma[which], col, !BACK, own, other);
                held = which;
            }
            float r = 1.0f;
            if (a.norm) {
                float sq = 0.0f;
#pragma unroll
                for (int j = 0; j < N; ++j) sq = fmaf(in.x[j], in.x[j], sq);
                r = 1.0f / sqrtf(group_sum<TPV>(sq) / float(a.dim) + a.eps);
            }
            if constexpr (!BACK) {
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    float t = in.x[j], p = pair.x[j];
                    if (a.norm) {
                        t = t * r * own.x[j];
                        p = p * r * other.x[j];
                    }
                    out.x[j] = col + j < 2 * a.half ? fmaf(t, c.x[j], p * s.x[j]) : t;
                }
            } else {
#pragma unroll
                for (int j = 0; j < N; ++j)
                    if (col + j < 2 * a.half) out.x[j] = fmaf(out.x[j], c.x[j], pair.x[j] * s.x[j]);  // dt
                if (a.norm) {
                    float dot = 0.0f;
#pragma unroll
                    for (int j = 0; j < N; ++j) {
                        in.x[j] *= r;  // n
                        const float add = out.x[j] * in.x[j];
                        sum[0].x[j] += which ? 0.0f : add;
                        sum[1].x[j] += which ? add : 0.0f;
                        out.x[j] = there ? out.x[j] * own.x[j] : 0.0f;
                        dot = fmaf(out.x[j], in.x[j], dot);
                    }
                    dot = group_sum<TPV>(dot) / float(a.dim);
#pragma unroll
                    for (int j = 0; j < N; ++j) out.x[j] = r * fmaf(-in.x[j], dot, out.x[j]);
                }
            }
            if (there) store_chunk(y + col, out);
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
    return {gpt, uint32_t(std::min<uint64_t>(blocks, back ? uint64_t(4 * cus) : uint64_t(1) << 20))};
}

template <class T, bool BACK>
hipError_t launch(RotateArgs a, int cus, hipStream_t st) {
    const int tpv = lanes(a.dim, sizeof(T) == 2);
    const RotateShape sh = rotate_shape(a.rows, a.heads + a.kv_heads, a.dim, sizeof(T) == 2, cus, BACK);
    a.gpt = sh.gpt;
    const size_t turns = size_t(kBlock / tpv / sh.gpt) * size_t(a.half) * 8, sums = BACK && a.part ? size_t(kBlock) * Chunk<T>::N * 4 : 0;
    const size_t bytes = std::max(turns, sums);
    const auto as = [&](auto n) {
        if (tpv == n) k_rotate<T, decltype(n)::value, BACK><<<sh.blocks, kBlock, bytes, st>>>(a);
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
    HIPCHECK(c, (io->precision == GATGPU_BF16 ? launch<uint16_t, true> : launch<float, true>)(a, c->cus, c->stream));
    if (a.part) {
        const uint32_t blocks = uint32_t(backward_bytes(c, io) / (2 * uint64_t(io->dim) * 4));
        HIPCHECK(c, launch_column_sums(a.part, blocks, uint32_t(io->dim), io->dgamma_q, io->dgamma_k, c->stream));
    }
    return GATGPU_OK;
}

}  // extern "C"
