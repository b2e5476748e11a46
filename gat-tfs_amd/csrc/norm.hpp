// Layer norm: what its kernels and its callers share (norm.hip).
#pragma once
#include "internal.hpp"

namespace gatgpu {

struct NormArgs {
    uint64_t rows = 0;
    uint32_t width = 0;
    int elu = 0;
    float eps = 0.0f;
    const float *gamma = nullptr, *beta = nullptr;
    float *mean = nullptr, *rstd = nullptr;
    // forward: rows of x (+ residual) to y, their sum to `sum`
    const void *x = nullptr, *residual = nullptr;
    void *y = nullptr, *sum = nullptr;
    uint64_t xs = 0, rs = 0, ys = 0, ss = 0;  // row strides (elements)
    // backward: h is the normalised input (x, or the forward's sum)
    const void *h = nullptr, *dy = nullptr, *dsum = nullptr;
    void* dx = nullptr;
    uint64_t hs = 0, dys = 0, dss = 0, dxs = 0;
    float* part = nullptr;  // [blocks][2][width] partial sums of dgamma and dbeta, or null
};

// Blocks (and partial rows) of the backward pass.
uint32_t norm_blocks(uint64_t rows, uint64_t width);
hipError_t launch_norm_forward(const NormArgs& a, bool bf16, hipStream_t s);
hipError_t launch_norm_backward(const NormArgs& a, bool bf16, uint32_t blocks, float* dgamma, float* dbeta, hipStream_t s);
// a[c], b[c] (either may be null): sums over the blocks of part[block][2][width], in one fixed order.
hipError_t launch_column_sums(const float* part, uint32_t blocks, uint32_t width, float* a, float* b, hipStream_t s);

}  // namespace gatgpu
