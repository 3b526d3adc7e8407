// The end of a dense layer's product: bias, activation, residual.
#pragma once

#include "activation.h"

namespace dopt {

struct NoEpilogue {
    static constexpr bool kOn = false;
};

// y = act(z) + residual with z = product + bias[column]; z itself to `pre`.  All but y may be null.
struct DenseEpilogue {
    static constexpr bool kOn = true;
    const float *bias, *residual;
    float *pre;
    int act;
    size_t N;   // columns

    __device__ __forceinline__ float bias_of(size_t col) const { return bias ? bias[col] : 0.0f; }
    __device__ __forceinline__ float value(float z) const
    {
        return with_activation(act, [&](auto kind) { return act_value<kind.value>(z); });
    }
    __device__ __forceinline__ float operator()(float sum, size_t i) const   // value i of the result
    {
        const float z = sum + bias_of(i % N);
        if (pre) pre[i] = z;
        const float y = value(z);
        return residual ? y + residual[i] : y;
    }
};

// dense.hip: the same for a product that lies in y already.
int dense_finish(size_t M, size_t N, const DenseEpilogue &e, float *y);
// Adds runs of column sums: eight columns of a workgroup of 256 by thirty-two lanes.
struct DenseFold {
    size_t runs, N;
    const float *sums;
    float *dbias;
};
__device__ __forceinline__ void dense_fold(const DenseFold &f, size_t block)
{
    __shared__ float red[32][9];
    const int col = threadIdx.x & 7, lane = threadIdx.x >> 3;
    const size_t c = block * 8 + col;
    float s = 0.0f;
    if (c < f.N) {
#pragma unroll 4
        for (size_t i = lane; i < f.runs; i += 32) s += f.sums[i * f.N + c];
    }
    red[lane][col] = s;
    __syncthreads();
    if (lane == 0 && c < f.N) {
        for (int i = 1; i < 32; i++) s += red[i][col];
        f.dbias[c] = s;
    }
}

// dense_wide.hip: x w^T for sizes that it takes; either may lie across, [K][rows].
struct WideSide {
    const float *values;
    bool across;
};
struct WideProduct {
    size_t M, N, K;
    WideSide x, w;
    float *y;
};
bool dense_wide_takes(size_t M, size_t N, size_t K);
size_t dense_wide_scratch(const WideProduct *p, int n);
// One or two of them with the same epilogue; with the fold, if its dbias is there.
int dense_wide(const WideProduct *p, int n, const DenseEpilogue &e, const DenseFold &fold);
// sgemm.hip: x w^T with that epilogue, x [M, K], w [N, K].
int product_dense(size_t M, size_t N, size_t K, const float *x, const float *w, const DenseEpilogue &e, float *y);

}  // namespace dopt
