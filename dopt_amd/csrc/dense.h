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
// dense_wide.hip: x w^T with that epilogue for large sizes; either may lie across, [K][rows].
struct WideSide {
    const float *values;
    bool across;
};
bool dense_wide_takes(size_t M, size_t N, size_t K);
size_t dense_wide_scratch(size_t M, size_t N, size_t K);
int dense_wide(size_t M, size_t N, size_t K, const WideSide &x, const WideSide &w, const DenseEpilogue &e, float *y);
// sgemm.hip: x w^T with that epilogue, x [M, K], w [N, K].
int product_dense(size_t M, size_t N, size_t K, const float *x, const float *w, const DenseEpilogue &e, float *y);

}  // namespace dopt
