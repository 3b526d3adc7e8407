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

// A value's magnitude as an integer, whose order is its, infinity and NaN last.  (By value: of an element of a vector the builtin takes
// the first one's bits.)
__device__ __forceinline__ unsigned magnitude(float v) { return __builtin_bit_cast(unsigned, v) & 0x7fffffffu; }

// The largest magnitudes of runs of the rows of matrices [K][columns], for each column.
struct Tops {
    struct One {
        const float *x;
        size_t columns, K;
        unsigned *tops;   // [run][column]
        int runs;
        unsigned blocks;
    } o[3];
    int n;
    unsigned blocks;
};
__device__ __forceinline__ void column_tops(const Tops &t, unsigned block)   // 256 threads
{
    typedef float vec __attribute__((ext_vector_type(4), aligned(4)));
    __shared__ unsigned red[4][256];
    int which = 0;
    while (which + 1 < t.n && block >= t.o[which].blocks) block -= t.o[which++].blocks;
    const Tops::One &o = t.o[which];
    const unsigned tiles = (unsigned)((o.columns + 255) / 256);
    const size_t col = min((size_t)(block % tiles) * 256 + (threadIdx.x & 63) * 4, o.columns - 4), run = block / tiles;
    const size_t from = o.K * run / o.runs, to = o.K * (run + 1) / o.runs;
    const int row = threadIdx.x >> 6;
    unsigned top[4] = {0, 0, 0, 0};
    size_t k = from + row;
    auto see = [&](vec v) {
#pragma unroll
        for (int e = 0; e < 4; e++) top[e] = max(top[e], magnitude(v[e]));
    };
    for (; k + 28 < to; k += 32) {
        vec v[8];
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = *(const vec *)(o.x + (k + 4 * i) * o.columns + col);
#pragma unroll
        for (int i = 0; i < 8; i++) see(v[i]);
    }
    for (; k < to; k += 4) see(*(const vec *)(o.x + k * o.columns + col));
#pragma unroll
    for (int e = 0; e < 4; e++) red[row][(threadIdx.x & 63) * 4 + e] = top[e];
    __syncthreads();
    if (row) return;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const int c = (threadIdx.x & 63) * 4 + e;
        o.tops[run * o.columns + col + e] = max(max(red[0][c], red[1][c]), max(red[2][c], red[3][c]));
    }
}

// dense_wide.hip: x w^T for sizes that it takes; either may lie across, [K][rows].
struct WideSide {
    const float *values;
    bool across;
    int runs = 0;   // of an operand across whose runs' largest magnitudes the caller finds: their number
};
struct WideProduct {
    size_t M, N, K;
    WideSide x, w;
    float *y;
};
bool dense_wide_takes(size_t M, size_t N, size_t K);
size_t dense_wide_scratch(const WideProduct *p, int n);
// Where in that scratch the caller's largest magnitudes belong (null without any), and what finds the others.
unsigned *dense_wide_tops(const WideProduct *p, int n, char *scratch, Tops *others);
// One or two of them with the same epilogue; with the fold, if its dbias is there.  `found`: the largest magnitudes are in their places.
int dense_wide(const WideProduct *p, int n, const DenseEpilogue &e, const DenseFold &fold, bool found);
// sgemm.hip: x w^T with that epilogue, x [M, K], w [N, K].
int product_dense(size_t M, size_t N, size_t K, const float *x, const float *w, const DenseEpilogue &e, float *y);

}  // namespace dopt
