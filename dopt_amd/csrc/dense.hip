// The dense layer with its activation and residual, forward and backward, around the products of sgemm.hip.
// The reference spells the layer as separate operations (nnet/source/dopt/nnet/layers/dense.d:107,143, layers/relu.d).
//
//     pre = x w^T + bias,  y = act(pre) + residual
//     dz = dy act'(pre),  dx = dz w,  dw = dz^T x,  dbias = column sums of dz;  the residual's gradient is dy
//
// The products are those of sgemm.hip for small sizes - one row of 4096 from 4096, 67 MB of w, takes 13.2 us (5.1 TB/s), [256 x 512]
// from 784 steps 7.1 us, two thirds of that a launch - and those of dense_wide.hip for others.  Both end with bias, activation and residual
// in the wavefronts that hold the sums, but for the largest tile of sgemm.hip and for sums in parts, where a pass over them does.
#include <algorithm>
#include <type_traits>

#include "common.h"
#include "dense.h"

namespace {

using namespace dopt;

constexpr int kBlock = 256;

unsigned flat_grid(size_t n)
{
    const size_t blocks = ceil_div(n, (size_t)kBlock), cap = (size_t)num_cus() * 16;
    return (unsigned)(blocks < cap ? blocks : cap);
}

// y holds the product.  V values at a time of a row whose length is a multiple of V.
template <int V>
__global__ __launch_bounds__(kBlock) void dense_epilogue_k(size_t n, DenseEpilogue e, float *y)
{
    typedef float vec __attribute__((ext_vector_type(V), aligned(4)));
    with_activation(e.act, [&](auto kind) {
        for (size_t i = ((size_t)blockIdx.x * kBlock + threadIdx.x) * V; i < n; i += (size_t)gridDim.x * kBlock * V) {
            vec z = *(const vec *)(y + i), o;
            if (e.bias) z += *(const vec *)(e.bias + i % e.N);
            if (e.pre) *(vec *)(e.pre + i) = z;
#pragma unroll
            for (int k = 0; k < V; k++) ((float *)&o)[k] = act_value<kind.value>(((float *)&z)[k]);
            if (e.residual) o += *(const vec *)(e.residual + i);
            *(vec *)(y + i) = o;
        }
    });
}

// dz = dy act'(pre), where there is an activation, and its sums over runs of rows: a workgroup takes 64 V columns by four rows at a time.  The
// last V columns end with the matrix, whatever of them other lanes form as well, to the same bits.  Likewise the largest magnitudes of
// the runs, and, behind them, those of matrices that wait for nothing here.
// Bound by memory: [2066 x 4431], 110 MB, took 29 us by single columns and, with the magnitudes of w and x, 27 by four; [1000 x 1777] with
// them, 34 MB, takes 8.8 us, where a launch of their own took 7.  The sums cost no pass.
template <int V>
__global__ __launch_bounds__(kBlock) void dense_dz_k(size_t M, size_t N, int runs, int act, const float *dy, const float *pre, float *dz, float *sums,
                                                     unsigned *tops, Tops others)
{
    typedef float vec __attribute__((ext_vector_type(V), aligned(4)));
    __shared__ float red[4][64 * V];
    const size_t tiles = (N + 64 * V - 1) / (64 * V), run = blockIdx.x / tiles, first = blockIdx.x % tiles * 64 * V;
    if (run >= (size_t)runs) {
        column_tops(others, (unsigned)(blockIdx.x - tiles * runs));
        return;
    }
    const size_t col = min(first + (threadIdx.x & 63) * V, N - V);
    const size_t from = M * run / runs, to = M * (run + 1) / runs;
    const int row = threadIdx.x >> 6;
    float s[V], all[V];
    unsigned top[V];
#pragma unroll
    for (int e = 0; e < V; e++) {
        s[e] = all[e] = 0.0f;
        top[e] = 0;
    }
    with_activation(act, [&](auto kind) {
        constexpr bool kPlain = decltype(kind)::value == DOPT_HIP_ACT_NONE;
        auto one = [&](const float *d, const float *z, size_t at) {
            float o[V];
#pragma unroll
            for (int e = 0; e < V; e++) {
                o[e] = act_grad<kind.value>(d[e], z[e]);
                s[e] += o[e];
                top[e] = max(top[e], magnitude(o[e]));
                if (!kPlain) dz[at + e] = o[e];
            }
        };
        size_t m = from + row;
        for (; m + 12 < to; m += 16) {
            if (((m - from) & 255) < 4) {   // sums of 64 values each: 1024 equal ones in a row are rounded the same way to 1.5e-5 of their sum
#pragma unroll
                for (int e = 0; e < V; e++) {
                    all[e] += s[e];
                    s[e] = 0.0f;
                }
            }
            vec d[4], z[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                d[i] = *(const vec *)(dy + (m + 4 * i) * N + col);
                if (!kPlain) z[i] = *(const vec *)(pre + (m + 4 * i) * N + col);
            }
#pragma unroll
            for (int i = 0; i < 4; i++) one((const float *)&d[i], kPlain ? (const float *)&d[i] : (const float *)&z[i], (m + 4 * i) * N + col);
        }
        for (; m < to; m += 4) {
            const vec d = *(const vec *)(dy + m * N + col), z = kPlain ? d : *(const vec *)(pre + m * N + col);
            one((const float *)&d, (const float *)&z, m * N + col);
        }
    });
    auto place = [&](size_t c) { return run * N + min(first + c / V * V, N - V) + c % V; };
    if (sums) {
#pragma unroll
        for (int e = 0; e < V; e++) red[row][(threadIdx.x & 63) * V + e] = all[e] + s[e];
        __syncthreads();
        for (size_t c = threadIdx.x; c < 64 * V; c += kBlock) sums[place(c)] = (red[0][c] + red[1][c]) + (red[2][c] + red[3][c]);
    }
    if (!tops) return;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < V; e++) red[row][(threadIdx.x & 63) * V + e] = __builtin_bit_cast(float, top[e]);
    __syncthreads();
    for (size_t c = threadIdx.x; c < 64 * V; c += kBlock)
        tops[place(c)] = max(max(magnitude(red[0][c]), magnitude(red[1][c])), max(magnitude(red[2][c]), magnitude(red[3][c])));
}

__global__ __launch_bounds__(kBlock) void dense_fold_k(DenseFold f) { dense_fold(f, (size_t)blockIdx.y * kLaunchBlocks + blockIdx.x); }

int check(const char *who, size_t M, size_t N, size_t K, int act)
{
    DOPT_REQUIRE(known_activation(act), "%s: there is no activation %d", who, act);
    DOPT_REQUIRE(M < ((size_t)1 << 30) && N < ((size_t)1 << 30) && K < ((size_t)1 << 30) && M * N < ((size_t)1 << 40) &&
                     M * K < ((size_t)1 << 40) && N * K < ((size_t)1 << 40),
                 "%s: dimensions too large", who);
    return DOPT_HIP_OK;
}

}  // namespace

namespace dopt {

int dense_finish(size_t M, size_t N, const DenseEpilogue &e, float *y)
{
    if (N % 4 == 0) hipLaunchKernelGGL(dense_epilogue_k<4>, dim3(flat_grid(M * N / 4)), dim3(kBlock), 0, stream(), M * N, e, y);
    else hipLaunchKernelGGL(dense_epilogue_k<1>, dim3(flat_grid(M * N)), dim3(kBlock), 0, stream(), M * N, e, y);
    DOPT_LAUNCH_CHECK();
    return DOPT_HIP_OK;
}

}  // namespace dopt

extern "C" {

int dopt_hip_dense_act(size_t M, size_t N, size_t K, int act, const float *x, const float *w, const float *bias, const float *residual,
                       float *y, float *pre)
{
    if (int rc = check("dopt_hip_dense_act", M, N, K, act)) return rc;
    if (M * N == 0) return DOPT_HIP_OK;
    DOPT_REQUIRE(y && (K == 0 || (x && w)), "dopt_hip_dense_act: null argument");
    const size_t f = sizeof(float), out = M * N * f;
    for (const float *o : {y, pre})
        DOPT_REQUIRE(!overlaps(o, out, x, M * K * f) && !overlaps(o, out, w, N * K * f) && !overlaps(o, out, bias, N * f) && !overlaps(o, out, residual, out),
                     "dopt_hip_dense_act: a result overlaps an operand");
    DOPT_REQUIRE(!overlaps(y, out, pre, out), "dopt_hip_dense_act: y and pre overlap");
    const DenseEpilogue e{bias, residual, pre, act, N};
    if (dense_wide_takes(M, N, K)) {
        const WideProduct p{M, N, K, {x, false}, {w, false}, y};
        return dense_wide(&p, 1, e, DenseFold{}, false);
    }
    return product_dense(M, N, K, x, w, e, y);
}

int dopt_hip_dense_act_grad(size_t M, size_t N, size_t K, int act, const float *dy, const float *pre, const float *x, const float *w,
                            float *dx, float *dw, float *dbias)
{
    if (int rc = check("dopt_hip_dense_act_grad", M, N, K, act)) return rc;
    DOPT_REQUIRE(M * N == 0 || (dy && (act == DOPT_HIP_ACT_NONE || pre)), "dopt_hip_dense_act_grad: null argument");
    DOPT_REQUIRE(M * K == 0 || !dx || N == 0 || w, "dopt_hip_dense_act_grad: the gradient of x needs w");
    DOPT_REQUIRE(N * K == 0 || !dw || M == 0 || x, "dopt_hip_dense_act_grad: the gradient of w needs x");
    const size_t f = sizeof(float), sizes[] = {M * K * f, N * K * f, N * f};
    const float *const results[] = {dx, dw, dbias};
    for (int i = 0; i < 3; i++) {
        DOPT_REQUIRE(!overlaps(results[i], sizes[i], dy, M * N * f) && !overlaps(results[i], sizes[i], pre, M * N * f) &&
                         !overlaps(results[i], sizes[i], x, M * K * f) && !overlaps(results[i], sizes[i], w, N * K * f),
                     "dopt_hip_dense_act_grad: a result overlaps an operand");
        for (int j = 0; j < i; j++) DOPT_REQUIRE(!overlaps(results[i], sizes[i], results[j], sizes[j]), "dopt_hip_dense_act_grad: two results overlap");
    }
    DOPT_ENSURE_INIT();
    const bool plain = act == DOPT_HIP_ACT_NONE;
    const float *dz = dy;
    float *sums = nullptr;
    const int V = N >= 4 ? 4 : 1;
    const size_t tiles = ceil_div(std::max(N, (size_t)1), (size_t)(64 * V));
    // Enough workgroups to fill the chip, of sixteen rows and more; no more than 64 runs where every tile of dz' layout reads their largest
    // magnitudes ([2066 x 462] from 4431 and its like in 114 runs 147 us, in 64 or 32 of them 136).
    const bool turns = dw && dense_wide_takes(N, K, M);
    const size_t most = turns ? std::min((size_t)64, ceil_div(M, (size_t)16)) : ceil_div(M, (size_t)16);
    const int runs = (int)std::max((size_t)1, std::min(most, ceil_div((size_t)num_cus() * 8, tiles)));
    // the products that dense_wide.hip takes, in its launches
    WideProduct wide[2];
    int wides = 0;
    if (dx && dense_wide_takes(M, K, N)) wide[wides++] = WideProduct{M, K, N, {dz, false}, {w, true}, dx};
    const bool wide_x = wides > 0;
    const bool pass = M * N > 0 && (!plain || dbias);   // over dz, which then finds what the products need of it
    if (turns) wide[wides++] = WideProduct{N, K, M, {dz, true, pass ? runs : 0}, {x, true}, dw};
    const bool wide_w = wides > (int)wide_x;
    size_t held = 0;
    if (pass) {
        // dz, its sums and what the products park beside them share one request, which none of them has to grow
        auto rounded = [](size_t bytes) { return ceil_div(bytes, (size_t)256) * 256; };
        const size_t first = plain ? 0 : rounded(M * N * sizeof(float));
        held = first + rounded((size_t)runs * N * sizeof(float));
        const size_t more = std::max({dense_wide_scratch(wide, wides), !dx || wide_x ? 0 : product_scratch(0, 0, M, K, N),
                                      !dw || wide_w ? 0 : product_scratch(1, 0, N, K, M)});
        char *const to = (char *)workspace(held + more);
        if (!to) return DOPT_HIP_ERR_OOM;
        if (!plain) dz = (float *)to;
        sums = (float *)(to + first);
        for (int i = 0; i < wides; i++) wide[i].x.values = dz;
        Tops others{};
        unsigned *const tops = wides ? dense_wide_tops(wide, wides, to + held, &others) : nullptr;
        const dim3 grid((unsigned)(tiles * runs) + others.blocks);
        if (V == 4)
            hipLaunchKernelGGL(dense_dz_k<4>, grid, dim3(kBlock), 0, stream(), M, N, runs, act, dy, pre, (float *)to, dbias ? sums : nullptr, tops, others);
        else
            hipLaunchKernelGGL(dense_dz_k<1>, grid, dim3(kBlock), 0, stream(), M, N, runs, act, dy, pre, (float *)to, dbias ? sums : nullptr, tops, others);
        DOPT_LAUNCH_CHECK();
    }
    const DenseFold fold{sums ? (size_t)runs : 0, N, sums, N > 0 ? dbias : nullptr};
    if (fold.dbias && !wides) {
        const size_t blocks = ceil_div(N, (size_t)8);
        hipLaunchKernelGGL(dense_fold_k, dim3((unsigned)std::min(blocks, kLaunchBlocks), (unsigned)ceil_div(blocks, kLaunchBlocks)), dim3(kBlock), 0, stream(),
                           fold);
        DOPT_LAUNCH_CHECK();
    }
    workspace_hold(held);
    int rc = DOPT_HIP_OK;
    if (wides) rc = dense_wide(wide, wides, DenseEpilogue{nullptr, nullptr, nullptr, DOPT_HIP_ACT_NONE, K}, fold, pass);
    if (!rc && dx && !wide_x && M * K > 0) rc = dopt_hip_sgemm_t(0, 0, M, K, N, dz, w, dx);
    if (!rc && dw && !wide_w && N * K > 0) rc = dopt_hip_sgemm_t(1, 0, N, K, M, dz, x, dw);
    workspace_hold(0);
    return rc;
}

}  // extern "C"
