// The dense layer with its activation and residual, forward and backward, around the products of sgemm.hip.
// The reference spells the layer as separate operations (nnet/source/dopt/nnet/layers/dense.d:107,143, layers/relu.d).
//
//     pre = x w^T + bias,  y = act(pre) + residual
//     dz = dy act'(pre),  dx = dz w,  dw = dz^T x,  dbias = column sums of dz;  the residual's gradient is dy
#include <type_traits>

#include "activation.h"
#include "common.h"

namespace {

using namespace dopt;

constexpr int kBlock = 256;

unsigned flat_grid(size_t n)
{
    const size_t blocks = ceil_div(n, (size_t)kBlock), cap = (size_t)num_cus() * 16;
    return (unsigned)(blocks < cap ? blocks : cap);
}

// y holds the product.
template <int kAct>
__global__ __launch_bounds__(kBlock) void dense_epilogue_k(size_t n, size_t N, const float *bias, const float *residual, float *y, float *pre)
{
    for (size_t i = (size_t)blockIdx.x * kBlock + threadIdx.x; i < n; i += (size_t)gridDim.x * kBlock) {
        const float z = bias ? y[i] + bias[i % N] : y[i];
        if (pre) pre[i] = z;
        const float v = act_value<kAct>(z);
        y[i] = residual ? v + residual[i] : v;
    }
}

template <int kAct>
__global__ __launch_bounds__(kBlock) void dense_dz_k(size_t n, const float *dy, const float *pre, float *dz)
{
    for (size_t i = (size_t)blockIdx.x * kBlock + threadIdx.x; i < n; i += (size_t)gridDim.x * kBlock) dz[i] = act_grad<kAct>(dy[i], pre[i]);
}

__global__ __launch_bounds__(kBlock) void dense_columns_k(size_t M, size_t N, const float *dz, float *dbias)
{
    const size_t c = (size_t)blockIdx.x * kBlock + threadIdx.x;
    if (c >= N) return;
    float s = 0.0f;
    for (size_t m = 0; m < M; m++) s += dz[m * N + c];
    dbias[c] = s;
}

int check(const char *who, size_t M, size_t N, size_t K, int act)
{
    DOPT_REQUIRE(known_activation(act), "%s: there is no activation %d", who, act);
    DOPT_REQUIRE(M < ((size_t)1 << 30) && N < ((size_t)1 << 30) && K < ((size_t)1 << 30) && M * N < ((size_t)1 << 40) &&
                     M * K < ((size_t)1 << 40) && N * K < ((size_t)1 << 40),
                 "%s: dimensions too large", who);
    return DOPT_HIP_OK;
}

}  // namespace

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
    if (int rc = dopt_hip_sgemm_t(0, 1, M, N, K, x, w, y)) return rc;
    return with_activation(act, [&](auto a) -> int {
        hipLaunchKernelGGL(dense_epilogue_k<a.value>, dim3(flat_grid(M * N)), dim3(kBlock), 0, stream(), M * N, N, bias, residual, y, pre);
        DOPT_LAUNCH_CHECK();
        return DOPT_HIP_OK;
    });
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
    const float *dz = dy;
    if (act != DOPT_HIP_ACT_NONE && M * N > 0) {
        // dz and what the products park beside it share one request, which none of them has to grow
        const size_t own = ceil_div(M * N * sizeof(float), (size_t)256) * 256;
        const size_t more = std::max(dx ? product_scratch(0, 0, M, K, N) : 0, dw ? product_scratch(1, 0, N, K, M) : 0);
        float *const to = (float *)workspace(own + more);
        if (!to) return DOPT_HIP_ERR_OOM;
        with_activation(act, [&](auto a) {
            hipLaunchKernelGGL(dense_dz_k<a.value>, dim3(flat_grid(M * N)), dim3(kBlock), 0, stream(), M * N, dy, pre, to);
        });
        DOPT_LAUNCH_CHECK();
        workspace_hold(own);
        dz = to;
    }
    int rc = DOPT_HIP_OK;
    if (dx && M * K > 0) rc = dopt_hip_sgemm_t(0, 0, M, K, N, dz, w, dx);
    if (!rc && dw && N * K > 0) rc = dopt_hip_sgemm_t(1, 0, N, K, M, dz, x, dw);
    workspace_hold(0);
    if (rc) return rc;
    if (dbias && N > 0) {
        hipLaunchKernelGGL(dense_columns_k, dim3((unsigned)ceil_div(N, (size_t)kBlock)), dim3(kBlock), 0, stream(), M, N, dz, dbias);
        DOPT_LAUNCH_CHECK();
    }
    return DOPT_HIP_OK;
}

}  // extern "C"
