// Group norm with an activation behind it, forward and backward, for [N, C, inner] and channels-last [N, inner, C] tensors.
// No counterpart in the reference, whose only norm is over the batch (cuda/source/dopt/cuda/nnet/cudnn7.d:547-654); the packed
// results follow its batch norm's (core/source/dopt/core/ops/nnet.d:222-235).
//
//     z = (x - mean) rstd scale[c] + bias[c],  y = act(z);  mean, biased variance of a group: C / G channels x inner values
//     dz = dy act'(z),  dbias[c] = sum dz,  dscale[c] = sum dz xhat,
//     dx = rstd (dz scale[c] - s1 - xhat s2),  s1, s2 the group's means of dz scale and dz scale xhat
#include <type_traits>

#include "activation.h"
#include "common.h"

namespace {

using namespace dopt;

constexpr int kBlock = 256;

// Where value i of a group's L lies, and of which channel it is.
struct Place {
    size_t C, inner, Cg, G;
    int last;
    __device__ size_t at(size_t n, size_t g, size_t i) const
    {
        if (!last) return (n * C + g * Cg) * inner + i;
        return (n * inner + i / Cg) * C + g * Cg + i % Cg;
    }
    __device__ size_t channel(size_t g, size_t i) const { return g * Cg + (last ? i % Cg : i / inner); }
};

// The sum over a workgroup of 256, in every thread.
__device__ float block_sum(float v, float *red)
{
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
    __syncthreads();   // the last sum has been read
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return (red[0] + red[1]) + (red[2] + red[3]);
}

// A workgroup per group.
template <int kAct>
__global__ __launch_bounds__(kBlock) void gn_fwd_k(Place p, float eps, const float *x, const float *scale, const float *bias, float *y,
                                                   float *means, float *rstds)
{
    __shared__ float red[4];
    const size_t n = blockIdx.x / p.G, g = blockIdx.x % p.G, L = p.Cg * p.inner;
    float s = 0.0f;
    for (size_t i = threadIdx.x; i < L; i += kBlock) s += x[p.at(n, g, i)];
    const float mean = L ? block_sum(s, red) / (float)L : 0.0f;
    float q = 0.0f;
    for (size_t i = threadIdx.x; i < L; i += kBlock) {
        const float d = x[p.at(n, g, i)] - mean;
        q += d * d;
    }
    const float rstd = 1.0f / sqrtf((L ? block_sum(q, red) / (float)L : 0.0f) + eps);
    for (size_t i = threadIdx.x; i < L; i += kBlock) {
        const size_t at = p.at(n, g, i), c = p.channel(g, i);
        y[at] = act_value<kAct>((x[at] - mean) * rstd * scale[c] + bias[c]);
    }
    if (threadIdx.x == 0) {
        means[blockIdx.x] = mean;
        rstds[blockIdx.x] = rstd;
    }
}

// A workgroup per sample and channel: its sums of dz and dz xhat.
template <int kAct>
__global__ __launch_bounds__(kBlock) void gn_sums_k(Place p, const float *dy, const float *x, const float *scale, const float *bias,
                                                    const float *means, const float *rstds, float2 *sums)
{
    __shared__ float red[4];
    const size_t n = blockIdx.x / p.C, c = blockIdx.x % p.C, g = c / p.Cg;
    const float mean = means[n * p.G + g], rstd = rstds[n * p.G + g], a = scale[c], b = bias[c];
    float s = 0.0f, q = 0.0f;
    for (size_t i = threadIdx.x; i < p.inner; i += kBlock) {
        const size_t at = p.last ? (n * p.inner + i) * p.C + c : (n * p.C + c) * p.inner + i;
        const float xhat = (x[at] - mean) * rstd, dz = act_grad<kAct>(dy[at], xhat * a + b);
        s += dz;
        q += dz * xhat;
    }
    s = block_sum(s, red);
    q = block_sum(q, red);
    if (threadIdx.x == 0) sums[blockIdx.x] = make_float2(s, q);
}

// A workgroup per group.
template <int kAct>
__global__ __launch_bounds__(kBlock) void gn_dx_k(Place p, const float *dy, const float *x, const float *scale, const float *bias,
                                                  const float *means, const float *rstds, const float2 *sums, float *dx)
{
    const size_t n = blockIdx.x / p.G, g = blockIdx.x % p.G, L = p.Cg * p.inner;
    const float mean = means[blockIdx.x], rstd = rstds[blockIdx.x];
    float s1 = 0.0f, s2 = 0.0f;
    for (size_t c = g * p.Cg; c < (g + 1) * p.Cg; c++) {
        const float2 v = sums[n * p.C + c];
        s1 += v.x * scale[c];
        s2 += v.y * scale[c];
    }
    s1 /= (float)L;
    s2 /= (float)L;
    for (size_t i = threadIdx.x; i < L; i += kBlock) {
        const size_t at = p.at(n, g, i), c = p.channel(g, i);
        const float xhat = (x[at] - mean) * rstd, a = scale[c];
        const float dz = act_grad<kAct>(dy[at], xhat * a + bias[c]);
        dx[at] = rstd * (dz * a - s1 - xhat * s2);
    }
}

__global__ __launch_bounds__(kBlock) void gn_fold_k(size_t N, size_t C, const float2 *sums, float *dscale, float *dbias)
{
    const size_t c = (size_t)blockIdx.x * kBlock + threadIdx.x;
    if (c >= C) return;
    float s = 0.0f, q = 0.0f;
    for (size_t n = 0; n < N; n++) {
        const float2 v = sums[n * C + c];
        s += v.x;
        q += v.y;
    }
    dbias[c] = s;
    dscale[c] = q;
}

int check(const char *who, size_t N, size_t C, size_t inner, size_t groups, int act)
{
    DOPT_REQUIRE(groups > 0 && C % groups == 0, "%s: %zu channels cannot be parted into %zu groups", who, C, groups);
    DOPT_REQUIRE(known_activation(act), "%s: there is no activation %d", who, act);
    DOPT_REQUIRE(N < ((size_t)1 << 31) && C < ((size_t)1 << 31) && inner < ((size_t)1 << 40) && N * C < ((size_t)1 << 31),
                 "%s: dimensions too large", who);
    return DOPT_HIP_OK;
}

}  // namespace

extern "C" {

int dopt_hip_group_norm(size_t N, size_t C, size_t inner, size_t groups, int channels_last, float eps, int act, const float *x,
                        const float *scale, const float *bias, float *packed)
{
    if (int rc = check("dopt_hip_group_norm", N, C, inner, groups, act)) return rc;
    const size_t total = N * C * inner;
    if (N * C == 0) return DOPT_HIP_OK;
    DOPT_REQUIRE(packed && (total == 0 || (x && scale && bias)), "dopt_hip_group_norm: null argument");
    const size_t out = (total + 2 * N * groups) * sizeof(float), per = C * sizeof(float);
    DOPT_REQUIRE(!overlaps(packed, out, x, total * sizeof(float)) && !overlaps(packed, out, scale, per) && !overlaps(packed, out, bias, per),
                 "dopt_hip_group_norm: the result overlaps an operand");
    DOPT_ENSURE_INIT();
    const Place p{C, inner, C / groups, groups, channels_last != 0};
    return with_activation(act, [&](auto a) -> int {
        hipLaunchKernelGGL(gn_fwd_k<a.value>, dim3((unsigned)(N * groups)), dim3(kBlock), 0, stream(), p, eps, x, scale, bias, packed,
                           packed + total, packed + total + N * groups);
        DOPT_LAUNCH_CHECK();
        return DOPT_HIP_OK;
    });
}

int dopt_hip_group_norm_grad(size_t N, size_t C, size_t inner, size_t groups, int channels_last, int act, const float *dy, const float *x,
                             const float *scale, const float *bias, const float *stats, float *packed)
{
    if (int rc = check("dopt_hip_group_norm_grad", N, C, inner, groups, act)) return rc;
    if (C == 0) return DOPT_HIP_OK;
    const size_t total = N * C * inner;
    DOPT_REQUIRE(packed && (total == 0 || (dy && x && scale && bias && stats)), "dopt_hip_group_norm_grad: null argument");
    const size_t out = (total + 2 * C) * sizeof(float), per = C * sizeof(float), in = total * sizeof(float);
    DOPT_REQUIRE(!overlaps(packed, out, dy, in) && !overlaps(packed, out, x, in) && !overlaps(packed, out, scale, per) &&
                     !overlaps(packed, out, bias, per) && !overlaps(packed, out, stats, 2 * N * groups * sizeof(float)),
                 "dopt_hip_group_norm_grad: the result overlaps an operand");
    DOPT_ENSURE_INIT();
    const Place p{C, inner, C / groups, groups, channels_last != 0};
    const float *means = stats, *rstds = stats + N * groups;
    float2 *sums = nullptr;
    if (total && !(sums = (float2 *)workspace(N * C * sizeof(float2)))) return DOPT_HIP_ERR_OOM;
    if (total) {
        if (int rc = with_activation(act, [&](auto a) -> int {
                hipLaunchKernelGGL(gn_sums_k<a.value>, dim3((unsigned)(N * C)), dim3(kBlock), 0, stream(), p, dy, x, scale, bias, means, rstds,
                                   sums);
                DOPT_LAUNCH_CHECK();
                hipLaunchKernelGGL(gn_dx_k<a.value>, dim3((unsigned)(N * groups)), dim3(kBlock), 0, stream(), p, dy, x, scale, bias, means,
                                   rstds, sums, packed);
                DOPT_LAUNCH_CHECK();
                return DOPT_HIP_OK;
            }))
            return rc;
    }
    hipLaunchKernelGGL(gn_fold_k, dim3((unsigned)ceil_div(C, (size_t)kBlock)), dim3(kBlock), 0, stream(), total ? N : 0, C, sums,
                       packed + total, packed + total + C);
    DOPT_LAUNCH_CHECK();
    return DOPT_HIP_OK;
}

}  // extern "C"
