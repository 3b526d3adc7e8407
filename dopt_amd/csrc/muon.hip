// Updates that treat a weight as a matrix: the momentum's orthogonalised form takes the place of the momentum.
// No counterpart in the reference, whose rules are elementwise (online/source/dopt/online/{sgd,adam,amsgrad}.d).
//
//     m' = mu m + g,  u = g + mu m' (nesterov) or m',  X = u / (|u| + 1e-7) in the 2-norm of all values
//     `iterations` times, on the side of fewer rows:  A = X X^T,  X' = a X + (b A + c A A) X
//     w' = (1 - lr decay) w - lr sqrt(max(1, rows / cols)) X
#include <cmath>
#include <vector>

#include "common.h"

namespace {

using namespace dopt;

constexpr int kBlock = 256, kParts = 64;
constexpr float kA = 3.4445f, kB = -4.7750f, kC = 2.0315f, kEps = 1e-7f;

struct Handle {
    std::vector<dopt_hip_matrix_ref> refs;
    float *x = nullptr, *y = nullptr, *a = nullptr, *aa = nullptr;
    double *parts = nullptr;
};

unsigned flat_grid(size_t n) { return (unsigned)std::min(ceil_div(n, (size_t)kBlock), (size_t)num_cus() * 16); }

__device__ inline float step_value(float g, float m, float mu, int nesterov) { return nesterov ? g + mu * m : m; }

__global__ __launch_bounds__(kBlock) void muon_momentum_k(size_t n, const float *g, float *m, float mu, int nesterov, double *parts)
{
    __shared__ double red[kBlock];
    double s = 0.0;
    for (size_t i = (size_t)blockIdx.x * kBlock + threadIdx.x; i < n; i += (size_t)kParts * kBlock) {
        const float v = mu * m[i] + g[i];
        m[i] = v;
        const double u = step_value(g[i], v, mu, nesterov);
        s += u * u;
    }
    red[threadIdx.x] = s;
    for (int k = kBlock / 2; k > 0; k >>= 1) {
        __syncthreads();
        if ((int)threadIdx.x < k) red[threadIdx.x] += red[threadIdx.x + k];
    }
    if (threadIdx.x == 0) parts[blockIdx.x] = red[0];
}

// x[r][c] with r the shorter side.
__global__ __launch_bounds__(kBlock) void muon_scale_k(size_t rows, size_t cols, const float *g, const float *m, float mu, int nesterov,
                                                       const double *parts, float *x)
{
    double s = 0.0;
    for (int i = 0; i < kParts; i++) s += parts[i];
    const float by = (float)(1.0 / (sqrt(s) + (double)kEps));
    const size_t n = rows * cols;
    const bool tall = rows > cols;
    for (size_t i = (size_t)blockIdx.x * kBlock + threadIdx.x; i < n; i += (size_t)gridDim.x * kBlock) {
        const float v = step_value(g[i], m[i], mu, nesterov) * by;
        x[tall ? i % cols * rows + i / cols : i] = v;
    }
}

__global__ __launch_bounds__(kBlock) void muon_lincomb_k(size_t n, float p, const float *a, float q, const float *b, float *o)
{
    for (size_t i = (size_t)blockIdx.x * kBlock + threadIdx.x; i < n; i += (size_t)gridDim.x * kBlock) o[i] = p * a[i] + q * b[i];
}

__global__ __launch_bounds__(kBlock) void muon_apply_k(size_t rows, size_t cols, const float *x, float keep, float by, float *w)
{
    const size_t n = rows * cols;
    const bool tall = rows > cols;
    for (size_t i = (size_t)blockIdx.x * kBlock + threadIdx.x; i < n; i += (size_t)gridDim.x * kBlock)
        w[i] = keep * w[i] - by * x[tall ? i % cols * rows + i / cols : i];
}

void release(Handle *h)
{
    for (void *p : {(void *)h->x, (void *)h->y, (void *)h->a, (void *)h->aa, (void *)h->parts}) dopt_hip_free(p);
    delete h;
}

}  // namespace

extern "C" {

int dopt_hip_muon_create(int nmatrices, const dopt_hip_matrix_ref *refs, void **handle)
{
    DOPT_REQUIRE(handle != nullptr, "dopt_hip_muon_create: handle is null");
    *handle = nullptr;
    DOPT_REQUIRE(nmatrices >= 0 && (nmatrices == 0 || refs), "dopt_hip_muon_create: bad list of matrices");
    for (int i = 0; i < nmatrices; i++) {
        const dopt_hip_matrix_ref &r = refs[i];
        DOPT_REQUIRE(r.rows <= 65536 && r.cols <= ((size_t)1 << 28) && r.rows * r.cols <= ((size_t)1 << 28) && std::min(r.rows, r.cols) <= 16384,
                     "dopt_hip_muon_create: matrix %d is too large", i);
        const size_t n = r.rows * r.cols;
        DOPT_REQUIRE(n == 0 || (r.w && r.g && r.m), "dopt_hip_muon_create: matrix %d has a null w, g or m", i);
        // all matrices are updated at the same time: what one writes nobody else may read or write
        const size_t bytes = n * sizeof(float);
        for (int j = 0; j <= i; j++) {
            const dopt_hip_matrix_ref &q = refs[j];
            const size_t k = q.rows * q.cols * sizeof(float);
            const void *written[] = {r.w, r.m}, *theirs[] = {q.w, q.m, q.g};
            bool shared = overlaps(r.g, bytes, q.w, k) || overlaps(r.g, bytes, q.m, k);
            for (int a = 0; a < 2; a++)
                for (int b = 0; b < 3; b++) shared = shared || ((i != j || a != b) && overlaps(written[a], bytes, theirs[b], k));
            DOPT_REQUIRE(!shared, "dopt_hip_muon_create: matrices %d and %d share memory that is written", j, i);
        }
    }
    DOPT_ENSURE_INIT();
    Handle *h = new Handle();
    size_t most = 0, side = 0;
    for (int i = 0; i < nmatrices; i++) {
        if (refs[i].rows * refs[i].cols == 0) continue;
        h->refs.push_back(refs[i]);
        most = std::max(most, refs[i].rows * refs[i].cols);
        side = std::max(side, std::min(refs[i].rows, refs[i].cols));
    }
    int rc = scratch_alloc((void **)&h->x, most * sizeof(float));
    if (!rc) rc = scratch_alloc((void **)&h->y, most * sizeof(float));
    if (!rc) rc = scratch_alloc((void **)&h->a, side * side * sizeof(float));
    if (!rc) rc = scratch_alloc((void **)&h->aa, side * side * sizeof(float));
    if (!rc) rc = scratch_alloc((void **)&h->parts, kParts * sizeof(double));
    if (rc) {
        release(h);
        return rc;
    }
    *handle = h;
    return DOPT_HIP_OK;
}

int dopt_hip_muon_destroy(void *handle)
{
    if (handle) release((Handle *)handle);
    return DOPT_HIP_OK;
}

int dopt_hip_muon_step(void *handle, float lr, float mu, int nesterov, float decay, int iterations)
{
    DOPT_REQUIRE(handle != nullptr, "dopt_hip_muon_step: handle is null");
    DOPT_REQUIRE(iterations >= 0 && iterations <= 100, "dopt_hip_muon_step: %d iterations", iterations);
    Handle *h = (Handle *)handle;
    for (const dopt_hip_matrix_ref &r : h->refs) {
        const size_t n = r.rows * r.cols, s = std::min(r.rows, r.cols), l = std::max(r.rows, r.cols);
        hipLaunchKernelGGL(muon_momentum_k, dim3(kParts), dim3(kBlock), 0, stream(), n, r.g, r.m, mu, nesterov, h->parts);
        hipLaunchKernelGGL(muon_scale_k, dim3(flat_grid(n)), dim3(kBlock), 0, stream(), r.rows, r.cols, r.g, r.m, mu, nesterov, h->parts, h->x);
        DOPT_LAUNCH_CHECK();
        for (int it = 0; it < iterations; it++) {
            if (int rc = dopt_hip_sgemm_t(0, 1, s, s, l, h->x, h->x, h->a)) return rc;
            if (int rc = dopt_hip_sgemm_t(0, 1, s, s, s, h->a, h->a, h->aa)) return rc;   // A is symmetric
            hipLaunchKernelGGL(muon_lincomb_k, dim3(flat_grid(s * s)), dim3(kBlock), 0, stream(), s * s, kB, h->a, kC, h->aa, h->aa);
            if (int rc = dopt_hip_sgemm_t(0, 0, s, l, s, h->aa, h->x, h->y)) return rc;
            hipLaunchKernelGGL(muon_lincomb_k, dim3(flat_grid(n)), dim3(kBlock), 0, stream(), n, kA, h->x, 1.0f, h->y, h->x);
            DOPT_LAUNCH_CHECK();
        }
        const float by = lr * std::sqrt(std::max(1.0f, (float)r.rows / (float)r.cols));
        hipLaunchKernelGGL(muon_apply_k, dim3(flat_grid(n)), dim3(kBlock), 0, stream(), r.rows, r.cols, h->x, 1.0f - lr * decay, by, r.w);
        DOPT_LAUNCH_CHECK();
    }
    return DOPT_HIP_OK;
}

}  // extern "C"
