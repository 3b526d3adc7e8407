// The norm of all gradients of a training step, what clipping multiplies them by, and the clipped gradients.
// No counterpart in the reference, whose updaters take gradients as they come (online/source/dopt/online/*.d).
//
//     norm = sqrt(sum over all tensors of g^2),  factor = norm <= max ? 1 : max / norm,  out = factor g
//
// The squares and their sum are formed in 64 bits: a value's square neither overflows nor vanishes there, and a sum of any length
// rounds to the norm's last place.  The updates read the factor where they read the gradients (optim.hip, muon.hip), so that clipping costs them no pass.
// Bound by memory: four bytes a value for the norm, eight more where the clipped gradients are written.  36.5 million values: the norm 24.7 us (5.9 TB/s, the last
// cache's share included), the clipped gradients 44.8 behind it, which start with what the norm has read last; 670 thousand 5.0 and 3.4, a launch each.
#include <algorithm>
#include <cmath>
#include <new>
#include <vector>

#include "common.h"

namespace {

using namespace dopt;

constexpr int kBlock = 512;
constexpr int kQuads = 4;                                // sixteen bytes each, of a thread and chunk
constexpr size_t kChunk = (size_t)kBlock * kQuads * 4;   // values

struct Tensor {
    const float *g;
    float *out;
    size_t n;
    int vec;   // both on 16-byte boundaries
};
struct Chunk {
    unsigned tensor;
    size_t offset;
};

struct Handle {
    size_t nchunks = 0;
    unsigned blocks = 1;        // of the launch that forms the squares
    bool has_out = true;
    Tensor *tensors = nullptr;  // device, these three
    Chunk *chunks = nullptr;
    double *parts = nullptr;    // a block's sum
    unsigned *arrived = nullptr;   // counts of them; zero between two calls
    std::vector<dopt_hip_gradient_ref> refs;
};

// The workgroup's sum, in every thread.
__device__ __forceinline__ double block_sum(double s)
{
    __shared__ double red[kBlock / 64];
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    s = red[0];
#pragma unroll
    for (int i = 1; i < kBlock / 64; i++) s += red[i];
    __syncthreads();
    return s;
}

// Blocks are counted by kTeam, and teams where their last block arrives: additions to one place go one after the other, ten
// nanoseconds each (1024 blocks in one count took 10 us at the end of the launch).
constexpr unsigned kTeam = 32, kApart = 32;   // values between two counts: a line each

__device__ __forceinline__ bool completes(unsigned *count, unsigned of)   // leaves it zero for the next call
{
    if (__hip_atomic_fetch_add(count, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1 != of) return false;
    __hip_atomic_store(count, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return true;
}
__device__ __forceinline__ bool arrives(unsigned *counts)   // true in the block that is the last of all
{
    const unsigned team = blockIdx.x / kTeam, teams = (gridDim.x + kTeam - 1) / kTeam;
    return completes(counts + (1 + team) * kApart, min(kTeam, gridDim.x - team * kTeam)) && (teams == 1 || completes(counts, teams));
}

// The block that arrives last adds the others' sums, in their order.
__global__ __launch_bounds__(kBlock) void gradient_squares_k(const Tensor *tensors, const Chunk *chunks, size_t nchunks, double *parts, unsigned *arrived,
                                                             float most, float *result)
{
    __shared__ bool last;
    double s = 0.0;
    auto add = [&](float v) { s = __builtin_fma((double)v, (double)v, s); };
    for (size_t ci = blockIdx.x; ci < nchunks; ci += gridDim.x) {
        const Chunk ch = chunks[ci];
        const Tensor t = tensors[ch.tensor];
        const size_t to = min(ch.offset + kChunk, t.n);
        if (t.vec && to - ch.offset == kChunk) {
            float4 v[kQuads];
#pragma unroll
            for (int u = 0; u < kQuads; u++) v[u] = ((const float4 *)(t.g + ch.offset))[u * kBlock + threadIdx.x];
#pragma unroll
            for (int u = 0; u < kQuads; u++) {
                add(v[u].x);
                add(v[u].y);
                add(v[u].z);
                add(v[u].w);
            }
        } else {
            for (size_t i = ch.offset + threadIdx.x; i < to; i += kBlock) add(t.g[i]);
        }
    }
    s = block_sum(s);
    if (threadIdx.x == 0) {
        __hip_atomic_store((unsigned long long *)parts + blockIdx.x, __builtin_bit_cast(unsigned long long, s), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        // The sum is where every XCD reads it once its store has been acknowledged; only then does the block count.  (An acquire and release
        // of the atomic itself writes back and drops each L2 with every block: 63 us instead of 24 for 36.5 million values.)
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        last = arrives(arrived);
    }
    __syncthreads();
    if (!last) return;
    s = 0.0;
    for (unsigned i = threadIdx.x; i < gridDim.x; i += kBlock)
        s += __builtin_bit_cast(double, __hip_atomic_load((unsigned long long *)parts + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
    s = sqrt(block_sum(s));
    if (threadIdx.x) return;
    result[0] = (float)s;
    result[1] = s <= (double)most ? 1.0f : (float)((double)most / s);
}

__global__ __launch_bounds__(kBlock) void gradient_scale_k(const Tensor *tensors, const Chunk *chunks, size_t nchunks, const float *result)
{
    const float by = result[1];
    for (size_t ci = blockIdx.x; ci < nchunks; ci += gridDim.x) {
        const Chunk ch = chunks[nchunks - 1 - ci];   // what the norm has read last first
        const Tensor t = tensors[ch.tensor];
        if (by == 1.0f && t.g == t.out) continue;
        const size_t to = min(ch.offset + kChunk, t.n);
        if (t.vec && to - ch.offset == kChunk) {
            float4 v[kQuads];
#pragma unroll
            for (int u = 0; u < kQuads; u++) v[u] = ((const float4 *)(t.g + ch.offset))[u * kBlock + threadIdx.x];
#pragma unroll
            for (int u = 0; u < kQuads; u++)
                ((float4 *)(t.out + ch.offset))[u * kBlock + threadIdx.x] = float4{v[u].x * by, v[u].y * by, v[u].z * by, v[u].w * by};
        } else {
            for (size_t i = ch.offset + threadIdx.x; i < to; i += kBlock) t.out[i] = t.g[i] * by;
        }
    }
}

// Whether a result shares memory with anything but the gradient that it replaces.
bool tangled(int n, const dopt_hip_gradient_ref *refs)
{
    struct Range {
        uintptr_t from, to;
        bool written;
    };
    std::vector<Range> all;
    for (int i = 0; i < n; i++) {
        const uintptr_t g = (uintptr_t)refs[i].g, out = (uintptr_t)refs[i].out, bytes = refs[i].n * sizeof(float);
        if (!bytes) continue;
        if (g != out) all.push_back(Range{g, g + bytes, false});
        if (out) all.push_back(Range{out, out + bytes, true});
    }
    std::sort(all.begin(), all.end(), [](const Range &a, const Range &b) { return a.from < b.from; });
    uintptr_t any = 0, written = 0;   // where what began before ends
    for (const Range &r : all) {
        if (r.from < (r.written ? any : written)) return true;
        any = std::max(any, r.to);
        if (r.written) written = std::max(written, r.to);
    }
    return false;
}

void release(Handle *h)
{
    dopt_hip_free(h->tensors);
    dopt_hip_free(h->chunks);
    dopt_hip_free(h->parts);
    dopt_hip_free(h->arrived);
    delete h;
}

int fill(Handle *h, int n, const dopt_hip_gradient_ref *refs)
{
    std::vector<Tensor> tensors;
    std::vector<Chunk> chunks;
    for (int i = 0; i < n; i++) {
        const dopt_hip_gradient_ref &r = refs[i];
        if (r.n > 0 && !r.out) h->has_out = false;
        tensors.push_back(Tensor{r.g, r.out, r.n, aligned16(r.g) && aligned16(r.out)});
        for (size_t at = 0; at < r.n; at += kChunk) chunks.push_back(Chunk{(unsigned)i, at});
    }
    h->refs.assign(refs, refs + n);
    h->nchunks = chunks.size();
    h->blocks = (unsigned)std::max((size_t)1, std::min(chunks.size(), (size_t)num_cus() * 4));
    int rc = dopt_hip_malloc((void **)&h->parts, h->blocks * sizeof(double));
    if (!rc) rc = dopt_hip_malloc((void **)&h->arrived, (1 + ceil_div(h->blocks, kTeam)) * kApart * sizeof(unsigned));   // (zero-filled)
    if (rc || chunks.empty()) return rc;
    rc = dopt_hip_malloc((void **)&h->tensors, tensors.size() * sizeof(Tensor));
    if (!rc) rc = dopt_hip_malloc((void **)&h->chunks, chunks.size() * sizeof(Chunk));
    if (!rc) rc = dopt_hip_copy_h2d(h->tensors, tensors.data(), tensors.size() * sizeof(Tensor));
    if (!rc) rc = dopt_hip_copy_h2d(h->chunks, chunks.data(), chunks.size() * sizeof(Chunk));
    return rc;
}

int norm(const Handle *h, float most, float *result, const char *who)
{
    DOPT_REQUIRE(result != nullptr, "%s: the result is null", who);
    DOPT_REQUIRE(most >= 0.0f, "%s: the largest norm is %g", who, (double)most);
    for (const dopt_hip_gradient_ref &r : h->refs)
        DOPT_REQUIRE(!overlaps(result, 2 * sizeof(float), r.g, r.n * sizeof(float)) && !overlaps(result, 2 * sizeof(float), r.out, r.n * sizeof(float)),
                     "%s: the norm's place lies in a gradient", who);
    hipLaunchKernelGGL(gradient_squares_k, dim3(h->blocks), dim3(kBlock), 0, stream(), h->tensors, h->chunks, h->nchunks, h->parts, h->arrived, most, result);
    DOPT_LAUNCH_CHECK();
    return DOPT_HIP_OK;
}

}  // namespace

extern "C" {

int dopt_hip_gradient_norm_create(int ntensors, const dopt_hip_gradient_ref *refs, void **handle)
{
    DOPT_REQUIRE(handle != nullptr, "dopt_hip_gradient_norm_create: handle is null");
    *handle = nullptr;
    DOPT_REQUIRE(ntensors >= 0 && (ntensors == 0 || refs), "dopt_hip_gradient_norm_create: bad tensor list");
    for (int i = 0; i < ntensors; i++) {
        DOPT_REQUIRE(refs[i].n == 0 || refs[i].g, "dopt_hip_gradient_norm_create: tensor %d is null", i);
        DOPT_REQUIRE(refs[i].n < (size_t)1 << 40, "dopt_hip_gradient_norm_create: tensor %d is too large", i);
    }
    Handle *h = nullptr;
    int rc;
    try {
        DOPT_REQUIRE(!tangled(ntensors, refs), "dopt_hip_gradient_norm_create: a result overlaps another result or a gradient that is not its own");
        DOPT_ENSURE_INIT();
        h = new Handle();
        rc = fill(h, ntensors, refs);
    } catch (const std::bad_alloc &) {
        rc = fail(DOPT_HIP_ERR_OOM, "dopt_hip_gradient_norm_create: out of host memory");
    }
    if (rc) {
        if (h) release(h);
        return rc;
    }
    *handle = h;
    return DOPT_HIP_OK;
}

int dopt_hip_gradient_norm_destroy(void *handle)
{
    if (handle) release((Handle *)handle);
    return DOPT_HIP_OK;
}

int dopt_hip_gradient_norm(void *handle, float max_norm, float *result)
{
    DOPT_REQUIRE(handle != nullptr, "dopt_hip_gradient_norm: handle is null");
    return norm((const Handle *)handle, max_norm, result, "dopt_hip_gradient_norm");
}

int dopt_hip_gradient_clip(void *handle, float max_norm, float *result)
{
    DOPT_REQUIRE(handle != nullptr, "dopt_hip_gradient_clip: handle is null");
    const Handle *const h = (const Handle *)handle;
    DOPT_REQUIRE(h->has_out, "dopt_hip_gradient_clip: a tensor has no place for its result");
    if (int rc = norm(h, max_norm, result, "dopt_hip_gradient_clip")) return rc;
    if (h->nchunks == 0) return DOPT_HIP_OK;
    const unsigned grid = (unsigned)std::min(h->nchunks, (size_t)num_cus() * 8);
    hipLaunchKernelGGL(gradient_scale_k, dim3(grid), dim3(kBlock), 0, stream(), h->tensors, h->chunks, h->nchunks, result);
    DOPT_LAUNCH_CHECK();
    return DOPT_HIP_OK;
}

}  // extern "C"
