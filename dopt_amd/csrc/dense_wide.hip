// Large dense layers forward: both operands are laid out once as two fp16 parts and go to the matrix instruction from there, the layer's end
// rides in the product.
//
// Rows are scaled by powers of two, each to a largest value in [2^14, 2^15), so h + l is off by at most 2^-22 of a value and 2^-40 of
// the largest one of its row (fp16's last subnormal place).  l l is left out, 2^-22 of a product at most.  Together with sums in fp32
//     |error| <= (K 2^-24 + 2^-20) sum |x| |w| + 2^-39 K max |x row| max |w row|
// that is, fp32's own rounding of a long sum unless a row spans more than fifteen binary orders and its largest values meet zeros.
// Three bf16 parts, which sgemm.hip uses for operands of any kind, keep 24 bits and take twice the matrix work.
//
// Bound by the matrix instructions: 6 M N K operations.
#include <algorithm>

#include "common.h"
#include "dense.h"
#include "half_parts.h"

namespace {

using namespace dopt;

typedef float v4f_any __attribute__((ext_vector_type(4), aligned(4)));
typedef int v4i __attribute__((ext_vector_type(4)));

constexpr int kBlock = 256, kTile = 256, kThreads = 512, kStages = 4, kStage = 32768;
constexpr int kInf = 1 << 20, kNan = 1 << 21;   // in a row's shift: it holds infinities, NaN

struct Operand {
    const float *x;
    size_t rows, padded;
    char *parts;
    int *shift;   // of each row: it is held times 2^shift
};

// (by value: of an element of a vector the builtin takes the first one's bits)
__device__ __forceinline__ unsigned magnitude(float v) { return __builtin_bit_cast(unsigned, v) & 0x7fffffffu; }

// Four rows per workgroup: a wavefront finds its row's largest value, then all of them lay out the four.  Bound by memory; the second
// reading finds most of the four rows in the L2.  Padding and rows that are not finite become zeros.
__global__ __launch_bounds__(kBlock) void wide_split_k(Operand a, Operand b, unsigned blocks_a, size_t K, size_t steps)
{
    __shared__ int shifts[4];
    const Operand o = blockIdx.x < blocks_a ? a : b;
    const size_t row0 = (size_t)(blockIdx.x < blocks_a ? blockIdx.x : blockIdx.x - blocks_a) * 4;
    const int w = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const size_t row = row0 + w;
    unsigned top = 0;   // of the values' magnitudes as integers, whose order is theirs, infinity and NaN last
    if (row < o.rows) {
        const float *const x = o.x + row * K;
        const size_t whole = K / 4 * 4;
#pragma unroll 8
        for (size_t k = lane * 4; k < whole; k += 256) {
            const v4f v = *(const v4f_any *)(x + k);
#pragma unroll
            for (int e = 0; e < 4; e++) top = max(top, magnitude(v[e]));
        }
        for (size_t k = whole + lane; k < K; k += 64) top = max(top, magnitude(x[k]));
    }
#pragma unroll
    for (int m = 32; m; m >>= 1) top = max(top, (unsigned)__shfl_xor((int)top, m, 64));
    int shift = 0;
    if (top > 0x7f800000u) shift = kNan;
    else if (top == 0x7f800000u) shift = kInf;
    else if (top >= 0x800000u) shift = 14 + 127 - (int)(top >> 23);
    else if (top) shift = 14 + 149 - (31 - __builtin_clz(top));
    if (lane == 0) {
        shifts[w] = shift;
        if (row < o.padded) o.shift[row] = shift;
    }
    __syncthreads();
    // sixteen steps of the four rows by eight threads, which store 256 bytes in a line
    const int r = threadIdx.x >> 1 & 3, half = threadIdx.x & 1;
    const int by = shifts[r];
    const bool live = row0 + r < o.rows && by < kInf;
    const float *const x = o.x + (row0 + r) * K;
    for (size_t s = threadIdx.x >> 3; s < steps; s += kBlock / 8) {
        const size_t k = s * 16 + half * 8;
        float v[8];
        if (live && k + 8 <= K) {
            const v4f p = *(const v4f_any *)(x + k), q = *(const v4f_any *)(x + k + 4);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                v[e] = p[e];
                v[4 + e] = q[e];
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = live && k + e < K ? x[k + e] : 0.0f;
        }
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = __builtin_ldexpf(v[e], by < kInf ? by : 0);
        v2u h0, l0, h1, l1;
        split4(v, h0, l0);
        split4(v + 4, h1, l1);
        char *const at = o.parts + ((row0 >> 5) * steps + s) * 2048;
        const int in = (int)(row0 & 31) + r;
        *(v4u *)(at + piece_at(in, 2 * half)) = v4u{h0.x, h0.y, h1.x, h1.y};
        *(v4u *)(at + piece_at(in, 2 * half + 1)) = v4u{l0.x, l0.y, l1.x, l1.y};
    }
}

struct Wide {
    size_t M, N, K, steps;
    const float *x, *w;
    const char *xp, *wp;
    const int *xs, *ws;
    unsigned tiles, mtiles, ntiles;
};

// What is not finite in a tile's operands: the sums of those rows and columns as fp32 instructions make them.
__device__ __noinline__ void rough_sums(const Wide &q, const DenseEpilogue &ep, float *y, size_t m0, size_t n0, const int *shift)
{
    for (int i = threadIdx.x; i < kTile * kTile; i += kThreads) {
        const size_t m = m0 + i / kTile, n = n0 + i % kTile;
        const int most = max(shift[i / kTile], shift[kTile + i % kTile]);
        if (m >= q.M || n >= q.N || most < kInf) continue;
        const bool nan = most == kNan;
        float s = nan ? __builtin_nanf("") : 0.0f;
        if (!nan)
            for (size_t k = 0; k < q.K; k++) s += q.x[m * q.K + k] * q.w[n * q.K + k];
        y[m * q.N + n] = ep(s, m * q.N + n);
    }
}

// A tile of 256 x 256 by eight wavefronts of 128 x 64: the accumulators are half of the registers, and a stage of 16 steps, 32 KB, feeds
// 24 matrix instructions of each.  Three stages are on their way behind the one in use.
__global__ __launch_bounds__(kThreads, 2) void wide_product_k(Wide q, DenseEpilogue ep, float *y)
{
    extern __shared__ __attribute__((aligned(16))) char lds[];
    unsigned id;
    if (!xcd_remap(blockIdx.x, q.tiles, &id)) return;
    // eight rows of tiles together, column by column: what an XCD works on at a time shares rows and columns
    const unsigned band = 8 * q.ntiles, first = id / band * 8, high = min(8u, q.mtiles - first);
    const unsigned mt = first + id % band % high, nt = id % band / high;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), wm = w >> 2, wn = w & 3;
    const size_t row_of_blocks = q.steps * 2048;
    const char *const left = q.xp + (mt * 8 + w) * row_of_blocks, *const right = q.wp + (nt * 8 + w) * row_of_blocks;
    v16f acc[4][2];
    zero_acc(acc);
    pipeline<kStages, kStage, 4>(
        lds, (int)q.steps,
        [&](int k, char *to) {
            bring(left + (size_t)k * 2048, 2, lane, to + w * 2048);
            bring(right + (size_t)k * 2048, 2, lane, to + 16384 + w * 2048);
        },
        [&](const char *now) { multiply(now + wm * 8192, now + 16384 + wn * 4096, lane, acc); });

    int *const shift = (int *)lds;
    const size_t m0 = (size_t)mt * kTile, n0 = (size_t)nt * kTile;
    const int mine = threadIdx.x < kTile ? q.xs[m0 + threadIdx.x] : q.ws[n0 + threadIdx.x - kTile];
    shift[threadIdx.x] = mine;
    const bool rough = __syncthreads_or(mine >= kInf);
    // 32 rows at a time through LDS, so that a row's 64 values are stored by sixteen lanes
    float *const image = (float *)(lds + 2048) + w * (32 * 68);
    const int col = 4 * (lane & 15);
    const size_t n = n0 + wn * 64 + col;
    const bool inside = m0 + kTile <= q.M && n0 + kTile <= q.N && !rough;
    const v4i sn = *(const v4i *)(shift + kTile + wn * 64 + col);
    v4f bias{0.0f, 0.0f, 0.0f, 0.0f};
    if (ep.bias) {
#pragma unroll
        for (int e = 0; e < 4; e++) bias[e] = n + e < q.N ? ep.bias[n + e] : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
            for (int e = 0; e < 16; e++) image[(8 * (e >> 2) + 4 * (lane >> 5) + (e & 3)) * 68 + 32 * j + (lane & 31)] = acc[i][j][e];
        asm volatile("" ::: "memory");   // (a wavefront's LDS accesses stay in their order)
        const int r0 = wm * 128 + i * 32 + (lane >> 4);
        with_activation(ep.act, [&](auto kind) {
            if (inside) {
                v4f res[8];
                if (ep.residual) {
#pragma unroll
                    for (int t = 0; t < 8; t++) res[t] = *(const v4f_any *)(ep.residual + (m0 + r0 + 4 * t) * q.N + n);
                }
#pragma unroll
                for (int t = 0; t < 8; t++) {
                    v4f z = *(const v4f *)(image + (4 * t + (lane >> 4)) * 68 + col), o;
                    const int sm = shift[r0 + 4 * t];
                    const size_t at = (m0 + r0 + 4 * t) * q.N + n;
#pragma unroll
                    for (int e = 0; e < 4; e++) z[e] = __builtin_ldexpf(z[e], -(sm + sn[e])) + bias[e];
                    if (ep.pre) *(v4f_any *)(ep.pre + at) = z;
#pragma unroll
                    for (int e = 0; e < 4; e++) o[e] = act_value<kind.value>(z[e]);
                    if (ep.residual) o += res[t];
                    *(v4f_any *)(y + at) = o;
                }
            } else {
                for (int t = 0; t < 8; t++) {
                    const int sm = shift[r0 + 4 * t];
                    const size_t m = m0 + r0 + 4 * t;
                    if (m >= q.M || sm >= kInf) continue;
                    for (int e = 0; e < 4; e++) {
                        const int s = shift[kTile + wn * 64 + col + e];
                        if (n + e >= q.N || s >= kInf) continue;
                        const size_t at = m * q.N + n + e;
                        const float z = __builtin_ldexpf(image[(4 * t + (lane >> 4)) * 68 + col + e], -(sm + s)) + ep.bias_of(n + e);
                        if (ep.pre) ep.pre[at] = z;
                        const float o = act_value<kind.value>(z);
                        y[at] = ep.residual ? o + ep.residual[at] : o;
                    }
                }
            }
        });
        asm volatile("" ::: "memory");
    }
    if (rough) rough_sums(q, ep, y, m0, n0, shift);
}

}  // namespace

namespace dopt {

bool dense_wide_takes(size_t M, size_t N, size_t K)
{
    return M >= 1024 && N >= 1024 && K >= 512 && ceil_div(M, (size_t)kTile) < ((size_t)1 << 20) && ceil_div(N, (size_t)kTile) < ((size_t)1 << 10);
}

int dense_wide(size_t M, size_t N, size_t K, const float *x, const float *w, const DenseEpilogue &e, float *y)
{
    const size_t mp = ceil_div(M, (size_t)kTile) * kTile, np = ceil_div(N, (size_t)kTile) * kTile, steps = ceil_div(K, (size_t)16);
    char *const to = (char *)workspace((mp + np) * (steps * 64 + sizeof(int)));
    if (!to) return DOPT_HIP_ERR_OOM;
    char *const xp = to, *const wp = xp + mp * steps * 64;
    int *const xs = (int *)(wp + np * steps * 64), *const ws = xs + mp;
    const unsigned blocks = (unsigned)(mp / 4);
    hipLaunchKernelGGL(wide_split_k, dim3(blocks + (unsigned)(np / 4)), dim3(kBlock), 0, stream(), Operand{x, M, mp, xp, xs}, Operand{w, N, np, wp, ws}, blocks,
                       K, steps);
    DOPT_LAUNCH_CHECK();
    static bool raised = false;
    if (!raised) DOPT_HIP_CHECK(hipFuncSetAttribute((const void *)wide_product_k, hipFuncAttributeMaxDynamicSharedMemorySize, kStages * kStage));
    raised = true;
    const unsigned mt = (unsigned)(mp / kTile), nt = (unsigned)(np / kTile);
    hipLaunchKernelGGL(wide_product_k, dim3(xcd_grid(mt * nt)), dim3(kThreads), kStages * kStage, stream(),
                       Wide{M, N, K, steps, x, w, xp, wp, xs, ws, mt * nt, mt, nt}, e, y);
    DOPT_LAUNCH_CHECK();
    return DOPT_HIP_OK;
}

}  // namespace dopt
