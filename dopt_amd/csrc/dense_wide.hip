// Products of large dense layers, forward and backward: both operands are laid out once as two fp16 parts and go to the matrix instruction
// from there, the layer's end rides in the product.
//
// Rows are scaled by powers of two, each to a largest value in [2^14, 2^15), so h + l is off by at most 2^-22 of a value and 2^-40 of
// the largest one of its row (fp16's last subnormal place).  l l is left out, 2^-22 of a product at most.  Together with sums in fp32
//     |error| <= (K 2^-24 + 2^-20) sum |x| |w| + 2^-39 K max |x row| max |w row|
// that is, fp32's own rounding of a long sum unless a row spans more than fifteen binary orders and its largest values meet zeros.
// Three bf16 parts, which sgemm.hip uses for operands of any kind, keep 24 bits and take twice the matrix work.
//
// Bound by the matrix instructions: 6 M N K operations.
#include <algorithm>
#include <type_traits>

#include "common.h"
#include "dense.h"
#include "half_parts.h"

namespace {

using namespace dopt;

typedef float v4f_any __attribute__((ext_vector_type(4), aligned(4)));
typedef int v4i __attribute__((ext_vector_type(4)));

constexpr int kTile = 256, kThreads = 512, kStages = 4, kStage = 32768;
constexpr int kInf = 1 << 20, kNan = 1 << 21;   // in a row's shift: it holds infinities, NaN

struct Operand {
    const float *x;
    size_t rows, padded;
    char *parts;
    int *shift;   // of each row: it is held times 2^shift
};

// (by value: of an element of a vector the builtin takes the first one's bits)
__device__ __forceinline__ unsigned magnitude(float v) { return __builtin_bit_cast(unsigned, v) & 0x7fffffffu; }

// What a row is held times, from its largest magnitude.
__device__ __forceinline__ int shift_of(unsigned top)
{
    if (top > 0x7f800000u) return kNan;
    if (top == 0x7f800000u) return kInf;
    if (top >= 0x800000u) return 14 + 127 - (int)(top >> 23);
    return top ? 14 + 149 - (31 - __builtin_clz(top)) : 0;
}

// Eight steps of a row of a block.
__device__ __forceinline__ void store_parts(char *block, int row, int half, const float *v)
{
    v2u h0, l0, h1, l1;
    split4(v, h0, l0);
    split4(v + 4, h1, l1);
    *(v4u *)(block + piece_at(row, 2 * half)) = v4u{h0.x, h0.y, h1.x, h1.y};
    *(v4u *)(block + piece_at(row, 2 * half + 1)) = v4u{l0.x, l0.y, l1.x, l1.y};
}

// Four rows per workgroup, eight values of a row to each of its threads and those of kUnits further places, in registers between the
// search for the rows' largest values and the layout: sixteen steps of the four rows are stored by eight threads, 256 bytes
// in a line.  Bound by memory; read twice, through an L2 that holds no row for so long, [8192 + 4096] rows of 4096 took 106 us.
// Longer rows than the registers hold are.  Padding and rows that are not finite become zeros.
constexpr int kUnits = 8;
__global__ __launch_bounds__(1024) void wide_split_k(Operand a, Operand b, unsigned blocks_a, size_t K, size_t steps)
{
    __shared__ unsigned tops[16][4];
    const Operand o = blockIdx.x < blocks_a ? a : b;
    const size_t row0 = (size_t)(blockIdx.x < blocks_a ? blockIdx.x : blockIdx.x - blocks_a) * 4;
    const int lane = threadIdx.x & 63, r = threadIdx.x >> 1 & 3, half = threadIdx.x & 1, waves = blockDim.x >> 6;
    const size_t stride = blockDim.x / 8, s0 = threadIdx.x / 8;
    const bool inside = row0 + r < o.rows;
    const float *const x = o.x + min(row0 + r, o.rows - 1) * K;
    v4f v[kUnits][2];
    unsigned top = 0;   // of the values' magnitudes as integers, whose order is theirs, infinity and NaN last
    auto load = [&](size_t step, bool whole, v4f *to) {   // whole: all of the workgroup's steps lie inside
        const size_t k = step * 16 + half * 8;
        if (whole) {
            to[0] = *(const v4f_any *)(x + k);
            to[1] = *(const v4f_any *)(x + k + 4);
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) to[e / 4][e % 4] = k + e < K ? x[k + e] : 0.0f;
        }
    };
    auto see = [&](const v4f *of) {
#pragma unroll
        for (int e = 0; e < 8; e++) top = max(top, magnitude(of[e / 4][e % 4]));
    };
#pragma unroll
    for (int i = 0; i < kUnits; i++)
        if (i * stride < steps) load(s0 + i * stride, (i + 1) * stride * 16 <= K, v[i]);
#pragma unroll
    for (int i = 0; i < kUnits; i++)
        if (i * stride < steps) see(v[i]);
    for (size_t i = kUnits; i * stride < steps; i++) {
        v4f more[2];
        load(s0 + i * stride, (i + 1) * stride * 16 <= K, more);
        see(more);
    }
#pragma unroll
    for (int m = 32; m; m >>= 1)
        if (m != 2 && m != 4) top = max(top, (unsigned)__shfl_xor((int)top, m, 64));
    if ((lane & ~6) == 0) tops[threadIdx.x >> 6][r] = top;
    __syncthreads();
    top = tops[0][r];
    for (int i = 1; i < waves; i++) top = max(top, tops[i][r]);
    const int shift = inside ? shift_of(top) : 0;
    if (threadIdx.x < 8 && half == 0) o.shift[row0 + r] = shift;
    const bool live = inside && shift < kInf;
    auto put = [&](size_t step, const v4f *of) {
        if (step >= steps) return;
        float u[8];
#pragma unroll
        for (int e = 0; e < 8; e++) u[e] = live ? __builtin_ldexpf(of[e / 4][e % 4], shift) : 0.0f;
        store_parts(o.parts + ((row0 >> 5) * steps + step) * 2048, (int)(row0 & 31) + r, half, u);
    };
#pragma unroll
    for (int i = 0; i < kUnits; i++)
        if (i * stride < steps) put(s0 + i * stride, v[i]);
    for (size_t i = kUnits; i * stride < steps; i++) {
        v4f more[2];
        load(s0 + i * stride, (i + 1) * stride * 16 <= K, more);
        put(s0 + i * stride, more);
    }
}

// Operands that lie across the reduction, [K][rows]: the largest values of runs of K for each column, then a tile of 64 steps by 64 columns
// per workgroup, turned in LDS.
constexpr int kRuns = 32;
struct Across {
    Operand o;
    unsigned *tops;   // [run][row]
    unsigned tiles;   // of 256 columns; of 64 columns, padding included
};

__global__ __launch_bounds__(256) void wide_tops_k(Across a, size_t K, int runs)
{
    __shared__ unsigned red[4][256];
    const size_t col = min((size_t)(blockIdx.x % a.tiles) * 256 + (threadIdx.x & 63) * 4, a.o.rows - 4), run = blockIdx.x / a.tiles;
    const size_t from = K * run / runs, to = K * (run + 1) / runs;
    const int row = threadIdx.x >> 6;
    unsigned top[4] = {0, 0, 0, 0};
    size_t k = from + row;
    auto see = [&](v4f v) {
#pragma unroll
        for (int e = 0; e < 4; e++) top[e] = max(top[e], magnitude(v[e]));
    };
    for (; k + 28 < to; k += 32) {
        v4f v[8];
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = *(const v4f_any *)(a.o.x + (k + 4 * i) * a.o.rows + col);
#pragma unroll
        for (int i = 0; i < 8; i++) see(v[i]);
    }
    for (; k < to; k += 4) see(*(const v4f_any *)(a.o.x + k * a.o.rows + col));
#pragma unroll
    for (int e = 0; e < 4; e++) red[row][(threadIdx.x & 63) * 4 + e] = top[e];
    __syncthreads();
    if (row) return;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const int c = (threadIdx.x & 63) * 4 + e;
        a.tops[run * a.o.rows + col + e] = max(max(red[0][c], red[1][c]), max(red[2][c], red[3][c]));
    }
}

__global__ __launch_bounds__(256) void wide_turn_k(Across a, size_t K, size_t steps, int runs)
{
    __shared__ float tile[64][65];
    __shared__ unsigned tops[4][64];
    const size_t c0 = (size_t)(blockIdx.x % a.tiles) * 64, k0 = (size_t)(blockIdx.x / a.tiles) * 64;
    const int c = threadIdx.x & 63, w = threadIdx.x >> 6;
    const size_t col = min(c0 + c, a.o.rows - 1);
    float v[16];
#pragma unroll
    for (int u = 0; u < 16; u++) v[u] = a.o.x[min(k0 + w + 4 * u, K - 1) * a.o.rows + col];
    unsigned top = 0;
#pragma unroll
    for (int i = 0; i < kRuns / 4; i++) top = max(top, a.tops[min(w + 4 * i, runs - 1) * a.o.rows + col]);
    tops[w][c] = top;
    __syncthreads();
    const bool inside = c0 + c < a.o.rows;
    const int shift = inside ? shift_of(max(max(tops[0][c], tops[1][c]), max(tops[2][c], tops[3][c]))) : 0;
    if (k0 == 0 && w == 0) a.o.shift[c0 + c] = shift;
#pragma unroll
    for (int u = 0; u < 16; u++) {
        const int k = w + 4 * u;
        tile[k][c] = inside && shift < kInf && k0 + k < K ? __builtin_ldexpf(v[u], shift) : 0.0f;
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < 2; u++) {   // a wavefront stores a block at a time
        const int r = (threadIdx.x >> 1 & 31) + 32 * u, half = threadIdx.x & 1;
        const size_t step = k0 / 16 + w;
        if (step >= steps) break;
        float p[8];
#pragma unroll
        for (int e = 0; e < 8; e++) p[e] = tile[w * 16 + half * 8 + e][r];
        store_parts(a.o.parts + ((c0 + r) / 32 * steps + step) * 2048, r & 31, half, p);
    }
}

struct Wide {
    size_t M, N, K, steps;
    const float *x, *w;
    size_t xm, xk, wn, wk;   // between rows, between steps
    const char *xp, *wp;
    const int *xs, *ws;
    unsigned tiles, mtiles, ntiles;
};

// What is not finite in a tile's operands: the sums of those rows and columns as fp32 instructions make them.
__device__ __noinline__ void rough_sums(Wide q, DenseEpilogue ep, float *y, size_t m0, size_t n0, const int *shift)
{
    for (int i = threadIdx.x; i < kTile * kTile; i += kThreads) {
        const size_t m = m0 + i / kTile, n = n0 + i % kTile;
        const int most = max(shift[i / kTile], shift[kTile + i % kTile]);
        if (m >= q.M || n >= q.N || most < kInf) continue;
        const bool nan = most == kNan;
        float s = nan ? __builtin_nanf("") : 0.0f;
        if (!nan)
            for (size_t k = 0; k < q.K; k++) s += q.x[m * q.xm + k * q.xk] * q.w[n * q.wn + k * q.wk];
        y[m * q.N + n] = ep(s, m * q.N + n);
    }
}

__device__ __forceinline__ void phase()
{
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
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
    auto bring_stage = [&](int k) {
        char *const to = lds + (k & 3) * kStage;
        bring(left + (size_t)k * 2048, 2, lane, to + w * 2048);
        bring(right + (size_t)k * 2048, 2, lane, to + 16384 + w * 2048);
    };
    auto arrived = [&](int ahead) {   // all loads but those of the last `ahead` stages asked for
        if (ahead >= 2) settled<8>();
        else if (ahead == 1) settled<4>();
        else settled<0>();
    };
    const int steps = (int)q.steps;
    for (int k = 0; k < min(steps, 3); k++) bring_stage(k);
    arrived(min(steps, 3) - 1);
    phase();
    if (wm) phase();
    for (int k = 0; k < steps; k++) {
        Side<4> a;
        Side<2> b;
        const char *const now = lds + (k & 3) * kStage;
        a.read(now + wm * 8192, lane);
        b.read(now + 16384 + wn * 4096, lane);
        if (k + 3 < steps) bring_stage(k + 3);
        if (wm) arrived(min(steps - 2 - k, 2));
        else asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        phase();
        __builtin_amdgcn_s_setprio(1);
        multiply(a, b, acc);
        __builtin_amdgcn_s_setprio(0);
        if (!wm) arrived(min(steps - 2 - k, 2));
        phase();
    }
    if (!wm) phase();
    meet();

    int *const shift = (int *)lds;
    const size_t m0 = (size_t)mt * kTile, n0 = (size_t)nt * kTile;
    const int mine = threadIdx.x < kTile ? q.xs[m0 + threadIdx.x] : q.ws[n0 + threadIdx.x - kTile];
    shift[threadIdx.x] = mine;
    const bool rough = __syncthreads_or(mine >= kInf);
    // 32 rows at a time through LDS, so that a row's 64 values are stored by sixteen lanes
    float *const image = (float *)(lds + 2048) + w * (32 * 68);
    const bool inside = m0 + kTile <= q.M && n0 + kTile <= q.N && !rough;
    const size_t left_col = n0 + wn * 64;   // of the wavefront's 64
    // values one by one: beside values that are not finite, and where the matrix ends within the wavefront's first three columns
    const bool single = rough || (left_col < q.N && left_col + 4 > q.N);
    // quads end with the matrix: the lanes that would pass its end take its last quad once more
    const int col = single ? 4 * (lane & 15) : (int)(min(left_col + 4 * (lane & 15), q.N - 4) - left_col);
    const size_t n = left_col + col;
    int sn[4];
    v4f bias{0.0f, 0.0f, 0.0f, 0.0f};
    if (left_col < q.N && !single) {
#pragma unroll
        for (int e = 0; e < 4; e++) sn[e] = shift[kTile + wn * 64 + col + e];
        if (ep.bias) bias = *(const v4f_any *)(ep.bias + n);
    }
    // (a loop, whose sums move down: its code unrolled, for each activation, costs more to fetch than 96 moves)
#pragma unroll 1
    for (int i = 0; i < 4 && left_col < q.N; i++) {
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
            for (int e = 0; e < 16; e++) image[(8 * (e >> 2) + 4 * (lane >> 5) + (e & 3)) * 68 + 32 * j + (lane & 31)] = acc[0][j][e];
        asm volatile("" ::: "memory");   // (a wavefront's LDS accesses stay in their order)
        const int r0 = wm * 128 + i * 32 + (lane >> 4);
        with_activation(ep.act, [&](auto kind) {
            auto quads = [&](auto whole) {   // whole: nothing ends within the tile
                constexpr bool kWhole = decltype(whole)::value;
                v4f res[8];
                if (ep.residual) {
#pragma unroll
                    for (int t = 0; t < 8; t++) res[t] = *(const v4f_any *)(ep.residual + (kWhole ? m0 + r0 + 4 * t : min(m0 + r0 + 4 * t, q.M - 1)) * q.N + n);
                }
#pragma unroll
                for (int t = 0; t < 8; t++) {
                    const float *const from = image + (4 * t + (lane >> 4)) * 68 + col;
                    const int sm = shift[r0 + 4 * t];
                    const size_t m = m0 + r0 + 4 * t, at = m * q.N + n;
                    v4f z, o;
                    if (kWhole) z = *(const v4f *)from;
                    else z = v4f{from[0], from[1], from[2], from[3]};
#pragma unroll
                    for (int e = 0; e < 4; e++) z[e] = __builtin_ldexpf(z[e], -(sm + sn[e])) + bias[e];
#pragma unroll
                    for (int e = 0; e < 4; e++) o[e] = act_value<kind.value>(z[e]);
                    if (ep.residual) o += res[t];
                    if (kWhole || m < q.M) {
                        if (ep.pre) *(v4f_any *)(ep.pre + at) = z;
                        *(v4f_any *)(y + at) = o;
                    }
                }
            };
            if (inside) {
                quads(std::true_type{});
            } else if (!single) {
                quads(std::false_type{});
            } else {
                for (int t = 0; t < 8; t++) {
                    const int sm = shift[r0 + 4 * t];
                    const size_t m = m0 + r0 + 4 * t;
                    if (m >= q.M || sm >= kInf) continue;
                    for (int e = 0; e < 4; e++) {
                        if (n + e >= q.N) break;
                        const int s = shift[kTile + wn * 64 + col + e];
                        if (s >= kInf) continue;
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
#pragma unroll
        for (int k = 0; k < 3; k++)
#pragma unroll
            for (int j = 0; j < 2; j++) acc[k][j] = acc[k + 1][j];
    }
    if (rough) rough_sums(q, ep, y, m0, n0, shift);
}

}  // namespace

namespace dopt {

// Where a third of the chip's places for tiles are taken.  us here and on three bf16 parts, with 128, 512 and 1024 steps:
//     [1024 x 4096] 36 57 84 and 29 51 85    [1500 x 4096] 37 63 93 and 36 69 113    [4096 x 2500] 55 77 109 and 91 153 198
//     [4096 x 4097] 96 142 210 and 140 234 362    [8192 x 4096] 130 187 268 and 160 308 472
bool dense_wide_takes(size_t M, size_t N, size_t K)
{
    const size_t tiles = ceil_div(M, (size_t)kTile) * ceil_div(N, (size_t)kTile), rounds = ceil_div(tiles, (size_t)num_cus());
    return M >= 512 && N >= 512 && K >= 128 && tiles < ((size_t)1 << 30) && M * N * 3 >= rounds * num_cus() * kTile * kTile;
}

size_t dense_wide_scratch(size_t M, size_t N, size_t K)
{
    const size_t mp = ceil_div(M, (size_t)kTile) * kTile, np = ceil_div(N, (size_t)kTile) * kTile;
    return (mp + np) * (ceil_div(K, (size_t)16) * 64 + sizeof(int)) + kRuns * std::max(M, N) * sizeof(unsigned);
}

int dense_wide(size_t M, size_t N, size_t K, const WideSide &x, const WideSide &w, const DenseEpilogue &e, float *y)
{
    const size_t mp = ceil_div(M, (size_t)kTile) * kTile, np = ceil_div(N, (size_t)kTile) * kTile, steps = ceil_div(K, (size_t)16);
    char *const to = (char *)workspace(dense_wide_scratch(M, N, K));
    if (!to) return DOPT_HIP_ERR_OOM;
    char *const xp = to, *const wp = xp + mp * steps * 64;
    int *const xs = (int *)(wp + np * steps * 64), *const ws = xs + mp;
    unsigned *const tops = (unsigned *)(ws + np);
    const Operand both[] = {{x.values, M, mp, xp, xs}, {w.values, N, np, wp, ws}};
    const unsigned threads = steps > 512 ? 1024 : steps > 256 ? 512 : 256;   // rows in registers up to 16384
    if (!x.across && !w.across) {   // in one launch
        const unsigned blocks = (unsigned)(mp / 4);
        hipLaunchKernelGGL(wide_split_k, dim3(blocks + (unsigned)(np / 4)), dim3(threads), 0, stream(), both[0], both[1], blocks, K, steps);
        DOPT_LAUNCH_CHECK();
    } else {
        const bool across[] = {x.across, w.across};
        for (int i = 0; i < 2; i++) {
            const Operand &o = both[i];
            if (!across[i]) {
                const unsigned blocks = (unsigned)(o.padded / 4);
                hipLaunchKernelGGL(wide_split_k, dim3(blocks), dim3(threads), 0, stream(), o, o, blocks, K, steps);
                DOPT_LAUNCH_CHECK();
                continue;
            }
            const int runs = (int)std::min((size_t)kRuns, ceil_div(K, (size_t)64));
            Across a{o, tops, (unsigned)ceil_div(o.rows, (size_t)256)};
            hipLaunchKernelGGL(wide_tops_k, dim3(a.tiles * runs), dim3(256), 0, stream(), a, K, runs);
            DOPT_LAUNCH_CHECK();
            a.tiles = (unsigned)(o.padded / 64);
            hipLaunchKernelGGL(wide_turn_k, dim3(a.tiles * (unsigned)ceil_div(steps, (size_t)4)), dim3(256), 0, stream(), a, K, steps, runs);
            DOPT_LAUNCH_CHECK();
        }
    }
    static bool raised = false;
    if (!raised) DOPT_HIP_CHECK(hipFuncSetAttribute((const void *)wide_product_k, hipFuncAttributeMaxDynamicSharedMemorySize, kStages * kStage));
    raised = true;
    const unsigned mt = (unsigned)(mp / kTile), nt = (unsigned)(np / kTile);
    hipLaunchKernelGGL(wide_product_k, dim3(xcd_grid(mt * nt)), dim3(kThreads), kStages * kStage, stream(),
                       Wide{M, N, K, steps, x.values, w.values, x.across ? 1 : K, x.across ? M : 1, w.across ? 1 : K, w.across ? N : 1, xp, wp, xs, ws, mt * nt,
                            mt, nt},
                       e, y);
    DOPT_LAUNCH_CHECK();
    return DOPT_HIP_OK;
}

}  // namespace dopt
