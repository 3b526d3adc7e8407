// What products of two fp16 parts are made of (dense_wide.hip, dense_groups_wide.hip): the layout of operands, and a tile of a product with
// a dense layer's end.
#pragma once

#include <type_traits>

#include "common.h"
#include "dense.h"
#include "half_parts.h"

namespace dopt {

typedef float v4f_any __attribute__((ext_vector_type(4), aligned(4)));
typedef int v4i __attribute__((ext_vector_type(4)));

constexpr int kBig = 256, kSmall = 128;   // sides of tiles
// Blocks of 16 steps that are added in one accumulator: 4096 steps.  The instruction rounds down what lies below its guard bits, so a long sum
// of one sign drifts, and every instruction rounds a sum that is longer by then.  Products of non-negative values, off by on average and
// in the root mean square, relative to the result: 4096 steps -1.2e-7 and 5.3e-7 (a library's fp32 product 8.4e-7), 17001 in one accumulator
// -5.0e-7 and 1.2e-6 (1.7e-6), in five passes -1.0e-7 and 2.6e-7.  (Where half of both operands is zero the fp32 instruction rounds half as often:
// 4096 steps 5.7e-7 and a library's 4.9e-7.)  A pass more costs some 2 % of a product.
constexpr size_t kPass = 256;
constexpr int kInf = 1 << 20, kNan = 1 << 21;   // in a row's shift: it holds infinities, NaN

struct Operand {
    const float *x;
    size_t rows, padded, K, steps;
    char *parts;
    int *shift;         // of each row: it is held times 2^shift
    unsigned *tops;     // of one that lies across: the largest magnitudes of its runs, [run][row]
    int runs;
    unsigned blocks;    // of a launch
};

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
// in a line.  Bound by memory: [8192 + 4096] rows of 4096 take 79 to 86 us, read twice, which the L2 does not shorten, 106.  Longer rows than
// the registers hold are read twice.  Padding and rows that are not finite become zeros.
// Rows from row0 on, to the operand's place `to` and on (both multiples of four).
constexpr int kUnits = 8;
__device__ __forceinline__ void split_rows(const Operand &o, size_t row0, size_t to)
{
    __shared__ unsigned tops[16][4];
    const size_t K = o.K, steps = o.steps;
    const int lane = threadIdx.x & 63, r = threadIdx.x >> 1 & 3, half = threadIdx.x & 1, waves = blockDim.x >> 6;
    const size_t stride = blockDim.x / 8, s0 = threadIdx.x / 8;
    const bool inside = row0 + r < o.rows;
    const float *const x = o.x + min(row0 + r, o.rows - 1) * K;
    v4f v[kUnits][2];
    unsigned top = 0;   // of the values' magnitudes as integers, whose order is theirs, infinity and NaN last
    // the loads of all places go out together, whatever lies behind the row's end; then the end is put right
    auto load = [&](size_t step, v4f *to) {
        const size_t k = min(step * 16 + half * 8, K - 8);
        to[0] = *(const v4f_any *)(x + k);
        to[1] = *(const v4f_any *)(x + k + 4);
    };
    auto end = [&](size_t step, v4f *of) {
        const size_t k = step * 16 + half * 8;
        if (k + 8 <= K) return;
        float t[8];
#pragma unroll
        for (int e = 0; e < 8; e++) t[e] = x[min(k + e, K - 1)];
#pragma unroll
        for (int e = 0; e < 8; e++) of[e / 4][e % 4] = k + e < K ? t[e] : 0.0f;
    };
    auto see = [&](const v4f *of) {
#pragma unroll
        for (int e = 0; e < 8; e++) top = max(top, magnitude(of[e / 4][e % 4]));
    };
#pragma unroll
    for (int i = 0; i < kUnits; i++)
        if (i * stride < steps) load(s0 + i * stride, v[i]);
#pragma unroll
    for (int i = 0; i < kUnits; i++)
        if (i * stride < steps) {
            if ((i + 1) * stride * 16 > K) end(s0 + i * stride, v[i]);
            see(v[i]);
        }
    for (size_t i = kUnits; i * stride < steps; i++) {
        v4f more[2];
        load(s0 + i * stride, more);
        end(s0 + i * stride, more);
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
    if (threadIdx.x < 8 && half == 0) o.shift[to + r] = shift;
    const bool live = inside && shift < kInf;
    auto put = [&](size_t step, const v4f *of) {
        if (step >= steps) return;
        float u[8];
#pragma unroll
        for (int e = 0; e < 8; e++) u[e] = live ? __builtin_ldexpf(of[e / 4][e % 4], shift) : 0.0f;
        store_parts(o.parts + ((to >> 5) * steps + step) * 2048, (int)(to & 31) + r, half, u);
    };
#pragma unroll
    for (int i = 0; i < kUnits; i++)
        if (i * stride < steps) put(s0 + i * stride, v[i]);
    for (size_t i = kUnits; i * stride < steps; i++) {
        v4f more[2];
        load(s0 + i * stride, more);
        end(s0 + i * stride, more);
        put(s0 + i * stride, more);
    }
}

// A tile of 64 steps by 64 columns, from (k0, c0) on, of an operand that lies across the reduction, [K][rows], turned in LDS.
__device__ __forceinline__ void turn_tile(const Operand &o, size_t c0, size_t k0)
{
    __shared__ float tile[64][65];
    __shared__ unsigned tops[4][64];
    const size_t K = o.K, steps = o.steps;
    const int c = threadIdx.x & 63, w = threadIdx.x >> 6;
    const size_t col = min(c0 + c, o.rows - 1);
    float v[16];
#pragma unroll
    for (int u = 0; u < 16; u++) v[u] = o.x[min(k0 + w + 4 * u, K - 1) * o.rows + col];
    unsigned top = 0;
#pragma unroll 8
    for (int i = w; i < o.runs; i += 4) top = max(top, o.tops[i * o.rows + col]);
    tops[w][c] = top;
    __syncthreads();
    const bool inside = c0 + c < o.rows;
    const int shift = inside ? shift_of(max(max(tops[0][c], tops[1][c]), max(tops[2][c], tops[3][c]))) : 0;
    if (k0 == 0 && w == 0) o.shift[c0 + c] = shift;
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
        store_parts(o.parts + ((c0 + r) / 32 * steps + step) * 2048, r & 31, half, p);
    }
}

struct Wide {
    size_t M, N, K, steps;
    const float *x, *w;
    size_t xm, xk, wn, wk;   // between rows, between steps
    const char *xp, *wp;
    const int *xs, *ws;
    float *y, *to;           // the result; the sums of splits, [split][M][N], where there are several
    char *waiting;           // each workgroup's sums between its passes
    unsigned tiles, mtiles, ntiles, splits;
};
// What is not finite in a tile's operands: the sums of those rows and columns as fp32 instructions make them.
template <int kTile>
__device__ __noinline__ void rough_sums(Wide q, DenseEpilogue ep, float *y, size_t m0, size_t n0, size_t from, size_t to, const int *shift)
{
    for (int i = threadIdx.x; i < kTile * kTile; i += 2 * kTile) {
        const size_t m = m0 + i / kTile, n = n0 + i % kTile;
        const int most = max(shift[i / kTile], shift[kTile + i % kTile]);
        if (m >= q.M || n >= q.N || most < kInf) continue;
        const bool nan = most == kNan;
        float s = nan ? __builtin_nanf("") : 0.0f;
        if (!nan)
            for (size_t k = from; k < to; k++) s += q.x[m * q.xm + k * q.xk] * q.w[n * q.wn + k * q.wk];
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

// A stage of 16 steps of both sides of a tile: a wavefront brings a row of blocks of each.
__device__ __forceinline__ void bring_both(const char *left, const char *right, int k, int w, int lane, int sides, char *to)
{
    bring(left + (size_t)k * 2048, 2, lane, to + w * 2048);
    bring(right + (size_t)k * 2048, 2, lane, to + sides + w * 2048);
}

// Tiles of 256 x 256 by eight wavefronts of 128 x 64: the accumulators are half of the registers, and a stage, 32 KB, feeds 24 matrix
// instructions of each.  The halves of the workgroup, which share the CU's four SIMDs, read and multiply in turn; three stages are on
// their way.  (Reading and multiplying together, between one barrier per stage, took 908 us where this takes 815.)
template <int>
__device__ __forceinline__ void sums(const char *left, const char *right, int steps, int w, int lane, char *lds, v16f (&acc)[4][2])
{
    const int wm = w >> 2, wn = w & 3;
    auto arrived = [&](int ahead) {   // all loads but those of the last `ahead` stages asked for
        if (ahead >= 2) settled<8>();
        else if (ahead == 1) settled<4>();
        else settled<0>();
    };
    for (int k = 0; k < min(steps, 3); k++) bring_both(left, right, k, w, lane, 16384, lds + k * 32768);
    arrived(min(steps, 3) - 1);
    phase();
    if (wm) phase();
    for (int k = 0; k < steps; k++) {
        Side<4> a;
        Side<2> b;
        const char *const now = lds + (k & 3) * 32768;
        a.read(now + wm * 8192, lane);
        b.read(now + 16384 + wn * 4096, lane);
        // (into the stage that the other half read before this phase)
        if (k + 3 < steps) bring_both(left, right, k + 3, w, lane, 16384, lds + ((k + 3) & 3) * 32768);
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
}

// Tiles of 128 x 128 by four of 64 x 64, two workgroups to a CU with five stages, three with three.
template <int kStages>
__device__ __forceinline__ void sums(const char *left, const char *right, int steps, int w, int lane, char *lds, v16f (&acc)[2][2])
{
    pipeline<kStages, 16384, 4, 2, 2>(
        lds, steps, [&](int k, char *to) { bring_both(left, right, k, w, lane, 8192, to); },
        [&](const char *now, Side<2> &a, Side<2> &b) {
            a.read(now + (w >> 1) * 4096, lane);
            b.read(now + 8192 + (w & 1) * 4096, lane);
        },
        [&](const Side<2> &a, const Side<2> &b) { multiply(a, b, acc); });
}

// Between two passes a wavefront's sums wait in memory, where each lane finds its own again.
template <int MI>
__device__ __forceinline__ void waiting_sums(v16f (&acc)[MI][2], char *at, bool add, bool put)
{
#pragma unroll
    for (int i = 0; i < MI; i++)
#pragma unroll
        for (int j = 0; j < 2; j++) {
            v4f *const to = (v4f *)at + (i * 2 + j) * 256;
            if (add) {
                v4f old[4];
#pragma unroll
                for (int g = 0; g < 4; g++) old[g] = to[g * 64];
#pragma unroll
                for (int e = 0; e < 16; e++) acc[i][j][e] += old[e >> 2][e & 3];
            }
            if (put) {
#pragma unroll
                for (int g = 0; g < 4; g++) to[g * 64] = v4f{acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
            }
        }
}

template <int kTile, int kStages = 5>
constexpr int kLdsOf = kTile == kBig ? 4 * 32768 : kStages * 16384;

// A tile (mt, nt) of a product, the blocks [from, to) of its reduction, to y.  place_of_tile: which place among those that wait is its.
// kPasses: some part of a reduction is longer than a pass.  (The loop by itself, with its registers, takes 1.6 % of both gradients of
// [1000 x 1777] from 1111 where it runs once.)
template <int kTile, bool kPasses, int kStages = 5>
__device__ __forceinline__ void wide_tile(const Wide &q, const DenseEpilogue &ep, float *y, unsigned mt, unsigned nt, size_t from, size_t to,
                                          unsigned place_of_tile, char *lds)
{
    constexpr int MI = kTile / 64, kBlocks = kTile / 32;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int wm = kTile == kBig ? w >> 2 : w >> 1, wn = kTile == kBig ? w & 3 : w & 1;
    const size_t row_of_blocks = q.steps * 2048;
    const char *const left = q.xp + (mt * kBlocks + w) * row_of_blocks, *const right = q.wp + (nt * kBlocks + w) * row_of_blocks;
    const size_t m0 = (size_t)mt * kTile, n0 = (size_t)nt * kTile;
    v16f acc[MI][2];
    if constexpr (kPasses) {
        const unsigned passes = (unsigned)((to - from + kPass - 1) / kPass);
        char *const waiting = q.waiting + ((size_t)place_of_tile * (kTile / 32) + w) * (MI * 8192) + lane * 16;
#pragma unroll 1
        for (unsigned pass = 0;; pass++) {
            const size_t at = from + (to - from) * pass / passes, next = from + (to - from) * (pass + 1) / passes;
            zero_acc(acc);
            sums<kStages>(left + at * 2048, right + at * 2048, (int)(next - at), w, lane, lds, acc);
            if (passes == 1) break;
            waiting_sums(acc, waiting, pass > 0, pass + 1 < passes);
            if (pass + 1 == passes) break;
        }
    } else {
        zero_acc(acc);
        sums<kStages>(left + from * 2048, right + from * 2048, (int)(to - from), w, lane, lds, acc);
    }

    int *const shift = (int *)lds;
    const int mine = threadIdx.x < kTile ? q.xs[m0 + threadIdx.x] : q.ws[n0 + threadIdx.x - kTile];
    shift[threadIdx.x] = mine;
    // (whether any is not finite; the library's vote over a workgroup has LDS of its own, which would leave a CU one of them)
    const bool some = __any(mine >= kInf);
    if (lane == 0) shift[2 * kTile + w] = some;
    meet();
    bool rough = false;
#pragma unroll
    for (int i = 0; i < kTile / 32; i++) rough = rough || shift[2 * kTile + i];
    rough = __builtin_amdgcn_readfirstlane(rough);
    // 32 rows at a time through LDS, so that a row's 64 values are stored by sixteen lanes
    float *const image = (float *)(lds + 2304) + w * (32 * 68);
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
    for (int i = 0; i < MI && left_col < q.N; i++) {
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
            for (int e = 0; e < 16; e++) image[(8 * (e >> 2) + 4 * (lane >> 5) + (e & 3)) * 68 + 32 * j + (lane & 31)] = acc[0][j][e];
        asm volatile("" ::: "memory");   // (a wavefront's LDS accesses stay in their order)
        const int r0 = wm * (kTile / 2) + i * 32 + (lane >> 4);
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
        for (int k = 0; k + 1 < MI; k++)
#pragma unroll
            for (int j = 0; j < 2; j++) acc[k][j] = acc[k + 1][j];
    }
    if (rough) rough_sums<kTile>(q, ep, y, m0, n0, from * 16, min(to * 16, q.K), shift);
}

}  // namespace dopt
