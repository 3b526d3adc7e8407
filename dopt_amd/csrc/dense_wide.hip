// Products of dense layers of middling and large sizes, forward and backward: both operands are laid out once as two fp16 parts and go to
// the matrix instruction from there, the layer's end rides in the product.
//
// Rows are scaled by powers of two, each to a largest value in [2^14, 2^15), so h + l is off by at most 2^-22 of a value or 2^-39 of
// the largest one of its row (fp16's last subnormal place).  l l is left out, 2^-22 of a product at most.  Together with sums in fp32
//     |error| <= (K 2^-24 + 2^-20) sum |x| |w| + 2^-38 K max |x row| max |w row|
// that is, fp32's own rounding of a long sum unless a row spans more than seventeen binary orders and its largest values meet zeros.
// Three bf16 parts, which sgemm.hip uses for operands of any kind, keep 24 bits and take twice the matrix work.
//
// Bound by the matrix instructions, 6 M N K operations, where tiles are large: [8192 x 4096] from 4096 steps, 824 GFLOP, takes 730 us, 79 of
// them for the layout (402 MB, 5.1 TB/s) and 660 for the product (1250 TFLOP/s; a library's bf16 product of 4096 cubed reaches 1157) - once the
// card's clock has settled: in the first thirty products after a pause it takes up to 880.
// The matrix instructions are busy 72 % of its cycles, at the clock that is left when they are.  With tiles of 128 x 128 the bound is
// what a CU takes in, some 45 GB/s whoever asks for it: both gradients of [1000 x 1777] from 1111 take 66 us, 33 of them for the
// products, 9 for dz, 17 for the layout and 8 to add parts.
#include <algorithm>
#include <type_traits>

#include "common.h"
#include "dense.h"
#include "half_parts.h"

namespace {

using namespace dopt;

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
constexpr int kUnits = 8;
__device__ __forceinline__ void split_rows(const Operand &o, unsigned block)
{
    __shared__ unsigned tops[16][4];
    const size_t row0 = (size_t)block * 4, K = o.K, steps = o.steps;
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
        load(s0 + i * stride, more);
        end(s0 + i * stride, more);
        put(s0 + i * stride, more);
    }
}

// Operands that lie across the reduction, [K][rows]: the largest values of runs of K for each column, then a tile of 64 steps by 64 columns
// per workgroup, turned in LDS.
constexpr int kRuns = 32, kAcross = 3;
struct Layout {
    Operand rows[2], across[kAcross];
    int nrows, nacross;
    DenseFold fold;   // rides behind them
};

__global__ __launch_bounds__(256) void wide_tops_k(Tops t) { column_tops(t, blockIdx.x); }

__device__ __forceinline__ void turn_tile(const Operand &o, unsigned block)
{
    __shared__ float tile[64][65];
    __shared__ unsigned tops[4][64];
    const unsigned tiles = (unsigned)(o.padded / 64);
    const size_t K = o.K, steps = o.steps, c0 = (size_t)(block % tiles) * 64, k0 = (size_t)(block / tiles) * 64;
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

__global__ __launch_bounds__(1024) void wide_layout_k(Layout l)
{
    unsigned block = blockIdx.x;
    for (int i = 0; i < l.nrows; i++) {
        if (block < l.rows[i].blocks) return split_rows(l.rows[i], block);
        block -= l.rows[i].blocks;
    }
    for (int i = 0; i < l.nacross; i++) {
        if (block < l.across[i].blocks) return turn_tile(l.across[i], block);
        block -= l.across[i].blocks;
    }
    dense_fold(l.fold, block);
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
struct Wides {
    Wide q[2];
    unsigned per[2];   // an XCD's workgroups of each
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

// Tiles of 128 x 128 by four of 64 x 64, two workgroups to a CU.
__device__ __forceinline__ void sums(const char *left, const char *right, int steps, int w, int lane, char *lds, v16f (&acc)[2][2])
{
    pipeline<5, 16384, 4, 2, 2>(
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

template <int kTile>
constexpr int kLdsOf = kTile == kBig ? 4 * 32768 : 5 * 16384;

// kPasses: some part of a reduction is longer than a pass.  (The loop by itself, with its registers, takes 1.6 % of both gradients of
// [1000 x 1777] from 1111 where it runs once.)
template <int kTile, bool kPasses>
__global__ __launch_bounds__(2 * kTile, 2) void wide_product_k(Wides both, DenseEpilogue ep)
{
    constexpr int MI = kTile / 64, kBlocks = kTile / 32;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    // an XCD takes an eighth of each product, side by side; the one with the longer reduction first
    const unsigned xcd = blockIdx.x & 7, place = blockIdx.x >> 3;
    const bool second = place >= both.per[0];
    const Wide q = both.q[second];
    unsigned id = second ? xcd * both.per[1] + place - both.per[0] : xcd * both.per[0] + place;
    if (id >= q.tiles * q.splits) return;
    const unsigned split = id / q.tiles, place_of_tile = id;
    id %= q.tiles;
    const size_t from = q.steps * split / q.splits, to = q.steps * (split + 1) / q.splits;
    float *const y = q.splits > 1 ? q.to + split * q.M * q.N : q.y;
    if (q.splits > 1) ep = DenseEpilogue{nullptr, nullptr, nullptr, DOPT_HIP_ACT_NONE, q.N};   // it rides in the sum over the splits
    // eight rows of tiles together, column by column: what an XCD works on at a time shares rows and columns
    const unsigned band = 8 * q.ntiles, first = id / band * 8, high = min(8u, q.mtiles - first);
    const unsigned mt = first + id % band % high, nt = id % band / high;
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
            sums(left + at * 2048, right + at * 2048, (int)(next - at), w, lane, lds, acc);
            if (passes == 1) break;
            waiting_sums(acc, waiting, pass > 0, pass + 1 < passes);
            if (pass + 1 == passes) break;
        }
    } else {
        zero_acc(acc);
        sums(left + from * 2048, right + from * 2048, (int)(to - from), w, lane, lds, acc);
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

// Adds the splits of up to two products and ends them, four values at a time; the last four end with the product, whatever of them the
// quad before has written too.  Bound by memory ([1000 x 1111] of three and [1777 x 1111] of two: 41 MB, 8 us).
__global__ __launch_bounds__(256) void wide_join_k(Wides both, DenseEpilogue ep)
{
    auto quads_of = [](const Wide &q) { return q.splits > 1 ? (q.M * q.N + 3) / 4 : 0; };
    const size_t n0 = quads_of(both.q[0]), n1 = quads_of(both.q[1]);
    with_activation(ep.act, [&](auto kind) {
        for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n0 + n1; i += (size_t)gridDim.x * 256) {
            const Wide &q = both.q[i >= n0];
            const size_t n = q.M * q.N, at = min(4 * (i >= n0 ? i - n0 : i), n - 4);
            v4f z = *(const v4f_any *)(q.to + at), o;
#pragma unroll 4
            for (unsigned p = 1; p < q.splits; p++) z += *(const v4f_any *)(q.to + p * n + at);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                if (ep.bias) z[e] += ep.bias[(at + e) % q.N];
                o[e] = act_value<kind.value>(z[e]);
            }
            if (ep.pre) *(v4f_any *)(ep.pre + at) = z;
            if (ep.residual) o += *(const v4f_any *)(ep.residual + at);
            *(v4f_any *)(q.y + at) = o;
        }
    });
}

// The side of the tiles that suit a product; 0: none here.  Large ones where they take a third of the chip's places; small ones from
// two gigaflops on, unless the reduction is more than twelve times as long as the shorter side.  us here and on three bf16 parts, large tiles with 128, 512
// and 1024 steps:
//     [1500 x 4096] 37 63 93 and 36 69 113    [4096 x 2500] 55 77 109 and 91 153 198    [4096 x 4097] 96 142 210 and 140 234 362
//     [8192 x 4096] 130 187 268 and 160 308 472
// small ones with 512, 1024 and 4096:
//     [1024 x 1024] 28 30 56 and 22 38 65    [2048 x 1024] 32 40 89 and 39 49 113    [1024 x 4096] 37 51 155 and 50 82 199
//     [256 x 4096] 29 33 76 and 21 39 69
int tile_for(size_t M, size_t N, size_t K)
{
    const size_t tiles = ceil_div(M, (size_t)kBig) * ceil_div(N, (size_t)kBig), rounds = ceil_div(tiles, (size_t)num_cus());
    if (K < 128 || std::max(M, N) > (size_t)1 << 24) return 0;
    if (M >= 512 && N >= 512 && M * N * 3 >= rounds * num_cus() * kBig * kBig) return kBig;
    return std::min(M, N) >= 256 && K <= 12 * std::min(M, N) && M * N * K >= (size_t)900000000 ? kSmall : 0;
}

template <int kTile, bool kPasses>
int launch_tiles(const Wides &both, const DenseEpilogue &e)
{
    static bool raised = false;
    if (!raised) DOPT_HIP_CHECK(hipFuncSetAttribute((const void *)wide_product_k<kTile, kPasses>, hipFuncAttributeMaxDynamicSharedMemorySize, kLdsOf<kTile>));
    raised = true;
    hipLaunchKernelGGL((wide_product_k<kTile, kPasses>), dim3(8 * (both.per[0] + both.per[1])), dim3(2 * kTile), kLdsOf<kTile>, stream(), both, e);
    DOPT_LAUNCH_CHECK();
    return DOPT_HIP_OK;
}

int launch_products(int tile, const Wide *q, int n, const DenseEpilogue &e)
{
    Wides both{{q[0], q[n - 1]}, {0, 0}};
    if (n == 2 && q[1].steps * q[0].splits > q[0].steps * q[1].splits) std::swap(both.q[0], both.q[1]);
    for (int i = 0; i < n; i++) both.per[i] = (unsigned)ceil_div((size_t)both.q[i].tiles * both.q[i].splits, (size_t)8);
    const bool passes = q[0].waiting || q[n - 1].waiting;
    int rc;
    if (tile == kBig) rc = passes ? launch_tiles<kBig, true>(both, e) : launch_tiles<kBig, false>(both, e);
    else rc = passes ? launch_tiles<kSmall, true>(both, e) : launch_tiles<kSmall, false>(both, e);
    if (rc) return rc;
    if (n == 1) both.q[1].splits = 1;
    size_t values = 0;
    for (const Wide &p : both.q) values += p.splits > 1 ? p.M * p.N : 0;
    if (!values) return DOPT_HIP_OK;
    hipLaunchKernelGGL(wide_join_k, dim3((unsigned)std::min(ceil_div(values, (size_t)1024), (size_t)num_cus() * 16)), dim3(256), 0, stream(), both, e);
    DOPT_LAUNCH_CHECK();
    return DOPT_HIP_OK;
}

// Into how many parts the reductions of products in tiles of 128 x 128 are cut.  A stage takes 0.4 us where a CU has one workgroup, two
// of them 0.6; the sums of parts are written and read at about 6 TB/s, and adding them is a launch.  ([1024 x 1024] from 4096
// steps in eight parts 56 us, in one 112; [2048 x 2048] from 512 steps in two 47, in one 36.)
void cut(const WideProduct *p, int n, unsigned *splits)
{
    size_t stages[2] = {0, 0}, tiles[2] = {0, 0};
    unsigned now[2] = {1, 1};
    for (int i = 0; i < n; i++) {
        splits[i] = 1;
        if (tile_for(p[i].M, p[i].N, p[i].K) != kSmall) continue;
        stages[i] = ceil_div(p[i].K, (size_t)16);
        tiles[i] = ceil_div(p[i].M, (size_t)kSmall) * ceil_div(p[i].N, (size_t)kSmall);
    }
    double least = 0.0;
    for (;;) {   // the longest one is cut further
        size_t blocks = 0, longest = 0, bytes = 0;
        for (int i = 0; i < n; i++) {
            blocks += tiles[i] * now[i];
            longest = std::max(longest, ceil_div(stages[i], (size_t)now[i]));
            bytes += now[i] > 1 ? (2 * now[i] + 1) * p[i].M * p[i].N * sizeof(float) : 0;
        }
        const double us = (double)longest * (blocks <= (size_t)num_cus() ? 0.4 : 0.6 * (double)ceil_div(blocks, (size_t)num_cus() * 2)) +
                          (bytes ? 5.0 + (double)bytes / 6e6 : 0.0);
        if (least == 0.0 || us < least) {
            least = us;
            for (int i = 0; i < n; i++) splits[i] = now[i];
        }
        const int i = n == 2 && stages[1] * now[0] > stages[0] * now[1];
        if (blocks + tiles[i] > (size_t)num_cus() * 2 || stages[i] < (size_t)16 * (now[i] + 1)) return;
        now[i]++;
    }
}

// The launches of up to two products, in scratch from `to` on.
struct Plan {
    Layout l{};
    Tops tops{};
    Wide q[2];
    int tile[2];
    unsigned *callers = nullptr;   // largest magnitudes that the caller finds
    unsigned row_blocks = 0, blocks = 0;
    size_t longest = 0, bytes = 0;
};
Plan arrange(const WideProduct *p, int n, char *const scratch)
{
    Plan r;
    auto take = [&](size_t bytes) {
        char *const at = scratch ? scratch + r.bytes : nullptr;   // (null: for the size alone)
        r.bytes += ceil_div(bytes, (size_t)256) * 256;
        return at;
    };
    unsigned splits[2];
    cut(p, n, splits);
    for (int i = 0; i < n; i++) {
        const WideProduct &g = p[i];
        const size_t tile = r.tile[i] = tile_for(g.M, g.N, g.K), steps = ceil_div(g.K, (size_t)16);
        Operand sides[2];
        for (int k = 0; k < 2; k++) {
            const WideSide &side = k ? g.w : g.x;
            const size_t rows = k ? g.N : g.M, padded = ceil_div(rows, tile) * tile;
            Operand &o = sides[k] = Operand{side.values, rows, padded, g.K, steps, nullptr, nullptr, nullptr, 0, 0};
            o.parts = take(padded * steps * 64);
            o.shift = (int *)take(padded * sizeof(int));
            if (!side.across) {
                o.blocks = (unsigned)(padded / 4);
                r.row_blocks += o.blocks;
                r.longest = std::max(r.longest, steps);
                r.l.rows[r.l.nrows++] = o;
                continue;
            }
            o.runs = side.runs ? side.runs : (int)std::min((size_t)kRuns, ceil_div(g.K, (size_t)64));
            o.tops = (unsigned *)take(o.runs * rows * sizeof(unsigned));
            if (side.runs) {
                r.callers = o.tops;
            } else {
                const unsigned blocks = (unsigned)(ceil_div(rows, (size_t)256) * o.runs);
                r.tops.o[r.tops.n++] = Tops::One{o.x, rows, g.K, o.tops, o.runs, blocks};
                r.tops.blocks += blocks;
            }
            o.blocks = (unsigned)(padded / 64 * ceil_div(steps, (size_t)4));
            r.blocks += o.blocks;
            r.l.across[r.l.nacross++] = o;
        }
        float *const partial = splits[i] > 1 ? (float *)take(splits[i] * g.M * g.N * sizeof(float)) : nullptr;
        const size_t waits = ceil_div(steps, (size_t)splits[i]) > kPass ? splits[i] * sides[0].padded * sides[1].padded * sizeof(float) : 0;
        char *const waiting = waits ? take(waits) : nullptr;
        const unsigned mt = (unsigned)(sides[0].padded / tile), nt = (unsigned)(sides[1].padded / tile);
        r.q[i] = Wide{g.M, g.N, g.K, steps, g.x.values, g.w.values, g.x.across ? 1 : g.K, g.x.across ? g.M : 1, g.w.across ? 1 : g.K, g.w.across ? g.N : 1,
                      sides[0].parts, sides[1].parts, sides[0].shift, sides[1].shift, g.y, partial, waiting, mt * nt, mt, nt, splits[i]};
    }
    return r;
}

}  // namespace

namespace dopt {

bool dense_wide_takes(size_t M, size_t N, size_t K) { return tile_for(M, N, K) != 0; }

size_t dense_wide_scratch(const WideProduct *p, int n) { return arrange(p, n, nullptr).bytes; }

unsigned *dense_wide_tops(const WideProduct *p, int n, char *scratch, Tops *others)
{
    const Plan plan = arrange(p, n, scratch);
    *others = plan.tops;
    return plan.callers;
}

int dense_wide(const WideProduct *p, int n, const DenseEpilogue &e, const DenseFold &fold, bool found)
{
    char *const scratch = (char *)workspace(dense_wide_scratch(p, n));
    if (!scratch) return DOPT_HIP_ERR_OOM;
    Plan plan = arrange(p, n, scratch);
    Layout &l = plan.l;
    if (plan.tops.n && !found) {
        hipLaunchKernelGGL(wide_tops_k, dim3(plan.tops.blocks), dim3(256), 0, stream(), plan.tops);
        DOPT_LAUNCH_CHECK();
    }
    l.fold = fold;
    unsigned rows = plan.row_blocks, blocks = plan.blocks + (fold.dbias ? (unsigned)ceil_div(fold.N, (size_t)8) : 0);
    const unsigned threads = plan.longest > 512 ? 1024 : plan.longest > 256 ? 512 : 256;   // rows in registers up to 16384 steps
    if (threads > 256) {   // by themselves
        Layout alone = l;
        alone.nacross = 0;
        hipLaunchKernelGGL(wide_layout_k, dim3(rows), dim3(threads), 0, stream(), alone);
        DOPT_LAUNCH_CHECK();
        l.nrows = 0;
        rows = 0;
    }
    if (rows + blocks) {
        hipLaunchKernelGGL(wide_layout_k, dim3(rows + blocks), dim3(256), 0, stream(), l);
        DOPT_LAUNCH_CHECK();
    }
    if (n == 2 && plan.tile[0] == plan.tile[1]) return launch_products(plan.tile[0], plan.q, 2, e);
    for (int i = 0; i < n; i++)
        if (int rc = launch_products(plan.tile[i], plan.q + i, 1, e)) return rc;
    return DOPT_HIP_OK;
}

}  // namespace dopt
