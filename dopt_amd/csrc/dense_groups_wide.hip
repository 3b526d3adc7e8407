// Large products of dense layers of groups: operands are laid out once as two scaled fp16 parts, as dense_wide.hip's, and go to the matrix
// instruction from there.  Error and scales as there: row by row of x and w forward, of dz and by the columns of w_g for dx, by a
// group's columns of dz and x for dw.
//
// Rows of a group are laid out from a tile's boundary on, so that a tile holds rows of one group; the steps of dw's reductions from a boundary of
// 64 rows on.  How many tiles there are is found on the device: an XCD takes an eighth of them, side by side.
//
// Bound by the matrix instructions and, for the layouts, by memory.  Sixteen groups, [16384 x 4096] from 2048: the layout 259 us (1.34 GB, 5.2 TB/s), the
// product 772 (356 TFLOP/s; of every group's last tile a part is empty).  Gradients of eight groups, [8192 x 4096] from 1024: dz, its sums and the largest values
// 112, layouts 180 (both at memory's rate), both products 373.  [4096 x 2048] from 512, eight groups: 19 and 46, the latter with 576 tiles of
// 128 x 128 that all end, and write 67 MB, at about one time.
#include <algorithm>
#include <cmath>

#include "dense_groups.h"
#include "dense_wide.h"

namespace {

using namespace dopt;

constexpr int kStepShift = 6;   // rows of a tile of the turned operands' layout
constexpr Units kRests{31, true, true};   // a unit for each group, and for the rows in front of them and behind

// A group that these offsets leave empty, whatever came before (others may be empty as well).
__device__ __forceinline__ bool surely_empty(const Groups &q, unsigned g) { return q.offsets[g + 1] <= q.offsets[g]; }

// ------------------------------------------------------------------------------------------------ columns: dz, sums, largest magnitudes

// 256 columns of a run of rows: of 2^shift rows of a group, or of 256 rows of a group's w.  Of dy and pre dz, its sums and its largest
// magnitudes; of x and w the magnitudes.  A lane has four columns, a wavefront every fourth row; the last four columns end with the matrix, whatever of
// them other lanes form as well, to the same bits.  Bound by memory.
struct Columns {
    const float *x, *pre;
    float *dz, *sums;
    unsigned *tops;
    int cols, act;
    unsigned tiles, runs;   // runs: of a group's w, 0 for rows
    unsigned blocks;
};
struct ColumnJobs {
    Columns j[3];
    int n, shift, w_rows;
};
constexpr int kWeightRun = 256;
constexpr unsigned kColumnsRow = 1u << 22;   // workgroups of a row of the grid

__global__ __launch_bounds__(256) void groups_columns_k(Groups q, ColumnJobs jobs)
{
    __shared__ v4f_any red_sum[4][64];
    __shared__ unsigned red_top[4][64][4];
    unsigned block = blockIdx.y * kColumnsRow + blockIdx.x;
    int which = 0;
    while (which + 1 < jobs.n && block >= jobs.j[which].blocks) block -= jobs.j[which++].blocks;
    const Columns &j = jobs.j[which];
    if (block >= j.blocks) return;   // (behind the end of the grid's last row)
    const unsigned unit = block / j.tiles;
    const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
    const int c = min((int)(block % j.tiles) * 256 + 4 * lane, j.cols - 4);
    size_t row;
    int rows;
    if (j.runs) {
        const unsigned g = unit / j.runs, first = unit % j.runs * kWeightRun;
        if (surely_empty(q, g)) return;
        row = (size_t)g * jobs.w_rows + first;
        rows = min(kWeightRun, jobs.w_rows - (int)first);
    } else {
        const Segment s = find_unit<false>(q, jobs.shift, unit);
        if (s.group < 0) return;
        row = s.begin + ((size_t)s.unit << jobs.shift);
        rows = (int)min((size_t)s.end - row, (size_t)1 << jobs.shift);
    }
    const size_t pitch = (size_t)j.cols, at = row * pitch + c;
    float all[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    unsigned top[4] = {0, 0, 0, 0};
    with_activation(j.act, [&](auto kind) {
        constexpr bool kPlain = decltype(kind)::value == DOPT_HIP_ACT_NONE;
        float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        auto one = [&](const v4f_any &d, const v4f_any &z, size_t i) {
            v4f_any o;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float v = act_grad<kind.value>(d[e], z[e]);
                o[e] = v;
                sum[e] += v;
                top[e] = max(top[e], magnitude(v));
            }
            if (!kPlain && j.dz) *(v4f_any *)(j.dz + i) = o;
        };
        int r = wave;
        for (; r + 12 < rows; r += 16) {
            if ((r & 255) < 4) {   // sums of 64 values each
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    all[e] += sum[e];
                    sum[e] = 0.0f;
                }
            }
            v4f_any d[4], z[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                d[i] = *(const v4f_any *)(j.x + at + (r + 4 * i) * pitch);
                if (!kPlain) z[i] = *(const v4f_any *)(j.pre + at + (r + 4 * i) * pitch);
            }
#pragma unroll
            for (int i = 0; i < 4; i++) one(d[i], kPlain ? d[i] : z[i], at + (r + 4 * i) * pitch);
        }
        for (; r < rows; r += 4) {
            const v4f_any d = *(const v4f_any *)(j.x + at + r * pitch);
            one(d, kPlain ? d : *(const v4f_any *)(j.pre + at + r * pitch), at + r * pitch);
        }
#pragma unroll
        for (int e = 0; e < 4; e++) all[e] += sum[e];
    });
    red_sum[wave][lane] = v4f_any{all[0], all[1], all[2], all[3]};
#pragma unroll
    for (int e = 0; e < 4; e++) red_top[wave][lane][e] = top[e];
    __syncthreads();
    if (wave) return;
    const size_t to = (size_t)unit * pitch + c;
    if (j.sums) *(v4f_any *)(j.sums + to) = (red_sum[0][lane] + red_sum[1][lane]) + (red_sum[2][lane] + red_sum[3][lane]);
    if (j.tops) {
#pragma unroll
        for (int e = 0; e < 4; e++)
            j.tops[to + e] = max(max(red_top[0][lane][e], red_top[1][lane][e]), max(red_top[2][lane][e], red_top[3][lane][e]));
    }
}

// ------------------------------------------------------------------------------------------------ layouts

// Rows of groups, each group from a tile's boundary on.
struct RowsJob {
    const float *x;
    size_t K, steps;
    char *parts;
    int *shift;
    int tile_shift;
    unsigned blocks;
};
// Rows of each group's w.
struct WeightsJob {
    const float *x;
    size_t rows, padded, K, steps;
    char *parts;
    int *shift;
    unsigned blocks;
};
// Each group's w across, [K][rows].
struct WeightsAcross {
    const float *x;
    size_t rows, padded, K, steps;
    char *parts;
    int *shift;
    unsigned *tops;
    int runs;
    unsigned blocks;
};
// Rows of groups across: columns of x, over a group's rows.
struct RowsAcross {
    const float *x;
    size_t rows, padded;   // columns
    char *parts;
    int *shift;
    unsigned *tops;
    int run_shift;
    unsigned blocks;
};
struct GroupLayout {
    RowsJob rows;
    WeightsJob weights;
    WeightsAcross turned;
    RowsAcross across[2];
    // dbias of runs of 2^fold_shift rows, 32 columns to a block
    const float *sums;
    float *dbias;
    int columns, fold_shift;
    unsigned fold_tiles, fold_blocks;
    // rows of no group, of up to two results: cleared by so many blocks
    float *rest[2];
    size_t rest_cols[2];
    unsigned rest_blocks;
};

__device__ __forceinline__ void clear_rest(const Groups &q, float *p, size_t cols, unsigned block, unsigned blocks)
{
    if (!p) return;
    const Segment front = find_unit<kRests.rest, kRests.all>(q, kRests.shift, 0), back = find_unit<kRests.rest, kRests.all>(q, kRests.shift, q.G + 1);
    const size_t first = front.end, n = first + (back.end - back.begin);
    for (size_t i = (size_t)block * blockDim.x + threadIdx.x; i < n * cols; i += (size_t)blocks * blockDim.x)
        p[i < first * cols ? i : i + (back.begin - first) * cols] = 0.0f;
}

__global__ __launch_bounds__(1024) void groups_layout_k(Groups q, GroupLayout l)
{
    unsigned block = blockIdx.x;
    if (block < l.rows.blocks) {
        const RowsJob &j = l.rows;
        const size_t place = (size_t)block * 4;
        const Segment s = find_unit<false>(q, j.tile_shift, (unsigned)(place >> j.tile_shift));
        if (s.group < 0) return;
        const size_t row = ((size_t)s.unit << j.tile_shift) + (place & (((size_t)1 << j.tile_shift) - 1)), rows = s.end - s.begin;
        if (row >= rows) {   // what is multiplied from here on is not stored
            if (threadIdx.x < 4) j.shift[place + threadIdx.x] = 0;
            return;
        }
        const Operand o{j.x + s.begin * j.K, rows, 0, j.K, j.steps, j.parts, j.shift, nullptr, 0, 0};
        return split_rows(o, row, place);
    }
    block -= l.rows.blocks;
    if (block < l.weights.blocks) {
        const WeightsJob &j = l.weights;
        const unsigned of_group = (unsigned)(j.padded / 4), g = block / of_group;
        const size_t row = (size_t)(block % of_group) * 4, place = (size_t)g * j.padded + row;
        if (surely_empty(q, g)) return;
        if (row >= j.rows) {
            if (threadIdx.x < 4) j.shift[place + threadIdx.x] = 0;
            return;
        }
        const Operand o{j.x + g * j.rows * j.K, j.rows, 0, j.K, j.steps, j.parts, j.shift, nullptr, 0, 0};
        return split_rows(o, row, place);
    }
    block -= l.weights.blocks;
    if (block < l.turned.blocks) {
        const WeightsAcross &j = l.turned;
        const unsigned tiles = (unsigned)(j.padded / 64), of_group = tiles * (unsigned)((j.steps + 3) / 4), g = block / of_group, t = block % of_group;
        if (surely_empty(q, g)) return;
        const Operand o{j.x + g * j.rows * j.K, j.rows, j.padded, j.K, j.steps, j.parts + g * (j.padded / 32) * j.steps * 2048, j.shift + g * j.padded,
                        j.tops + (size_t)g * j.runs * j.rows, j.runs, 0};
        return turn_tile(o, (size_t)(t % tiles) * 64, (size_t)(t / tiles) * 64);
    }
    block -= l.turned.blocks;
    for (int i = 0; i < 2; i++) {
        const RowsAcross &j = l.across[i];
        if (block >= j.blocks) {
            block -= j.blocks;
            continue;
        }
        const unsigned tiles = (unsigned)(j.padded / 64);
        const Segment s = find_unit<false>(q, kStepShift, block / tiles);
        if (s.group < 0) return;
        const size_t K = s.end - s.begin, units = (K + 63) >> 6;
        const unsigned first_run = j.run_shift == kStepShift ? s.first : find_group(q, j.run_shift, (unsigned)s.group).first;
        const Operand o{j.x + s.begin * j.rows, j.rows, j.padded, K, 4 * units, j.parts + (j.padded / 32) * 4 * s.first * 2048, j.shift + s.group * j.padded,
                        j.tops + (size_t)first_run * j.rows, (int)((K + ((size_t)1 << j.run_shift) - 1) >> j.run_shift), 0};
        return turn_tile(o, (size_t)(block % tiles) * 64, (size_t)s.unit * 64);
    }
    if (block < l.fold_blocks) {
        __shared__ float red[8][33];
        return fold_runs(GroupLayer{q, l.columns, 0}, l.fold_shift, l.sums, l.dbias, block % l.fold_tiles, block / l.fold_tiles, 8, red);
    }
    block -= l.fold_blocks;
    for (int i = 0; i < 2; i++) clear_rest(q, l.rest[i], l.rest_cols[i], block, l.rest_blocks);
}

// ------------------------------------------------------------------------------------------------ products

// Rows of groups times each group's matrix: y [M, N] from x and w (forward), dx [M, K] from dz and w across.
struct RowsProduct {
    const float *x, *w;
    size_t N, K, steps, padded;   // columns of the result, its reduction, the matrix' padded columns
    size_t wn, wk;                // between its columns, between steps
    const char *xp, *wp;
    const int *xs, *ws;
    float *y;
    char *waiting;
    unsigned ntiles;
};
// dw from dz and x across.
struct WeightsProduct {
    const float *dz, *x;
    size_t N, K, dz_padded, x_padded;
    const char *dzp, *xp;
    const int *dzs, *xs;
    float *dw, *parts;       // parts: of several for a group, a matrix each, where that is not null
    char *waiting;
    unsigned mtiles, ntiles;
    int part_shift;          // of 2^part_shift rows
};
struct GroupProducts {
    RowsProduct rows;
    WeightsProduct weights;
    const float *bias;
    float *pre;
    int act;
    unsigned rows_per, weights_per;   // an XCD's workgroups of each, at most
};

template <int kTile, bool kPasses>
__global__ __launch_bounds__(2 * kTile, 2) void groups_product_k(Groups q, GroupProducts p)
{
    constexpr int kShift = kTile == kBig ? 8 : 7, kStages = 3;   // three workgroups of 128 x 128 to a CU: their numbers are rarely even
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const unsigned xcd = blockIdx.x & 7, place = blockIdx.x >> 3;
    if (place < p.rows_per) {
        const RowsProduct &r = p.rows;
        const unsigned mtiles = count_units<false>(q, kShift), tiles = mtiles * r.ntiles, per = (tiles + 7) / 8, id = xcd * per + place;
        if (place >= per || id >= tiles) return;
        // eight rows of tiles together, column by column: what an XCD works on at a time shares rows and columns
        const unsigned band = 8 * r.ntiles, first = id / band * 8, high = min(8u, mtiles - first);
        const unsigned t = first + id % band % high, nt = id % band / high;
        const Segment s = find_unit<false>(q, kShift, t);
        const size_t begin = s.begin, g = (size_t)s.group;
        const Wide z{s.end - begin, r.N, r.K, r.steps, r.x + begin * r.K, r.w + g * r.N * r.K, r.K, 1, r.wn, r.wk,
                     r.xp + (size_t)s.first * (kTile / 32) * r.steps * 2048, r.wp + g * (r.padded / 32) * r.steps * 2048, r.xs + (size_t)s.first * kTile,
                     r.ws + g * r.padded, nullptr, nullptr, r.waiting, 0, 0, 0, 1};
        const DenseEpilogue ep{p.bias ? p.bias + g * r.N : nullptr, nullptr, p.pre ? p.pre + begin * r.N : nullptr, p.act, r.N};
        wide_tile<kTile, kPasses, kStages>(z, ep, r.y + begin * r.N, s.unit, nt, 0, r.steps, id, lds);
        return;
    }
    const WeightsProduct &r = p.weights;
    const unsigned tiles = r.mtiles * r.ntiles, of_xcd = (tiles + 7) / 8, at = place - p.rows_per, item = at / of_xcd, tile = xcd * of_xcd + at % of_xcd;
    if (tile >= tiles) return;
    const unsigned mt = tile % r.mtiles, nt = tile / r.mtiles;
    unsigned group = item, part = 0;
    if (r.parts) {
        const Segment of = find_unit<false, true>(q, r.part_shift, item);
        if (of.group < 0) return;
        group = (unsigned)of.group;
        part = of.unit;
    }
    if (group >= q.G) return;
    const Segment s = find_group(q, kStepShift, group);
    const size_t g = group;
    float *const dw = r.parts ? r.parts + (size_t)item * r.N * r.K : r.dw + g * r.N * r.K;
    const size_t rows = s.end - s.begin;
    if (rows == 0) {
        const size_t m0 = (size_t)mt * kTile, n0 = (size_t)nt * kTile;
        for (int i = threadIdx.x; i < kTile * kTile; i += 2 * kTile)
            if (m0 + i / kTile < r.N && n0 + i % kTile < r.K) dw[(m0 + i / kTile) * r.K + n0 + i % kTile] = 0.0f;
        return;
    }
    const size_t steps = 4 * (size_t)s.unit, block = 4 * (size_t)s.first * 2048;
    const Wide z{r.N, r.K, rows, steps, r.dz + (size_t)s.begin * r.N, r.x + (size_t)s.begin * r.K, 1, r.N, 1, r.K,
                 r.dzp + (r.dz_padded / 32) * block, r.xp + (r.x_padded / 32) * block, r.dzs + g * r.dz_padded, r.xs + g * r.x_padded, nullptr, nullptr,
                 r.waiting, 0, 0, 0, 1};
    size_t from = 0, to = steps;
    if (r.parts) {
        from = (size_t)part << (r.part_shift - 4);
        to = min(steps, from + ((size_t)1 << (r.part_shift - 4)));
    }
    wide_tile<kTile, kPasses, kStages>(z, DenseEpilogue{nullptr, nullptr, nullptr, DOPT_HIP_ACT_NONE, r.K}, dw, mt, nt, from, to, item * tiles + tile, lds);
}

// ------------------------------------------------------------------------------------------------ the host's side

size_t padded_to(size_t n, size_t tile) { return ceil_div(n, tile) * tile; }

// Places in scratch, taken one after the other; without a base their size.
struct Scratch {
    char *base;
    size_t bytes = 0;
    template <class T = char>
    T *take(size_t n)
    {
        char *const at = base ? base + bytes : nullptr;
        bytes += ceil_div(n * sizeof(T), (size_t)256) * 256;
        return (T *)at;
    }
};

template <int kTile, bool kPasses>
int launch_tiles(const Groups &q, const GroupProducts &p)
{
    static bool raised = false;
    constexpr int lds = kLdsOf<kTile, 3>;
    const auto kernel = groups_product_k<kTile, kPasses>;
    if (!raised) DOPT_HIP_CHECK(hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds));
    raised = true;
    hipLaunchKernelGGL(kernel, dim3(8 * (p.rows_per + p.weights_per)), dim3(2 * kTile), lds, stream(), q, p);
    DOPT_LAUNCH_CHECK();
    return DOPT_HIP_OK;
}
int launch_products(const Groups &q, size_t tile, bool passes, const GroupProducts &p)
{
    if (tile == kBig) return passes ? launch_tiles<kBig, true>(q, p) : launch_tiles<kBig, false>(q, p);
    return passes ? launch_tiles<kSmall, true>(q, p) : launch_tiles<kSmall, false>(q, p);
}

// A row of workgroups has fewer than 2^32 threads.
void launch_columns(const Groups &q, const ColumnJobs &jobs, size_t blocks)
{
    const dim3 grid((unsigned)std::min(blocks, (size_t)kColumnsRow), (unsigned)ceil_div(blocks, (size_t)kColumnsRow));
    hipLaunchKernelGGL(groups_columns_k, grid, dim3(256), 0, stream(), q, jobs);
}

int shift_of_tile(size_t tile) { return tile == kBig ? 8 : 7; }

// Threads of a workgroup that lays out rows of so many steps: in registers up to 1024.
unsigned row_threads(size_t steps) { return steps > 512 ? 1024 : steps > 256 ? 512 : 256; }

// The side of the tiles: large ones for the largest products, of long groups (sixteen groups, [16384 x 4096] from 2048 steps: 1020 us, with small
// ones 1035; four groups, [16384 x 1024] from 512: 133 and 106, gradients 279 and 285).
size_t tile_for(size_t G, size_t M, size_t N, size_t K)
{
    const size_t tiles = (ceil_div(M, (size_t)kBig) + G / 2) * ceil_div(N, (size_t)kBig);
    return M >= 512 * G && M * N * K >= (size_t)30000000000 && tiles >= (size_t)num_cus() / 2 ? kBig : kSmall;
}

}  // namespace

namespace dopt {

int groups_dz(const GroupLayer &l, int act, int shift, const float *dy, const float *pre, float *dz, float *sums)
{
    ColumnJobs jobs{};
    const unsigned tiles = (unsigned)ceil_div((size_t)l.N, (size_t)256);
    const size_t blocks = tiles * most_units(l.q.M, l.q.G, shift);
    DOPT_REQUIRE(blocks < ((size_t)1 << 32), "dopt_hip_dense_groups_grad: dimensions too large");
    jobs.j[0] = Columns{dy, pre, dz, sums, nullptr, l.N, act, tiles, 0, (unsigned)blocks};
    jobs.n = 1;
    jobs.shift = shift;
    launch_columns(l.q, jobs, blocks);
    DOPT_LAUNCH_CHECK();
    return DOPT_HIP_OK;
}

// A launch has fewer than 2^32 threads: the layouts' rows are four to a workgroup of at most 1024.
static bool fits(size_t G, size_t M, size_t N, size_t K)
{
    const size_t most = (size_t)1 << 23;
    return M + kBig * G < most && G * (N + K + 2 * kBig) < most && M / 64 * (ceil_div(N, (size_t)64) + ceil_div(K, (size_t)64)) < most &&
           G * ceil_div(N, (size_t)64) * ceil_div(K, (size_t)64) < most;
}
// Launches, every byte that the layouts move, and the matrix instructions over whole tiles (half of one more for each group).
double groups_wide_us(size_t G, size_t M, size_t N, size_t K)
{
    if (K < 128 || N < 128 || !fits(G, M, N, K)) return HUGE_VAL;
    const double m = (double)M, weights = (double)G * N * K;
    return 29 + 8 * (m * K + weights) / 5e6 + 6 * (m + 64.0 * G) * N * K / 1.2e9;
}
double groups_wide_grad_us(size_t G, size_t M, size_t N, size_t K)
{
    if (K < 128 || N < 128 || !fits(G, M, N, K)) return HUGE_VAL;
    const double m = (double)M, weights = (double)G * N * K;
    return 32.7 + 1e-6 * (9.9 * m * N + 4.5 * m * K + 3.9 * weights) + 3.5e-9 * (m + 64.0 * G) * N * K;
}

int groups_wide(GroupLayer l, const float *x, const float *w, const float *bias, int act, float *y, float *pre)
{
    const size_t G = l.q.G, M = l.q.M, N = l.N, K = l.K, steps = ceil_div(K, (size_t)16), tile = tile_for(G, M, N, K);
    const size_t mtiles = most_units(M, G, shift_of_tile(tile)), rows = mtiles * tile, padded = padded_to(N, tile), ntiles = padded / tile;
    const bool passes = steps > kPass;
    GroupLayout lay{};
    GroupProducts p{};
    auto plan = [&](Scratch s) {
        lay.rows = RowsJob{x, K, steps, s.take(rows * steps * 64), s.take<int>(rows), shift_of_tile(tile), (unsigned)(rows / 4)};
        lay.weights = WeightsJob{w, N, padded, K, steps, s.take(G * padded * steps * 64), s.take<int>(G * padded), (unsigned)(G * padded / 4)};
        p.rows = RowsProduct{x, w, N, K, steps, padded, K, 1, lay.rows.parts, lay.weights.parts, lay.rows.shift, lay.weights.shift, y,
                             passes ? s.take(mtiles * ntiles * tile * tile * 4) : nullptr, (unsigned)ntiles};
        return s.bytes;
    };
    char *scratch;
    if (int rc = groups_scratch(&l.q, {Units{shift_of_tile(tile), false, false}, kRests}, plan(Scratch{nullptr}), &scratch)) return rc;
    plan(Scratch{scratch});
    lay.rest[0] = y;
    lay.rest[1] = pre;
    lay.rest_cols[0] = lay.rest_cols[1] = N;
    lay.rest_blocks = (unsigned)num_cus();
    p.bias = bias;
    p.pre = pre;
    p.act = act;
    p.rows_per = (unsigned)ceil_div(mtiles * ntiles, (size_t)8);
    const unsigned threads = steps <= 128 ? 128 : row_threads(steps);   // (fewer wavefronts with more in flight: 4096 rows of 512 15.4 us, with 256 threads 18.8)
    hipLaunchKernelGGL(groups_layout_k, dim3(lay.rows.blocks + lay.weights.blocks + lay.rest_blocks), dim3(threads), 0, stream(), l.q, lay);
    DOPT_LAUNCH_CHECK();
    return launch_products(l.q, tile, passes, p);
}

int groups_wide_grad(GroupLayer l, int act, const float *dy, const float *pre, const float *x, const float *w, float *dx, float *dw, float *dbias)
{
    const size_t G = l.q.G, M = l.q.M, N = l.N, K = l.K, steps = ceil_div(N, (size_t)16);
    const size_t tile = dw && G * ceil_div(N, (size_t)kBig) * ceil_div(K, (size_t)kBig) < (size_t)num_cus() ? (size_t)kSmall : tile_for(G, M, K, N);
    const size_t mtiles = most_units(M, G, shift_of_tile(tile)), rows = mtiles * tile, padded_n = padded_to(N, tile), padded_k = padded_to(K, tile);
    const size_t ktiles = padded_k / tile, wtiles = padded_n / tile * ktiles, units = most_units(M, G, kStepShift);
    int shift = kStepShift;   // rows of a run of sums and largest magnitudes: every tile of a turned layout reads all of a group's
    while ((M / G >> shift) > 64) shift++;
    const size_t runs = most_units(M, G, shift), w_runs = ceil_div(N, (size_t)kWeightRun);
    // Few tiles of dw: a group's reduction in parts, whose matrices are written and read once more.
    int part_shift = 13;
    while (part_shift > 8 && most_units(M, G, part_shift) * wtiles < (size_t)num_cus() * (tile == kBig ? 1 : 2)) part_shift--;
    const bool parted = dw && G * wtiles * 2 < (size_t)num_cus() * (tile == kBig ? 1 : 2) && M > (size_t)1 << part_shift;
    const size_t items = parted ? most_units(M, G, part_shift) : G, most_rows = parted ? (size_t)1 << part_shift : M;
    const bool plain = act == DOPT_HIP_ACT_NONE, passes = (dx && steps > kPass) || (dw && most_rows > kPass * 16);
    ColumnJobs jobs{};
    GroupLayout lay{};
    GroupProducts p{};
    float *sums = nullptr;
    auto plan = [&](Scratch s) {
        jobs.n = 0;
        auto job = [&](Columns j, size_t of) {
            j.tiles = (unsigned)ceil_div((size_t)j.cols, (size_t)256);
            j.blocks = (unsigned)(j.tiles * of);
            jobs.j[jobs.n++] = j;
        };
        float *const dz_to = plain ? nullptr : s.take<float>(M * N);
        const float *const dz = plain ? dy : dz_to;
        sums = dbias ? s.take<float>(runs * N) : nullptr;
        unsigned *const dz_tops = dw ? s.take<unsigned>(runs * N) : nullptr, *const x_tops = dw ? s.take<unsigned>(runs * K) : nullptr;
        unsigned *const w_tops = dx ? s.take<unsigned>(G * w_runs * K) : nullptr;
        if (!plain || dbias || dw) job(Columns{dy, pre, dz_to, sums, dz_tops, (int)N, act, 0, 0, 0}, runs);
        if (dw) job(Columns{x, nullptr, nullptr, nullptr, x_tops, (int)K, 0, 0, 0, 0}, runs);
        if (dx) job(Columns{w, nullptr, nullptr, nullptr, w_tops, (int)K, 0, 0, (unsigned)w_runs, 0}, G * w_runs);
        if (dx) {
            lay.rows = RowsJob{dz, N, steps, s.take(rows * steps * 64), s.take<int>(rows), shift_of_tile(tile), (unsigned)(rows / 4)};
            lay.turned = WeightsAcross{w, K, padded_k, N, steps, s.take(G * padded_k * steps * 64), s.take<int>(G * padded_k), w_tops, (int)w_runs,
                                       (unsigned)(G * (padded_k / 64) * ceil_div(steps, (size_t)4))};
            p.rows = RowsProduct{dz, w, K, N, steps, padded_k, 1, K, lay.rows.parts, lay.turned.parts, lay.rows.shift, lay.turned.shift, dx,
                                 passes ? s.take(mtiles * ktiles * tile * tile * 4) : nullptr, (unsigned)ktiles};
            p.rows_per = (unsigned)ceil_div(mtiles * ktiles, (size_t)8);
        }
        if (dw) {
            lay.across[0] = RowsAcross{dz, N, padded_n, s.take(units * 64 * padded_n * 4), s.take<int>(G * padded_n), dz_tops, shift,
                                       (unsigned)(units * (padded_n / 64))};
            lay.across[1] = RowsAcross{x, K, padded_k, s.take(units * 64 * padded_k * 4), s.take<int>(G * padded_k), x_tops, shift,
                                       (unsigned)(units * (padded_k / 64))};
            p.weights = WeightsProduct{dz, x, N, K, padded_n, padded_k, lay.across[0].parts, lay.across[1].parts, lay.across[0].shift, lay.across[1].shift,
                                       dw, parted ? s.take<float>(items * N * K) : nullptr, passes ? s.take(items * wtiles * tile * tile * 4) : nullptr,
                                       (unsigned)(padded_n / tile), (unsigned)ktiles, part_shift};
            p.weights_per = (unsigned)(items * ceil_div(wtiles, (size_t)8));
        }
        return s.bytes;
    };
    char *scratch;
    if (int rc = groups_scratch(&l.q, {Units{shift_of_tile(tile), false, false}, Units{kStepShift, false, false}, Units{shift, false, false},
                                       Units{part_shift, false, true}, kRests}, plan(Scratch{nullptr}), &scratch))
        return rc;
    plan(Scratch{scratch});
    jobs.shift = shift;
    jobs.w_rows = (int)N;
    unsigned blocks = 0;
    for (int i = 0; i < jobs.n; i++) blocks += jobs.j[i].blocks;
    if (blocks) launch_columns(l.q, jobs, blocks);
    DOPT_LAUNCH_CHECK();
    if (dbias) {
        lay.sums = sums;
        lay.dbias = dbias;
        lay.columns = (int)N;
        lay.fold_shift = shift;
        lay.fold_tiles = (unsigned)ceil_div(N, (size_t)32);
        lay.fold_blocks = (unsigned)G * lay.fold_tiles;
    }
    lay.rest[0] = dx;
    lay.rest_cols[0] = K;
    lay.rest_blocks = dx ? (unsigned)num_cus() : 0;
    const unsigned threads = row_threads(steps);
    if (dx && threads != 256) {   // rows by workgroups of their length, turned tiles by 256 threads
        GroupLayout alone = lay;
        alone.turned.blocks = alone.across[0].blocks = alone.across[1].blocks = alone.fold_blocks = alone.rest_blocks = 0;
        hipLaunchKernelGGL(groups_layout_k, dim3(alone.rows.blocks), dim3(threads), 0, stream(), l.q, alone);
        lay.rows.blocks = 0;
    }
    const unsigned all = lay.rows.blocks + lay.turned.blocks + lay.across[0].blocks + lay.across[1].blocks + lay.fold_blocks + lay.rest_blocks;
    hipLaunchKernelGGL(groups_layout_k, dim3(all), dim3(256), 0, stream(), l.q, lay);
    DOPT_LAUNCH_CHECK();
    if (int rc = launch_products(l.q, tile, passes, p)) return rc;
    return parted ? groups_join(l, part_shift, p.weights.parts, dw) : DOPT_HIP_OK;
}

}  // namespace dopt
