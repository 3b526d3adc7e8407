// Products of middle size of dense layers of groups: tiles of 64 x 64 whose operands become two fp16 parts on the way (split_tile.h), so that nothing is laid
// out and read again in front of them.  Small enough a tile to have some thousand of them; a workgroup's teams share a reduction where there
// are fewer than the chip holds.
//
// With many tiles bound by what a CU takes in: 16 KB a chunk of 32 steps in 830 cycles, 47 GB/s (of which the matrix instructions need 192, 110 vector
// instructions of each wavefront 450 and LDS 300): [16384 x 4096] from 2048 in sixteen groups 1450 us, dense_groups_wide.hip's 1030.  With few tiles by the
// way from memory to the sums, some 0.9 us a chunk: [1024 x 1024] from 1024 in eight groups 28 us.  Tiles of 128 x 128, by four wavefronts (two to a SIMD) or
// eight, take 1100 and 1090 us for the one and 53 and 42 for the other.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "dense_groups.h"
#include "split_tile.h"

namespace {

using namespace dopt;

constexpr int kTile = kSplitTile, kTileShift = 6;
constexpr int kRunShift = 6;
constexpr unsigned kMostParts = 16;   // of a reduction of y

// y = act(x w^T + bias): a tile of rows of a group, over one of several parts of the reduction where there are few tiles; those wait in `parts`, [part][M][N].
struct SplitForward {
    const float *x, *w, *bias;
    float *y, *pre, *parts;
    int act;
    unsigned tiles, count, steps;   // side by side; parts, and steps of each
};
template <int kTeams, bool kPasses>
__global__ __launch_bounds__(256 * kTeams) void groups_split_k(GroupLayer l, SplitForward f)
{
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const unsigned part = blockIdx.x / f.tiles, n0 = blockIdx.x % f.tiles * kTile;
    if (part >= f.count) return;
    const Segment s = find_unit<true>(l.q, kTileShift, unit_id());
    if (s.group < 0) return;
    const size_t N = l.N, K = l.K;
    if (s.group == (int)l.q.G) {
        if (f.parts) return;
        const size_t row = s.begin + ((size_t)s.unit << kTileShift);
        const int rows = (int)min(s.end - row, (size_t)kTile);
        for (int i = threadIdx.x; i < kTile * rows; i += 256 * kTeams) {
            const unsigned c = n0 + i % kTile;
            if (c >= N) continue;
            const size_t at = (row + i / kTile) * N + c;
            f.y[at] = 0.0f;
            if (f.pre) f.pre[at] = 0.0f;
        }
        return;
    }
    const size_t begin = s.begin, g = (size_t)s.group, from = (size_t)part * f.steps;
    const Matrix32 rows{f.x + begin * K + from, K, s.end - s.begin}, columns{f.w + g * N * K + from, K, (unsigned)N};
    DenseEpilogue ep{f.bias ? f.bias + g * N : nullptr, nullptr, f.pre ? f.pre + begin * N : nullptr, f.act, N};
    float *to = f.y;
    if (f.parts) {
        ep = DenseEpilogue{nullptr, nullptr, nullptr, DOPT_HIP_ACT_NONE, N};
        to = f.parts + part * (size_t)l.q.M * N;
    }
    split_tile<kTeams, true, false, false, kPasses>(rows, columns, (unsigned)min((size_t)f.steps, K - from), s.unit << kTileShift, n0, ep, to + begin * N, lds);
}
// Adds the parts, and the layer's end: a row of a group by 256 columns.  (All parts on their way at once: one after the other they took 20 us.)
__global__ __launch_bounds__(256) void groups_end_k(GroupLayer l, SplitForward f)
{
    const size_t N = l.N, c = (size_t)blockIdx.x * 256 + threadIdx.x;
    if ((size_t)blockIdx.x * 256 >= N) return;
    const Segment s = find_unit<true>(l.q, 0, unit_id());
    if (s.group < 0 || c >= N) return;
    const size_t at = ((size_t)s.begin + s.unit) * N + c, matrix = (size_t)l.q.M * N;
    if (s.group == (int)l.q.G) {
        f.y[at] = 0.0f;
        if (f.pre) f.pre[at] = 0.0f;
        return;
    }
    float part[kMostParts], z = 0.0f;
#pragma unroll
    for (unsigned p = 0; p < kMostParts; p++) part[p] = p < f.count ? f.parts[p * matrix + at] : 0.0f;
#pragma unroll
    for (unsigned p = 0; p < kMostParts; p++) z += part[p];
    const DenseEpilogue ep{f.bias ? f.bias + s.group * N : nullptr, nullptr, f.pre, f.act, N};
    z += ep.bias_of(c);
    if (f.pre) f.pre[at] = z;
    f.y[at] = ep.value(z);
}

// The gradients in one launch, as dense_groups.hip's: dx = dz w, whose reduction is often the longer one, is shared by teams and may be several parts
// ([109 x 2573] from 1017 in five groups 75 -> 57 us); dw = dz^T x over 2^shift rows of a group, a tile for each team; dbias.
struct SplitGrads {
    const float *dz, *x, *w, *sums;
    float *dx, *dw, *parts, *dbias;   // parts: of dw, or null
    float *dx_parts;                  // [part][M][K], or null
    unsigned dx_across, dx_count, dx_steps;
    int shift;
    unsigned dx_tiles, dw_tiles, fold_tiles;
    size_t dx_blocks, dw_blocks, fold_blocks;
};
constexpr unsigned kRow = 1u << 22;   // workgroups of a row of the grid

template <int kTeams, bool kPasses>
__global__ __launch_bounds__(256 * kTeams) void groups_split_grad_k(GroupLayer l, SplitGrads g)
{
    extern __shared__ __attribute__((aligned(16))) char lds[];
    size_t block = (size_t)blockIdx.y * kRow + blockIdx.x;
    const size_t N = l.N, K = l.K;
    if (block < g.dx_blocks) {
        const unsigned at = (unsigned)(block % g.dx_tiles), part = at / g.dx_across, k0 = at % g.dx_across * kTile;
        if (part >= g.dx_count) return;
        const Segment s = find_unit<true>(l.q, kTileShift, (unsigned)(block / g.dx_tiles));
        if (s.group < 0) return;
        const size_t begin = s.begin, from = (size_t)part * g.dx_steps;
        if (s.group == (int)l.q.G) {
            if (g.dx_parts) return;
            const size_t row = begin + ((size_t)s.unit << kTileShift);
            const int rows = (int)min(s.end - row, (size_t)kTile);
            for (int i = threadIdx.x; i < kTile * rows; i += 256 * kTeams)
                if (k0 + i % kTile < K) g.dx[(row + i / kTile) * K + k0 + i % kTile] = 0.0f;
            return;
        }
        float *const to = g.dx_parts ? g.dx_parts + part * (size_t)l.q.M * K : g.dx;
        return split_tile<kTeams, true, false, true, kPasses>(Matrix32{g.dz + begin * N + from, N, s.end - s.begin},
                                                              Matrix32{g.w + (s.group * N + from) * K, K, (unsigned)K},
                                                              (unsigned)min((size_t)g.dx_steps, N - from), s.unit << kTileShift, k0,
                                                              DenseEpilogue{nullptr, nullptr, nullptr, DOPT_HIP_ACT_NONE, K}, to + begin * K, lds);
    }
    block -= g.dx_blocks;
    if (block < g.dw_blocks) {
        // a tile for each team
        const unsigned first = (unsigned)(block % g.dw_tiles) * kTeams, unit = (unsigned)(block / g.dw_tiles), across = (unsigned)((K + kTile - 1) / kTile);
        const unsigned tile = first + threadIdx.x / 256, k0 = tile % across * kTile, n0 = tile / across * kTile;
        if (first / across * kTile >= N) return;
        const Segment s = find_unit<false, true>(l.q, g.shift, unit);
        if (s.group < 0) return;
        const size_t row = s.begin + ((size_t)s.unit << g.shift);
        const unsigned rows = (unsigned)min((size_t)s.end - row, (size_t)1 << g.shift);
        float *const to = g.parts ? g.parts + unit * N * K : g.dw + s.group * N * K;
        if (rows == 0) {
            for (int i = threadIdx.x & 255; i < kTile * kTile; i += 256)
                if (n0 + i / kTile < N && k0 + i % kTile < K) to[(n0 + i / kTile) * K + k0 + i % kTile] = 0.0f;
            return;
        }
        return split_tile<kTeams, false, true, true, kPasses>(Matrix32{g.dz + row * N, N, (unsigned)N}, Matrix32{g.x + row * K, K, (unsigned)K}, rows, n0, k0,
                                                              DenseEpilogue{nullptr, nullptr, nullptr, DOPT_HIP_ACT_NONE, K}, to, lds);
    }
    block -= g.dw_blocks;
    if (block < g.fold_blocks)
        fold_runs(l, kRunShift, g.sums, g.dbias, (unsigned)(block % g.fold_tiles), (unsigned)(block / g.fold_tiles), 8 * kTeams, (float(*)[33])lds);
}

constexpr int kLongestPart = 13;
// Rows of a part of a group's reduction, as a shift: fewer where the tiles would not fill the chip (a part's matrix is written and read).
int part_shift(size_t G, size_t M, size_t tiles)
{
    int shift = kLongestPart;
    while (shift > 8 && most_units(M, G, shift) * tiles < (size_t)num_cus()) shift--;
    return shift;
}
// Parts of [M, N] written and read by a launch of their own.
double parts_us(size_t parts, size_t M, size_t N) { return 4.5 + 8.0 * parts * M * N / 5e6 + 1e-3 * M * ceil_div(N, (size_t)256); }

// Tiles of both products, and chunks of each.
struct GradWork {
    double dx_tiles, dx_chunks, dw_tiles, dw_chunks;   // dx' chunks of a part
    size_t parts;                                      // of dx' reductions
    double chain() const { return std::max(dx_chunks, dw_chunks); }
    // One workgroup's chunks take longer than all of them over the chip: [1024 x 512] from 512 in eight groups with one team 31.4 us, with two 29.8, with
    // four 35.3; [2048 x 512] 39 46 49; [256 x 4096] from 1024 151 110 113; [1024 x 4096] 179 177 191.
    bool few() const { return dx_tiles * parts * dx_chunks + dw_tiles * dw_chunks < 1.5 * chain() * num_cus(); }
    double us() const
    {
        return (0.25 * dx_tiles * parts * (dx_chunks + 18) + 0.44 * dw_tiles * (dw_chunks + 0.2)) / num_cus() + 0.57 * chain();
    }
};
GradWork grad_work(size_t G, size_t M, size_t N, size_t K, double *total)
{
    const size_t tiles = ceil_div(N, (size_t)kTile) * ceil_div(K, (size_t)kTile);
    const int shift = part_shift(G, M, tiles);
    const double units = (size_t)1 << shift < M ? std::max((double)G, (double)M / ((size_t)1 << shift) + 0.5 * G) : (double)G;
    const double chunks = (double)ceil_div(N, (size_t)kChunk);
    GradWork best{group_tiles(G, M, K, kTile), chunks, units * tiles, M / units / kChunk + 0.5, 1};
    double least = best.us();
    for (size_t p = 2; p <= kMostParts && p <= chunks / 4; p *= 2) {
        GradWork w = best;
        w.parts = p;
        w.dx_chunks = chunks / p;
        const double us = w.us() + parts_us(p, M, K);
        if (us < least) least = us, best = w;
    }
    *total = least;
    return best;
}

// A product's time, and in how many parts its reduction is the fastest: another launch, and the parts written and read.  One group, [108 x 367] from 2458 whole
// 40 us (by the small products 31), in sixteen parts 15; four, [600 x 200] from 3986 57 (48) and 25, [3000 x 64] 50 (45) and 27.
double forward_us(size_t G, size_t M, size_t N, size_t K, size_t *parts)
{
    const double chunks = (double)ceil_div(K, (size_t)kChunk), tiles = group_tiles(G, M, N, kTile), weights = weights_us(G, M, N, K, 4e6);
    double best = HUGE_VAL;
    for (size_t p = 1; p == 1 || (p <= kMostParts && p <= chunks / 4); p *= 2) {
        const double products = chunks / p / 4 + 0.3 * tiles * (chunks + 6 * p) / num_cus();
        const double us = 5 + std::max(products, weights) + 8.0 * M * N / 5e6 + (p > 1 ? parts_us(p, M, N) : 0.0);
        if (us < best) best = us, *parts = p;
    }
    return best;
}

template <auto kKernel, int kTeams>
int allow()
{
    static bool raised = false;
    if (kSplitLds<kTeams> >= 60 * 1024 && !raised)
        DOPT_HIP_CHECK(hipFuncSetAttribute((const void *)kKernel, hipFuncAttributeMaxDynamicSharedMemorySize, kSplitLds<kTeams>));
    raised = true;
    return DOPT_HIP_OK;
}
template <int kMost, class F>
int with_teams(int teams, bool passes, F &&f)
{
    auto with = [&](auto n) { return passes ? f(n, std::true_type{}) : f(n, std::false_type{}); };
    if constexpr (kMost == 4)
        if (teams == 4) return with(std::integral_constant<int, 4>{});
    if (teams == 2) return with(std::integral_constant<int, 2>{});
    return with(std::integral_constant<int, 1>{});
}

int end_of_parts(const GroupLayer &l, const SplitForward &f)
{
    hipLaunchKernelGGL(groups_end_k, grid_of(ceil_div((size_t)l.N, (size_t)256), most_units(l.q.M, l.q.G + 2, 0)), dim3(256), 0, stream(), l, f);
    DOPT_LAUNCH_CHECK();
    return DOPT_HIP_OK;
}

}  // namespace

namespace dopt {

double groups_split_us(size_t G, size_t M, size_t N, size_t K)
{
    if (N < 4 || K < 4) return HUGE_VAL;   // (of no use, and sums of dz want four columns)
    size_t parts;
    return forward_us(G, M, N, K, &parts);
}
double groups_split_grad_us(size_t G, size_t M, size_t N, size_t K)
{
    if (N < 4 || K < 4) return HUGE_VAL;
    double products;
    grad_work(G, M, N, K, &products);
    return 11.5 + 3.4e-6 * M * N + products;
}

int groups_split(GroupLayer l, const float *x, const float *w, const float *bias, int act, float *y, float *pre)
{
    const size_t G = l.q.G, M = l.q.M, N = l.N, K = l.K, across = ceil_div(N, (size_t)kTile);
    size_t parts;
    forward_us(G, M, N, K, &parts);
    SplitForward f{x, w, bias, y, pre, nullptr, act, (unsigned)across, (unsigned)parts, (unsigned)(ceil_div(ceil_div(K, (size_t)kChunk), parts) * kChunk)};
    f.count = (unsigned)ceil_div(K, (size_t)f.steps);
    char *scratch;
    if (int rc = groups_scratch(&l.q, {Units{kTileShift, true, false}, Units{0, true, false}}, parts > 1 ? f.count * M * N * sizeof(float) : 0, &scratch)) return rc;
    if (parts > 1) f.parts = (float *)scratch;
    // (workgroups and one, two, four teams: 160 18.9 14.0 12.7 us, 288 22.1 19.4 23.7, 544 28.0 30.0 36.4, reductions of 512 steps)
    const double tiles = group_tiles(G, M, N, kTile) * parts;
    const int teams = tiles <= num_cus() ? 4 : tiles <= 2 * num_cus() ? 2 : 1;
    const int rc = with_teams<4>(teams, f.steps > kPass * 16, [&](auto n, auto passes) {
        constexpr auto kernel = groups_split_k<n.value, passes.value>;
        if (int rc = allow<kernel, n.value>()) return rc;
        hipLaunchKernelGGL(kernel, grid_of(across * f.count, most_units(M, G + 2, kTileShift)), dim3(256 * n.value), kSplitLds<n.value>, stream(), l, f);
        DOPT_LAUNCH_CHECK();
        return (int)DOPT_HIP_OK;
    });
    return rc || parts == 1 ? rc : end_of_parts(l, f);
}

int groups_split_grad(GroupLayer l, int act, const float *dy, const float *pre, const float *x, const float *w, float *dx, float *dw, float *dbias)
{
    const size_t G = l.q.G, M = l.q.M, N = l.N, K = l.K, tiles = ceil_div(N, (size_t)kTile) * ceil_div(K, (size_t)kTile);
    const int shift = dw ? part_shift(G, M, tiles) : kLongestPart;
    const bool direct = ((size_t)1 << shift) >= M, plain = act == DOPT_HIP_ACT_NONE;
    double unused;
    const GradWork work = grad_work(G, M, N, K, &unused);
    const size_t dw_units = most_units(M, G, shift), runs = most_units(M, G, kRunShift), f = sizeof(float), across = ceil_div(K, (size_t)kTile);
    const size_t steps = ceil_div(ceil_div(N, (size_t)kChunk), dx ? work.parts : 1) * kChunk, count = ceil_div(N, steps);
    auto rounded = [](size_t bytes) { return ceil_div(bytes, (size_t)256) * 256; };
    const size_t dz_bytes = plain ? 0 : rounded(M * N * f), sum_bytes = dbias ? rounded(runs * N * f) : 0, dx_bytes = count > 1 ? rounded(count * M * K * f) : 0;
    const size_t part_bytes = dw && !direct ? dw_units * N * K * f : 0, bytes = dz_bytes + sum_bytes + dx_bytes + part_bytes;
    char *scratch;
    if (int rc = groups_scratch(&l.q, {Units{kTileShift, true, false}, Units{kRunShift, false, false}, Units{shift, false, true}, Units{0, true, false}}, bytes, &scratch))
        return rc;
    float *const dz_to = plain ? nullptr : (float *)scratch, *const sums = (float *)(scratch + dz_bytes);
    float *const dx_parts = dx_bytes ? (float *)(scratch + dz_bytes + sum_bytes) : nullptr, *const parts = (float *)(scratch + dz_bytes + sum_bytes + dx_bytes);
    if (!plain || dbias)
        if (int rc = groups_dz(l, act, kRunShift, dy, pre, dz_to, dbias ? sums : nullptr)) return rc;
    const int teams = work.few() ? 2 : 1;
    SplitGrads g{plain ? dy : dz_to, x, w, sums, dx, dw, direct ? nullptr : parts, dbias, dx_parts, (unsigned)across, (unsigned)count, (unsigned)steps, shift,
                 (unsigned)abreast(across * count), (unsigned)abreast(ceil_div(tiles, (size_t)teams)), (unsigned)abreast(ceil_div(N, (size_t)32)), 0, 0, 0};
    if (dx) g.dx_blocks = g.dx_tiles * most_units(M, G + 2, kTileShift);
    if (dw) g.dw_blocks = g.dw_tiles * dw_units;
    if (dbias) g.fold_blocks = g.fold_tiles * G;
    const size_t blocks = g.dx_blocks + g.dw_blocks + g.fold_blocks;
    DOPT_REQUIRE(blocks < ((size_t)1 << 37), "dopt_hip_dense_groups_grad: dimensions too large");
    const dim3 grid((unsigned)std::min(blocks, (size_t)kRow), (unsigned)ceil_div(blocks, (size_t)kRow));
    const bool passes = (dx && steps > kPass * 16) || (dw && std::min(M, (size_t)1 << shift) > kPass * 16);
    const int rc = with_teams<2>(teams, passes, [&](auto n, auto passes) {
        constexpr auto kernel = groups_split_grad_k<n.value, passes.value>;
        if (int rc = allow<kernel, n.value>()) return rc;
        hipLaunchKernelGGL(kernel, grid, dim3(256 * n.value), kSplitLds<n.value>, stream(), l, g);
        DOPT_LAUNCH_CHECK();
        return (int)DOPT_HIP_OK;
    });
    if (rc) return rc;
    if (dx_parts)
        if (int rc = end_of_parts(GroupLayer{l.q, l.K, 0}, SplitForward{nullptr, nullptr, nullptr, dx, nullptr, dx_parts, DOPT_HIP_ACT_NONE, 0, (unsigned)count, 0})) return rc;
    return dw && !direct ? groups_join(l, shift, parts, dw) : DOPT_HIP_OK;
}

}  // namespace dopt
