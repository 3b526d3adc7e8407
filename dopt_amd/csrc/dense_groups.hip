// Dense layers whose rows fall into groups of consecutive rows with a weight matrix and a bias of their own, forward and backward: the
// layers of experts, domains or heads, where the sizes of the groups are known to the device alone.  No counterpart in the reference
// (its one dense layer is nnet/source/dopt/nnet/layers/dense.d).
//
//     rows o[g] .. o[g + 1] - 1:  pre = x w_g^T + bias_g,  y = act(pre);  rows of no group: zeros
//     dz = dy act'(pre),  dx = dz w_g,  dw_g = dz^T x and dbias_g = column sums of dz over the group's rows;  dx of no group's rows: zeros
//
// A workgroup finds its rows in the offsets itself: the grid has room for any sizes, workgroups beyond what there is end at once.
//
// Here are the small products: tiles of 32 x 32 by eight wavefronts that share the reduction, fp32 instructions, one launch forward, two backward.  Bound by
// a launch and by what the tiles read from the L2: 64 rows in eight groups, [64 x 512] from 512, 7.2 us, of which the latency of a launch is 3.4 and w 1.6.
// And products of single rows, which w bounds: one row of [4096 x 4096] 15.0 us, 67 MB at 4.5 TB/s.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "dense_groups.h"
#include "small_product.h"

namespace {

using namespace dopt;

constexpr int kTileShift = 5;    // rows of a tile: 32
typedef float v4f_any __attribute__((ext_vector_type(4), aligned(4)));   // sixteen bytes wherever they start
constexpr int kRunShift = 6;     // rows that a thread adds up for dbias before it rounds to memory: 64
typedef float SmallSums[32 * 33];

// y = act(x w^T + bias): a tile of 32 rows of a group by 32 columns.  kLong: a wavefront has more than 1024 steps, which are added in parts of so many; in
// one accumulator 2^20 equal products of one sign were off by 1e-3 of their sum.
template <bool kCut, bool kLong>
__global__ __launch_bounds__(64 * kSmallWaves) void groups_small_k(GroupLayer l, int kslice, const float *x, const float *w, const float *bias, float *y,
                                                                    float *pre, int act)
{
    __shared__ SmallSums red[kSmallWaves];
    const int n0 = (int)blockIdx.x * 32;
    if (n0 >= l.N) return;
    const Segment s = find_unit<true>(l.q, kTileShift, unit_id());
    if (s.group < 0) return;
    const size_t row = s.begin + ((size_t)s.unit << kTileShift);
    const int rows = (int)min(s.end - row, (size_t)32);
    if (s.group == (int)l.q.G) {
        for (int i = threadIdx.x; i < 32 * rows; i += 64 * kSmallWaves) {
            const int c = n0 + (i & 31);
            if (c >= l.N) continue;
            const size_t at = (row + (i >> 5)) * l.N + c;
            y[at] = 0.0f;
            if (pre) pre[at] = 0.0f;
        }
        return;
    }
    const DenseEpilogue ep{bias ? bias + (size_t)s.group * l.N : nullptr, nullptr, pre ? pre + row * l.N : nullptr, act, (size_t)l.N};
    sgemm_small_body<false, true, kCut, DenseEpilogue, kLong>(rows, l.N, l.K, l.K, l.K, kslice, x + row * l.K, w + (size_t)s.group * l.N * l.K, y + row * l.N,
                                                       nullptr, 0, nullptr, 0, nullptr, (int)blockIdx.x, 0, 0, l.K, red, ep);
}

// The same for groups of a handful of rows, as when single tokens are served: up to R rows of a group by eight columns, two to a wavefront, whose lanes
// read a row of w side by side, a kilobyte at a time, while x waits in LDS.  Bound by memory.  Sums of a lane are of 16 values, then of those, then of the lanes.
template <int R>
__global__ __launch_bounds__(256) void groups_few_k(GroupLayer l, const float *x, const float *w, const float *bias, float *y, float *pre, int act)
{
    constexpr int kColumns = 8, kChunk = 1024;
    constexpr int kShift = R / 2;   // R: 1, 2 or 4
    __shared__ __attribute__((aligned(16))) float rows_of[R][kChunk];
    const int n0 = (int)blockIdx.x * kColumns;
    if (n0 >= l.N) return;
    const Segment s = find_unit<true>(l.q, kShift, unit_id());
    if (s.group < 0) return;
    const size_t row = s.begin + ((size_t)s.unit << kShift), N = l.N, K = l.K;
    const int rows = (int)min(s.end - row, (size_t)R);
    if (s.group == (int)l.q.G) {
        for (int i = threadIdx.x; i < kColumns * rows; i += 256) {
            const int c = n0 + i % kColumns;
            if (c >= l.N) continue;
            const size_t at = (row + i / kColumns) * N + c;
            y[at] = 0.0f;
            if (pre) pre[at] = 0.0f;
        }
        return;
    }
    const int lane = (int)threadIdx.x & 63, c0 = n0 + 2 * ((int)threadIdx.x >> 6);
    const float *of[2];
#pragma unroll
    for (int j = 0; j < 2; j++) of[j] = w + (s.group * N + min(c0 + j, l.N - 1)) * K;
    auto quad = [&](const float *p, size_t k) {   // zero beyond the row's end
        if (k + 4 <= K) return *(const v4f_any *)(p + k);
        v4f_any v{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int e = 0; e < 3; e++)
            if (k + e < K) v[e] = p[k + e];
        return v;
    };
    v4f_any next[2][4];
    auto fetch = [&](size_t k0) {
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int j = 0; j < 2; j++) next[j][t] = quad(of[j], k0 + 256 * t + 4 * lane);
    };
    float all[R][2] = {};
    fetch(0);
    for (size_t k0 = 0; k0 < K; k0 += kChunk) {
        v4f_any own[2][4];
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int j = 0; j < 2; j++) own[j][t] = next[j][t];
        if (k0) __syncthreads();
#pragma unroll
        for (int r = 0; r < R; r++) {
            const v4f_any v = r < rows ? quad(x + (row + r) * K, k0 + 4 * threadIdx.x) : v4f_any{0.0f, 0.0f, 0.0f, 0.0f};
            *(v4f_any *)&rows_of[r][4 * threadIdx.x] = v;
        }
        __syncthreads();
        if (k0 + kChunk < K) fetch(k0 + kChunk);
        float part[R][2] = {};
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int r = 0; r < R; r++) {
                const v4f_any v = *(const v4f_any *)&rows_of[r][256 * t + 4 * lane];
#pragma unroll
                for (int j = 0; j < 2; j++)
#pragma unroll
                    for (int e = 0; e < 4; e++) part[r][j] = __builtin_fmaf(v[e], own[j][t][e], part[r][j]);
            }
#pragma unroll
        for (int r = 0; r < R; r++)
#pragma unroll
            for (int j = 0; j < 2; j++) all[r][j] += part[r][j];
    }
    float mine = 0.0f;   // lane 2 r + j has row r, column j
#pragma unroll
    for (int r = 0; r < R; r++)
#pragma unroll
        for (int j = 0; j < 2; j++) {
            float v = all[r][j];
#pragma unroll
            for (int m = 32; m; m >>= 1) v += __shfl_xor(v, m, 64);
            if (lane == 2 * r + j) mine = v;
        }
    const int r = lane >> 1, c = c0 + (lane & 1);
    if (r >= rows || c >= l.N) return;
    const DenseEpilogue ep{bias ? bias + s.group * N : nullptr, nullptr, pre ? pre + row * N : nullptr, act, N};
    y[(row + r) * N + c] = ep(mine, r * N + c);
}

// The gradients in one launch, each by its own workgroups: dx = dz w, a tile of 32 rows of a group by 32 of the K columns; dw = dz^T x over
// 2^shift rows of a group, a tile of 32 of the N rows by 32 of the K columns, which wait for groups_join_k in `parts` where a
// group is several such parts; dbias from the sums of runs of rows, 32 columns of a group by sixteen lanes.
struct SmallGrads {
    const float *dz, *x, *w, *sums;
    float *dx, *dw, *parts, *dbias;   // parts: or null
    int slice, shift;
    unsigned dx_tiles, dw_tiles, fold_tiles;           // workgroups side by side
    size_t dx_blocks, dw_blocks, fold_blocks;
};

template <bool kCut, bool kLong>
__device__ __forceinline__ void small_dx(const GroupLayer &l, const SmallGrads &g, unsigned tile, unsigned unit, SmallSums *red)
{
    const int k0 = (int)tile * 32;
    if (k0 >= l.K) return;
    const Segment s = find_unit<true>(l.q, kTileShift, unit);
    if (s.group < 0) return;
    const size_t row = s.begin + ((size_t)s.unit << kTileShift);
    const int rows = (int)min(s.end - row, (size_t)32);
    if (s.group == (int)l.q.G) {
        for (int i = threadIdx.x; i < 32 * rows; i += 64 * kSmallWaves)
            if (k0 + (i & 31) < l.K) g.dx[(row + (i >> 5)) * l.K + k0 + (i & 31)] = 0.0f;
        return;
    }
    sgemm_small_body<false, false, kCut, NoEpilogue, kLong>(rows, l.K, l.N, l.N, l.K, g.slice, g.dz + row * l.N, g.w + (size_t)s.group * l.N * l.K,
                                                            g.dx + row * l.K, nullptr, 0, nullptr, 0, nullptr, (int)tile, 0, 0, l.N, red);
}

__device__ __forceinline__ void small_dw(const GroupLayer &l, const SmallGrads &g, unsigned tile, unsigned unit, SmallSums *red)
{
    const unsigned tiles = (unsigned)(l.K + 31) / 32, bx = tile % tiles, by = tile / tiles;
    if ((int)by * 32 >= l.N) return;
    const Segment s = find_unit<false, true>(l.q, g.shift, unit);
    if (s.group < 0) return;
    const size_t row = s.begin + ((size_t)s.unit << g.shift), matrix = (size_t)l.N * l.K;
    const int rows = (int)min((size_t)s.end - row, (size_t)1 << g.shift);
    const int kslice = ((rows + kSmallWaves - 1) / kSmallWaves + 7) / 8 * 8;
    float *const to = g.parts ? g.parts + unit * matrix : g.dw + s.group * matrix;
    sgemm_small_body<true, false, false>(l.N, l.K, rows, l.N, l.K, kslice, g.dz + row * l.N, g.x + row * l.K, to, nullptr, 0, nullptr, 0, nullptr, (int)bx,
                                         (int)by, 0, rows, red);
}

constexpr unsigned kRow = 1u << 22;   // workgroups of a row of such a grid
template <bool kCut, bool kLong>
__global__ __launch_bounds__(64 * kSmallWaves) void groups_small_grad_k(GroupLayer l, SmallGrads g)
{
    __shared__ SmallSums red[kSmallWaves];
    size_t block = (size_t)blockIdx.y * kRow + blockIdx.x;
    if (block < g.dx_blocks) return small_dx<kCut, kLong>(l, g, (unsigned)(block % g.dx_tiles), (unsigned)(block / g.dx_tiles), red);
    block -= g.dx_blocks;
    if (block < g.dw_blocks) return small_dw(l, g, (unsigned)(block % g.dw_tiles), (unsigned)(block / g.dw_tiles), red);
    block -= g.dw_blocks;
    if (block < g.fold_blocks)
        fold_runs(l, kRunShift, g.sums, g.dbias, (unsigned)(block % g.fold_tiles), (unsigned)(block / g.fold_tiles), 2 * kSmallWaves, (float(*)[33])red);
}
// Adds a group's parts, of which an empty one has a matrix of zeros.
__global__ __launch_bounds__(256) void groups_join_k(GroupLayer l, int shift, const float *parts, float *dw)
{
    const size_t matrix = (size_t)l.N * l.K;
    const Segment s = find_group<true>(l.q, shift, unit_id());
    if (s.group < 0) return;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < matrix; i += (size_t)gridDim.x * 256) {
        const float *const from = parts + s.first * matrix + i;
        float all = 0.0f;
        for (unsigned p0 = 0; p0 < s.unit; p0 += 64) {   // sums of 64 values each
            float sum = 0.0f;
#pragma unroll 4
            for (unsigned p = p0; p < min(s.unit, p0 + 64); p++) sum += from[p * matrix];
            all += sum;
        }
        dw[s.group * matrix + i] = all;
    }
}

// dz (or null) of 64 rows of a group by 256 columns, and their sums, for fewer than four columns.
__global__ __launch_bounds__(256) void groups_dz_k(GroupLayer l, int act, const float *dy, const float *pre, float *dz, float *sums)
{
    const int c = (int)blockIdx.x * 256 + (int)threadIdx.x;
    if ((int)blockIdx.x * 256 >= l.N) return;
    const Segment s = find_unit<false>(l.q, kRunShift, unit_id());
    if (s.group < 0 || c >= l.N) return;
    const size_t row = s.begin + ((size_t)s.unit << kRunShift);
    const int rows = (int)min((size_t)s.end - row, (size_t)1 << kRunShift);
    const size_t at = row * l.N + c;
    float sum = 0.0f;
    with_activation(act, [&](auto kind) {
        constexpr bool kPlain = decltype(kind)::value == DOPT_HIP_ACT_NONE;
#pragma unroll 8
        for (int r = 0; r < rows; r++) {
            const size_t i = at + (size_t)r * l.N;
            const float v = kPlain ? dy[i] : act_grad<kind.value>(dy[i], pre[i]);
            sum += v;
            if (!kPlain && dz) dz[i] = v;
        }
    });
    if (sums) sums[(size_t)unit_id() * l.N + c] = sum;
}
// The fronts of a kind of units by a workgroup of sixteen wavefronts, sixteen pieces at a time.
struct FrontKinds {
    Units kind[kMostFronts];
};
__global__ __launch_bounds__(1024) void groups_fronts_k(Groups q, FrontKinds kinds, Front *fronts)
{
    __shared__ unsigned ends[16], counts[16];
    const Units kind = kinds.kind[blockIdx.x];
    Front *const to = fronts + (size_t)blockIdx.x * q.pieces;
    const unsigned lane = threadIdx.x & 63, wave = threadIdx.x >> 6, count = segments_of(q, kind.rest);
    unsigned units = 0, bound = first_row(q, kind.rest);
    for (unsigned base = 0; base < count; base += 1024) {
        const unsigned s = base + threadIdx.x;
        unsigned end = wave_scan(end_of(q, kind.rest, s), [](unsigned a, unsigned b) { return max(a, b); });
        if (lane == 63) ends[wave] = end;
        __syncthreads();
        unsigned before = bound;   // where what lies in front of the wavefront's piece ends
        for (unsigned i = 0; i < wave; i++) before = max(before, ends[i]);
        for (unsigned i = 0; i < 16; i++) bound = max(bound, ends[i]);
        end = max(end, before);
        unsigned begin = (unsigned)__shfl_up((int)end, 1, 64);
        if (lane == 0) begin = before;
        const unsigned n = s < count ? units_of(begin, end, kind.shift, kind.all) : 0;
        const unsigned upto = wave_scan(n, [](unsigned a, unsigned b) { return a + b; });
        if (lane == 63) counts[wave] = upto;
        __syncthreads();
        unsigned in_front = units;
        for (unsigned i = 0; i < wave; i++) in_front += counts[i];
        for (unsigned i = 0; i < 16; i++) units += counts[i];
        if (lane == 0 && s < count) to[s / 64] = Front{in_front, before};
        __syncthreads();
    }
}
__global__ __launch_bounds__(256) void groups_zero_k(size_t n, float *p)
{
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) p[i] = 0.0f;
}
int clear(float *p, size_t n)
{
    if (!p || !n) return DOPT_HIP_OK;
    hipLaunchKernelGGL(groups_zero_k, dim3((unsigned)std::min(ceil_div(n, (size_t)256), (size_t)num_cus() * 16)), dim3(256), 0, stream(), n, p);
    DOPT_LAUNCH_CHECK();
    return DOPT_HIP_OK;
}

constexpr size_t kBytes = (size_t)1 << 31;   // what a buffer resource of the small products covers

int check(const char *who, size_t G, size_t M, size_t N, size_t K, int act)
{
    DOPT_REQUIRE(known_activation(act), "%s: there is no activation %d", who, act);
    // the small products reach 2 GB of one group's w and of 256 rows
    DOPT_REQUIRE(G <= ((size_t)1 << 20) && M < ((size_t)1 << 31) && N <= ((size_t)1 << 20) && K <= ((size_t)1 << 20) &&
                     std::max(N, (size_t)1) * std::max(K, (size_t)1) < kBytes / 4 && M * std::max(N, K) < ((size_t)1 << 40) &&
                     G * N * K < ((size_t)1 << 40),
                 "%s: dimensions too large", who);
    return DOPT_HIP_OK;
}

// What the small products take, in us: launches, rounds of tiles of 32 x 32 that each read their operands, or all of w; of gradients their rows, and a
// workgroup for each tile of each group's dw.  The way that takes the least is taken; the costs are fitted to some 350 products and 120 gradients, of
// which a dozen take more than 10 % longer than by the fastest way.  Eight groups, small, split and wide:
//     [64 x 512] from 512 7.4 10.7 29       [1024 x 512] from 512 19 13 36       [4096 x 512] from 512 46 28 39       [16384 x 512] from 512 156 77 70
//     [1024 x 1024] from 1024 45 28 51      [8192 x 1024] from 1024 279 123 107  [512 x 4096] from 1024 104 50 85
// and gradients
//     [128 x 256] from 256 12 14 30         [1024 x 512] from 512 39 29 54       [4096 x 512] from 512 81 57 73       [16384 x 512] from 512 256 211 177
//     [2048 x 1024] from 1024 171 86 90     [8192 x 1024] from 1024 436 298 221  [256 x 4096] from 1024 269 110 243
double small_us(size_t G, size_t M, size_t N, size_t K)
{
    const double rounds = group_tiles(G, M, N, 32) / num_cus(), least = G * N * K > (size_t)1 << 26 ? 1.2 : 0.75;   // (w that the last cache does not hold)
    return 5 + std::max(0.0101 * K * std::max(rounds > 1 ? rounds + 0.5 : rounds, least), weights_us(G, M, N, K, 3.5e6));
}
double small_grad_us(size_t G, size_t M, size_t N, size_t K)
{
    const double m = (double)M, dw = ((double)N / 32 + 0.5) * ceil_div(K, (size_t)32);
    return 10.8 + 1e-6 * (10 * m * K + 7 * m * N + 13 * (group_tiles(G, M, K, 32) * N + dw * m)) + 6.6e-3 * G * dw;
}
// Rows of a group that groups_few_k takes at a time, and its time: w of the groups that have rows, or the products of whole units, and its chunks.  Eight groups,
// it and the small products: one row of [4096 x 4096] 15.0 and 62.6 us (w alone 13.1), two 29 and 68, eight 61 and 98, 32 121 and 131, 64 171 and 132;
// eight rows of [512 x 512] 5.4 and 6.0, of [4096 x 1024] 22.8 and 28.3, of 1024 from 4096 18.6 and 34.2.
int few_rows(size_t G, size_t M)
{
    const size_t rows = std::min(M, ceil_div(3 * M, 2 * G));
    return rows <= 1 ? 1 : rows <= 2 ? 2 : 4;
}
double few_us(size_t G, size_t M, size_t N, size_t K)
{
    const double rows = few_rows(G, M), chunks = (double)ceil_div(K, (size_t)1024), groups = groups_with_rows(G, M);
    const double units = std::max(groups, M / rows + (rows > 1 ? 0.75 * (groups - 1) : 0.0));
    return 1.1 * (4.9 + 0.4 * chunks + std::max(weights_us(G, M, N, K, 5.1e6), 0.3 * units * ceil_div(N, (size_t)8) * chunks * rows / num_cus()));
}
enum class Way { kFew, kSmall, kSplit, kWide };
Way way_of(double few, double small, double split, double wide)
{
    const double least = std::min(std::min(few, small), std::min(split, wide));
    return few == least ? Way::kFew : small == least ? Way::kSmall : split == least ? Way::kSplit : Way::kWide;
}

size_t slice_of(size_t depth) { return ceil_div(ceil_div(depth, (size_t)kSmallWaves), (size_t)8) * 8; }
// Calls with a reduction's kinds: its rows are no whole quads; a wavefront's share is longer than a part.
template <class F>
void with_reduction(size_t depth, F &&f)
{
    auto with = [&](auto cut) { slice_of(depth) > (size_t)kSmallPart ? f(cut, std::true_type{}) : f(cut, std::false_type{}); };
    depth % 4 ? with(std::true_type{}) : with(std::false_type{});
}

struct Span {
    const void *p;
    size_t bytes;
};
template <size_t I, size_t O>
int apart(const char *who, const Span (&in)[I], const Span (&out)[O])
{
    for (size_t i = 0; i < O; i++) {
        for (const Span &s : in) DOPT_REQUIRE(!overlaps(out[i].p, out[i].bytes, s.p, s.bytes), "%s: a result overlaps an operand", who);
        for (size_t k = 0; k < i; k++) DOPT_REQUIRE(!overlaps(out[i].p, out[i].bytes, out[k].p, out[k].bytes), "%s: two results overlap", who);
    }
    return DOPT_HIP_OK;
}

}  // namespace

namespace dopt {

int groups_scratch(Groups *q, std::initializer_list<Units> units, size_t bytes, char **scratch)
{
    const size_t pieces = ceil_div((size_t)q->G + 2, (size_t)64), kinds = q->G > kNoFronts ? units.size() : 0;
    const size_t front_bytes = ceil_div(kinds * pieces * sizeof(Front), (size_t)256) * 256;
    *scratch = nullptr;
    if (front_bytes + bytes == 0) return DOPT_HIP_OK;
    char *const at = (char *)workspace(front_bytes + bytes);
    if (!at) return DOPT_HIP_ERR_OOM;
    *scratch = at + front_bytes;
    if (!kinds) return DOPT_HIP_OK;
    DOPT_REQUIRE(kinds <= kMostFronts, "dopt_hip_dense_groups: more kinds of units than there are places for");
    FrontKinds all{};
    q->pieces = (unsigned)pieces;
    for (int &key : q->keys) key = -1;
    size_t i = 0;
    for (const Units &u : units) {
        all.kind[i] = u;
        q->keys[i++] = u.key();
    }
    hipLaunchKernelGGL(groups_fronts_k, dim3((unsigned)kinds), dim3(1024), 0, stream(), *q, all, (Front *)at);
    DOPT_LAUNCH_CHECK();
    q->fronts = (const Front *)at;
    return DOPT_HIP_OK;
}

int groups_join(const GroupLayer &l, int shift, const float *parts, float *dw)
{
    const size_t matrix = (size_t)l.N * l.K;
    hipLaunchKernelGGL(groups_join_k, grid_of(std::min(ceil_div(matrix, (size_t)256), (size_t)num_cus() * 8), l.q.G), dim3(256), 0, stream(), l, shift, parts, dw);
    DOPT_LAUNCH_CHECK();
    return DOPT_HIP_OK;
}

}  // namespace dopt

extern "C" {

int dopt_hip_dense_groups(size_t G, size_t M, size_t N, size_t K, int act, const int32_t *offsets, const float *x, const float *w, const float *bias,
                          float *y, float *pre)
{
    const char *const who = "dopt_hip_dense_groups";
    if (int rc = check(who, G, M, N, K, act)) return rc;
    if (M * N == 0) return DOPT_HIP_OK;
    DOPT_REQUIRE(y && (G == 0 || (offsets && (K == 0 || (x && w)))), "%s: null argument", who);
    const size_t f = sizeof(float), out = M * N * f;
    const Span in[] = {{offsets, (G + 1) * sizeof(int32_t)}, {x, M * K * f}, {w, G * N * K * f}, {bias, G * N * f}};
    const Span results[] = {{y, out}, {pre, out}};
    if (int rc = apart(who, in, results)) return rc;
    DOPT_ENSURE_INIT();
    GroupLayer l{Groups{offsets, (unsigned)G, (unsigned)M}, (int)N, (int)K};
    char *scratch;
    const Way way = G == 0 ? Way::kSmall : way_of(few_us(G, M, N, K), small_us(G, M, N, K), groups_split_us(G, M, N, K), groups_wide_us(G, M, N, K));
    if (way == Way::kSplit) return groups_split(l, x, w, bias, act, y, pre);
    if (way == Way::kWide) return groups_wide(l, x, w, bias, act, y, pre);
    if (way == Way::kFew) {
        auto few = [&](auto rows) {
            constexpr int R = decltype(rows)::value;
            if (int rc = groups_scratch(&l.q, {Units{R / 2, true, false}}, 0, &scratch)) return rc;
            hipLaunchKernelGGL(groups_few_k<R>, grid_of(ceil_div(N, (size_t)8), most_units(M, G + 2, R / 2)), dim3(256), 0, stream(), l, x, w, bias, y, pre, act);
            DOPT_LAUNCH_CHECK();
            return (int)DOPT_HIP_OK;
        };
        const int rows = few_rows(G, M);
        return rows == 4 ? few(std::integral_constant<int, 4>{}) : rows == 2 ? few(std::integral_constant<int, 2>{}) : few(std::integral_constant<int, 1>{});
    }
    const dim3 grid = grid_of(ceil_div(N, (size_t)32), most_units(M, G + 2, kTileShift));
    const int slice = (int)slice_of(K);
    if (int rc = groups_scratch(&l.q, {Units{kTileShift, true, false}}, 0, &scratch)) return rc;
    with_reduction(K, [&](auto cut, auto is_long) {
        hipLaunchKernelGGL((groups_small_k<cut.value, is_long.value>), grid, dim3(64 * kSmallWaves), 0, stream(), l, slice, x, w, bias, y, pre, act);
    });
    DOPT_LAUNCH_CHECK();
    return DOPT_HIP_OK;
}

int dopt_hip_dense_groups_grad(size_t G, size_t M, size_t N, size_t K, int act, const int32_t *offsets, const float *dy, const float *pre,
                               const float *x, const float *w, float *dx, float *dw, float *dbias)
{
    const char *const who = "dopt_hip_dense_groups_grad";
    if (int rc = check(who, G, M, N, K, act)) return rc;
    const bool some = G > 0 && M * N > 0;
    DOPT_REQUIRE(!some || (offsets && dy && (act == DOPT_HIP_ACT_NONE || pre)), "%s: null argument", who);
    DOPT_REQUIRE(!some || K == 0 || !dx || w, "%s: the gradient of x needs w", who);
    DOPT_REQUIRE(!some || K == 0 || !dw || x, "%s: the gradient of w needs x", who);
    DOPT_REQUIRE(G == 0 || offsets || M == 0, "%s: null argument", who);
    const size_t f = sizeof(float);
    const Span in[] = {{offsets, (G + 1) * sizeof(int32_t)}, {dy, M * N * f}, {pre, M * N * f}, {x, M * K * f}, {w, G * N * K * f}};
    const Span results[] = {{dx, M * K * f}, {dw, G * N * K * f}, {dbias, G * N * f}};
    if (int rc = apart(who, in, results)) return rc;
    DOPT_ENSURE_INIT();
    if (K == 0 || M * K == 0) dx = nullptr;
    if (G * N * K == 0) dw = nullptr;
    if (G * N == 0) dbias = nullptr;
    if (!dx && !dw && !dbias) return DOPT_HIP_OK;
    if (!some) {   // nothing to sum up
        if (int rc = clear(dx, M * K)) return rc;
        if (int rc = clear(dw, G * N * K)) return rc;
        return clear(dbias, G * N);
    }
    GroupLayer l{Groups{offsets, (unsigned)G, (unsigned)M}, (int)N, (int)K};
    const Way way = way_of(HUGE_VAL, small_grad_us(G, M, N, K), groups_split_grad_us(G, M, N, K), groups_wide_grad_us(G, M, N, K));
    if ((dx || dw) && way == Way::kSplit) return groups_split_grad(l, act, dy, pre, x, w, dx, dw, dbias);
    if ((dx || dw) && way == Way::kWide) return groups_wide_grad(l, act, dy, pre, x, w, dx, dw, dbias);
    // Rows of a part of a group's reduction: at most 8192, 1024 for each wavefront, so that sums of one sign are not rounded the same way for
    // long; fewer where the tiles would not fill the chip (a part's matrix is written and read).
    const size_t tiles = ceil_div(N, (size_t)32) * ceil_div(K, (size_t)32);
    int shift = 13;
    if (dw)
        while (shift > 8 && (most_units(M, G, shift) * tiles < (size_t)num_cus() * 4 || ((size_t)1 << shift) * std::max(N, K) * f >= kBytes)) shift--;
    const bool direct = ((size_t)1 << shift) >= M;
    const size_t dw_units = most_units(M, G, shift), runs = most_units(M, G, kRunShift);
    auto rounded = [](size_t bytes) { return ceil_div(bytes, (size_t)256) * 256; };
    const bool plain = act == DOPT_HIP_ACT_NONE;
    const size_t dz_bytes = plain || !(dx || dw) ? 0 : rounded(M * N * f), sum_bytes = dbias ? rounded(runs * N * f) : 0,
                 part_bytes = dw && !direct ? dw_units * N * K * f : 0;
    char *scratch;
    if (int rc = groups_scratch(&l.q, {Units{kTileShift, true, false}, Units{kRunShift, false, false}, Units{shift, false, true}},
                                dz_bytes + sum_bytes + part_bytes, &scratch))
        return rc;
    float *const dz_to = dz_bytes ? (float *)scratch : nullptr, *const sums = (float *)(scratch + dz_bytes), *const parts = (float *)(scratch + dz_bytes + sum_bytes);
    const float *const dz = plain ? dy : dz_to;
    if (!plain || dbias) {
        if (N >= 4) {
            if (int rc = groups_dz(l, act, kRunShift, dy, pre, dz_to, dbias ? sums : nullptr)) return rc;
        } else {
            hipLaunchKernelGGL(groups_dz_k, grid_of(ceil_div(N, (size_t)256), runs), dim3(256), 0, stream(), l, act, dy, pre, dz_to, dbias ? sums : nullptr);
            DOPT_LAUNCH_CHECK();
        }
    }
    SmallGrads g{dz, x, w, sums, dx, dw, direct ? nullptr : parts, dbias, (int)slice_of(N), shift, (unsigned)abreast(ceil_div(K, (size_t)32)),
                 (unsigned)abreast(tiles), (unsigned)abreast(ceil_div(N, (size_t)32)), 0, 0, 0};
    if (dx) g.dx_blocks = g.dx_tiles * most_units(M, G + 2, kTileShift);
    if (dw) g.dw_blocks = g.dw_tiles * dw_units;
    if (dbias) g.fold_blocks = g.fold_tiles * G;
    const size_t blocks = g.dx_blocks + g.dw_blocks + g.fold_blocks;
    DOPT_REQUIRE(blocks < ((size_t)1 << 37), "%s: dimensions too large", who);
    const dim3 grid((unsigned)std::min(blocks, (size_t)kRow), (unsigned)ceil_div(blocks, (size_t)kRow));
    with_reduction(dx ? N : 0, [&](auto cut, auto is_long) {
        hipLaunchKernelGGL((groups_small_grad_k<cut.value, is_long.value>), grid, dim3(64 * kSmallWaves), 0, stream(), l, g);
    });
    DOPT_LAUNCH_CHECK();
    return dw && !direct ? groups_join(l, shift, parts, dw) : DOPT_HIP_OK;
}

}  // extern "C"
