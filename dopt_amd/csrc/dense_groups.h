// What the kernels of dense layers of groups share (dense_groups.hip, dense_groups_wide.hip).
#pragma once

#include <cmath>

#include "common.h"
#include "dense.h"
#include "groups.h"

namespace dopt {

struct GroupLayer {
    Groups q;
    int N, K;   // of w_g [N, K]
};

// The ways of such products besides the small ones' (dense_groups.hip): of two fp16 parts of each value that are made on the way (dense_groups_split.hip)
// or laid out once (dense_groups_wide.hip).  What each takes of y [M, N] from K steps and of its gradients, in us, or infinity where it cannot.
double groups_split_us(size_t G, size_t M, size_t N, size_t K);
double groups_split_grad_us(size_t G, size_t M, size_t N, size_t K);
double groups_wide_us(size_t G, size_t M, size_t N, size_t K);
double groups_wide_grad_us(size_t G, size_t M, size_t N, size_t K);
int groups_split(GroupLayer l, const float *x, const float *w, const float *bias, int act, float *y, float *pre);
int groups_wide(GroupLayer l, const float *x, const float *w, const float *bias, int act, float *y, float *pre);
// dy and pre give dz, which is written where there is an activation; any result may be null.
int groups_split_grad(GroupLayer l, int act, const float *dy, const float *pre, const float *x, const float *w, float *dx, float *dw, float *dbias);
int groups_wide_grad(GroupLayer l, int act, const float *dy, const float *pre, const float *x, const float *w, float *dx, float *dw, float *dbias);
// dz (which may be null) of N >= 4 columns, and the sums (null too) of runs of 2^shift rows of a group.
int groups_dz(const GroupLayer &l, int act, int shift, const float *dy, const float *pre, float *dz, float *sums);

// dense_groups.hip: dw from the matrices of parts of 2^shift rows of a group, of which an empty group has one of zeros.
int groups_join(const GroupLayer &l, int shift, const float *parts, float *dw);

// Groups that have any of M rows which fall to them at random.
inline double groups_with_rows(size_t G, size_t M) { return G * (1 - std::pow(1 - 1.0 / G, (double)M)); }
// ... whose matrices come from memory at so many bytes a us.
inline double weights_us(size_t G, size_t M, size_t N, size_t K, double rate) { return groups_with_rows(G, M) * N * K * 4 / rate; }
// Tiles of `side` rows and columns, half of one more for each group.
inline double group_tiles(size_t G, size_t M, size_t N, size_t side) { return ((double)M / side + 0.5 * (G < M ? G : M)) * ceil_div(N, side); }

// dbias from the sums of runs of 2^shift rows of a group: `lanes` lanes to a column, of 32 side by side; red: a value of each.
__device__ __forceinline__ void fold_runs(const GroupLayer &l, int shift, const float *sums, float *dbias, unsigned tile, unsigned group, int lanes,
                                          float (*red)[33])
{
    const int c = (int)tile * 32 + (int)(threadIdx.x & 31), lane = (int)threadIdx.x >> 5;
    const Segment s = find_group(l.q, shift, group);
    if (s.group < 0) return;
    float all = 0.0f;
    if (c < l.N) {
        const float *const from = sums + (size_t)s.first * l.N + c;
        for (unsigned i0 = (unsigned)lane; i0 < s.unit; i0 += 64 * lanes) {   // sums of 64 values each
            float sum = 0.0f;
#pragma unroll 4
            for (unsigned i = i0; i < min(s.unit, i0 + 64 * lanes); i += lanes) sum += from[(size_t)i * l.N];
            all += sum;
        }
    }
    red[lane][threadIdx.x & 31] = all;
    __syncthreads();
    if (lane || c >= l.N) return;
    for (int i = 1; i < lanes; i++) all += red[i][threadIdx.x];
    dbias[(size_t)s.group * l.N + c] = all;
}

constexpr unsigned kGridRow = 65535;   // units along the second side of a grid; more go to the third
__device__ __forceinline__ unsigned unit_id() { return blockIdx.z * kGridRow + blockIdx.y; }
// Workgroups for so many tiles side by side: a multiple of eight, so that a tile of columns - and what it reads of a weight - stays on one XCD, unless that
// leaves XCDs with less to do or nothing.
inline size_t abreast(size_t tiles)
{
    const size_t eights = ceil_div(tiles, (size_t)8) * 8;
    return 5 * eights <= 6 * tiles ? eights : tiles;
}
inline dim3 grid_of(size_t tiles, size_t units)
{
    const size_t x = abreast(tiles);
    return dim3((unsigned)x, (unsigned)(units < kGridRow ? units : kGridRow), (unsigned)ceil_div(units, (size_t)kGridRow));
}

}  // namespace dopt
