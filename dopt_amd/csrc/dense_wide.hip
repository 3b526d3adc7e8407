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

#include "dense_wide.h"

namespace {

using namespace dopt;

// Operands that lie across the reduction, [K][rows]: the largest values of runs of K for each column, then a tile of 64 steps by 64 columns
// per workgroup, turned in LDS.
constexpr int kRuns = 32, kAcross = 3;
struct Layout {
    Operand rows[2], across[kAcross];
    int nrows, nacross;
    DenseFold fold;   // rides behind them
};

__global__ __launch_bounds__(256) void wide_tops_k(Tops t) { column_tops(t, blockIdx.x); }

__global__ __launch_bounds__(1024) void wide_layout_k(Layout l)
{
    unsigned block = blockIdx.x;
    for (int i = 0; i < l.nrows; i++) {
        if (block < l.rows[i].blocks) return split_rows(l.rows[i], (size_t)block * 4, (size_t)block * 4);
        block -= l.rows[i].blocks;
    }
    for (int i = 0; i < l.nacross; i++) {
        if (block < l.across[i].blocks) {
            const unsigned tiles = (unsigned)(l.across[i].padded / 64);
            return turn_tile(l.across[i], (size_t)(block % tiles) * 64, (size_t)(block / tiles) * 64);
        }
        block -= l.across[i].blocks;
    }
    dense_fold(l.fold, block);
}

struct Wides {
    Wide q[2];
    unsigned per[2];   // an XCD's workgroups of each
};

template <int kTile, bool kPasses>
__global__ __launch_bounds__(2 * kTile, 2) void wide_product_k(Wides both, DenseEpilogue ep)
{
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
    wide_tile<kTile, kPasses>(q, ep, y, mt, nt, from, to, place_of_tile, lds);
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
