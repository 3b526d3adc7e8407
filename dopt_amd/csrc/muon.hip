// Updates that treat a weight as a matrix: the momentum's orthogonalised form takes the place of the momentum.
// No counterpart in the reference, whose rules are elementwise (online/source/dopt/online/{sgd,adam,amsgrad}.d).
//
//     m' = mu m + g,  u = g + mu m' (nesterov) or m',  X = u / (|u| + 1e-7) in the 2-norm of all values
//     `iterations` times, on the side of fewer rows:  A = X X^T,  X' = a X + (b A + c A A) X
//     w' = (1 - lr decay) w - lr sqrt(max(1, rows / cols)) X
//
// All matrices of a handle go through each step in the same launches, so a network of twenty layers takes twenty launches and not
// hundreds.
//
// Iterations are taken in groups of up to three.  P(A) = a I + b A + c A A is a polynomial of A, so that all of
//     A1 = P0 A0 P0,  Q = P2 P1 P0,  X3 = Q X0
// are products of matrices that commute: inside a group only the small side's square matrices are multiplied, every result is
// symmetric (half of its tiles are formed, and stored twice), and X is read and written once per group: 6 s^2 l + 14 s^3
// operations for five iterations on [s, l] instead of 15 s^2 l + 5 s^3.  An error of A, 2^-24 of its largest eigenvalue, grows by
// a^2 with each iteration that A is carried on rather than formed again: within three by 142, to 1e-5 of a direction that is
// still weak; all five at once would make it 1e-2.  (A's diagonal is a sum of squares, which the matrix instruction lets drift downwards: parts of
// 262144 steps, those of [1 x 4194304], leave an update 4e-6 off, of 16384 steps 1e-6.)
//
// The products run on the fp16 matrix instruction with every value as the sum of two fp16 numbers, h = fp16(v) and
// l = fp16(v - h), of the three products h h + h l + l h that matter, in fp32 sums.  Two parts hold 22 bits, and l l is 2^-24 of
// h h on average: together half a bit more than fp32 rounds away from each product, with random signs.  fp16's small range does
// no harm here, where no value is large: |X| <= 1 by its scaling and the iteration keeps singular values below 1.21, so entries
// of X stay under 1.21, of A under 1.47, of P under 3.45 and of Q under 41, and are held times 2^13 (Q: 2^10); what lies below
// 2^-14 of fp16 loses bits only against 2^-34 of the largest entry possible.  That is half the matrix work of three bf16 parts,
// which the products of sgemm.hip need for operands of any size, and a value takes the four bytes that it takes in fp32.
//
// Operands run along the reduction: the square matrices are symmetric, and X is kept both as it is and transposed.  They lie in
// blocks of 32 rows by 16 steps, 2 KB one after the other along a row of blocks; a row of a block is 64 bytes, h and l parts of eight
// values (16 bytes each) and of the next eight.  So whatever a workgroup brings or stores are whole kilobytes in a line, spread
// over all channels of the L2: row by row, at a pitch of 2 KB, the rows of a tile met in two channels of sixteen and the products
// took three times as long.  Inside a row the four pieces lie at place piece ^ (row / 4 mod 4), in memory as in LDS, so that
// lanes which read the same piece of neighbouring rows touch different banks.
//
// Measured: VGG-16's sixteen matrices 448 to 465 us by the machine (39 for the momenta and 44 for X, at 5 TB/s; 66 for the two A and 15 for
// their parts, 129 for X after three and five iterations, 13 x 12.1 for square products, each a launch and what a CU takes in of its
// operands), eight of up to [640 x 5760] 760 to 810 (67, 83, 132, 18, 276, 13 x 15), one [64 x 576] 53.
#include <algorithm>
#include <cmath>
#include <cstring>
#include <new>
#include <vector>

#include "common.h"
#include "half_parts.h"

namespace {

using namespace dopt;

constexpr int kBlock = 256;
constexpr size_t kChunk = 8192;   // values per workgroup of the momentum's pass
constexpr float kA = 3.4445f, kB = -4.7750f, kC = 2.0315f, kEps = 1e-7f;
constexpr int kScaleBits = 13, kScaleBitsQ = 10, kSquares = 6, kGroup = 3;
constexpr float kUp = 0x1p13f;

struct Matrix {
    float *w;
    const float *g;
    float *m;
    float4 *partial;              // sums of parts of A's reduction
    double *parts;                // the momentum's pass: sums of squares
    int rows, cols;               // as w lies
    int s, l;                     // the shorter and the longer side: X is [s][l]
    int sp, lp;                   // ... in whole tiles
    int nparts, tall;             // tall: X is w transposed
    int quads;                    // tall, and rows of w are whole 16-byte pieces
    float wide;                   // sqrt(max(1, rows / cols))
};

enum Kind { kSmall, kMid, kWide };   // 64 x 64, 128 x 128, 128 x 256

// What a workgroup does, with all that it needs for its loads: looked up in a table of matrices, the addresses came a memory latency
// later.
struct Tile {
    char *sq, *x;          // the square matrices; X, X after a group of iterations, and their transposes
    int sp, lp;
    int job, i, j, kind;   // job < 0: nothing to do; kind: the tile's sides
    int from, to;          // the part of the reduction, in 32 steps
    int slot, parts;       // slot >= 0: where its sums wait for those of the other parts, in 16 KB
    __device__ char *square(int k) const { return sq + (size_t)k * sp * sp * 4; }
    __device__ char *along(int turn) const { return x + (size_t)turn * sp * lp * 4; }
    __device__ char *across(int turn) const { return x + (size_t)(2 + turn) * sp * lp * 4; }
};

struct Step {
    float mu, by, keep;
    int nesterov;
};

// d = alpha l r + beta c + gamma I, in square matrices by number; the factors take the matrices' scales along.
struct SquareOp {
    int l, r, d, c;
    float alpha, beta, gamma;
};
struct SquareOps {
    SquareOp op[2];   // by blockIdx.y: products that do not wait for each other
};

struct Handle {
    std::vector<Matrix> jobs;
    void *memory = nullptr;
    Matrix *d_jobs = nullptr;
    Tile *chunks = nullptr, *scales = nullptr, *grams = nullptr, *meets = nullptr, *squares = nullptr, *wides = nullptr;   // device
    unsigned nchunks = 0, nscales = 0, ngrams = 0, nmeets = 0, nsquares = 0, nwides = 0;
    bool small = false;   // no shorter side of more than 64
};

__device__ __forceinline__ float step_value(float g, float m, const Step &st) { return st.nesterov ? g + st.mu * m : m; }

// Bound by memory: reads g and m, writes m.
__global__ __launch_bounds__(kBlock) void muon_momentum_k(const Matrix *jobs, const Tile *chunks, Step st)
{
    const Tile t = chunks[blockIdx.x];
    const Matrix q = jobs[t.job];
    const size_t n = (size_t)q.rows * q.cols, from = (size_t)t.i * kChunk, to = min(from + kChunk, n);
    const Global<const float> g = global(q.g);
    const Global<float> m = global(q.m);
    double s = 0.0;
    if ((((uintptr_t)q.g | (uintptr_t)q.m) & 15) == 0) {
        constexpr int kQuads = kChunk / kBlock / 4;
        const size_t whole = from + (to - from) / 4 * 4;
        v4f a[kQuads], b[kQuads];
#pragma unroll
        for (int u = 0; u < kQuads; u++) {
            const size_t i = from + ((size_t)u * kBlock + threadIdx.x) * 4;
            if (i < whole) {
                a[u] = *(Global<const v4f>)(m + i);
                b[u] = *(Global<const v4f>)(g + i);
            }
        }
#pragma unroll
        for (int u = 0; u < kQuads; u++) {
            const size_t i = from + ((size_t)u * kBlock + threadIdx.x) * 4;
            if (i < whole) {
                const v4f v = {st.mu * a[u].x + b[u].x, st.mu * a[u].y + b[u].y, st.mu * a[u].z + b[u].z, st.mu * a[u].w + b[u].w};
                *(Global<v4f>)(m + i) = v;
                const double p = step_value(b[u].x, v.x, st), r = step_value(b[u].y, v.y, st), y = step_value(b[u].z, v.z, st),
                             z = step_value(b[u].w, v.w, st);
                s += (p * p + r * r) + (y * y + z * z);
            }
        }
        for (size_t i = whole + threadIdx.x; i < to; i += kBlock) {
            const float v = st.mu * m[i] + g[i];
            m[i] = v;
            const double p = step_value(g[i], v, st);
            s += p * p;
        }
    } else {
        for (size_t i = from + threadIdx.x; i < to; i += kBlock) {
            const float v = st.mu * m[i] + g[i];
            m[i] = v;
            const double p = step_value(g[i], v, st);
            s += p * p;
        }
    }
    __shared__ double red[4];
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) global(q.parts)[t.i] = (red[0] + red[1]) + (red[2] + red[3]);
}

// X = u / (|u| + eps), as it is and transposed, a 64 x 64 tile of w's layout per workgroup; zero outside.
__global__ __launch_bounds__(kBlock) void muon_scale_k(const Matrix *jobs, const Tile *tiles, Step st)
{
    __shared__ double red[kBlock / 64];
    __shared__ float tile[64][65];
    const Tile t = tiles[blockIdx.x];
    const Matrix q = jobs[t.job];
    double s = 0.0;
    for (int i = threadIdx.x; i < q.nparts; i += kBlock) s += global(q.parts)[i];
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    float v[16];
#pragma unroll
    for (int u = 0; u < 16; u++) {
        const int r = t.i * 64 + (int)(threadIdx.x >> 6) + 4 * u, c = t.j * 64 + (int)(threadIdx.x & 63);
        const size_t at = (size_t)r * q.cols + c;
        const size_t safe = r < q.rows && c < q.cols ? at : 0;   // (no branch: the loads go out together)
        v[u] = step_value(global(q.g)[safe], global(q.m)[safe], st);
    }
    __syncthreads();
    const float by = (float)((double)kUp / (sqrt((red[0] + red[1]) + (red[2] + red[3])) + (double)kEps));
    // times a power of two behind the rounding of the quotient; an infinite norm leaves NaN where u is not finite
#pragma unroll
    for (int u = 0; u < 16; u++) {
        const int r = (int)(threadIdx.x >> 6) + 4 * u;
        const bool in = t.i * 64 + r < q.rows && t.j * 64 + (int)(threadIdx.x & 63) < q.cols;
        tile[r][threadIdx.x & 63] = in ? v[u] * by : 0.0f;
    }
    __syncthreads();
    // rows of w's layout are rows of X, or of its transpose
    char *const along = q.tall ? t.across(0) : t.along(0), *const across = q.tall ? t.along(0) : t.across(0);
    const int along_p = q.tall ? q.sp : q.lp, across_p = q.tall ? q.lp : q.sp;   // steps of a row
#pragma unroll
    for (int u = 0; u < 2; u++) {   // a wavefront stores a block at a time
        const int r = (int)(threadIdx.x >> 1 & 31) + 32 * u, c = (int)(threadIdx.x >> 6) * 16 + (int)(threadIdx.x & 1) * 8;
        float p[8], o[8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            p[e] = tile[r][c + e];
            o[e] = tile[c + e][r];
        }
        const int piece = 2 * (threadIdx.x & 1), h = piece_at(r, piece), l = piece_at(r, piece + 1);
        v2u h0, l0, h1, l1;
        split4(p, h0, l0);
        split4(p + 4, h1, l1);
        Global<char> at = global(along + block_at(t.i * 64 + r, t.j * 64 + c, along_p));
        *(Global<v4u>)(at + h) = v4u{h0.x, h0.y, h1.x, h1.y};
        *(Global<v4u>)(at + l) = v4u{l0.x, l0.y, l1.x, l1.y};
        split4(o, h0, l0);
        split4(o + 4, h1, l1);
        at = global(across + block_at(t.j * 64 + r, t.i * 64 + c, across_p));
        *(Global<v4u>)(at + h) = v4u{h0.x, h0.y, h1.x, h1.y};
        *(Global<v4u>)(at + l) = v4u{l0.x, l0.y, l1.x, l1.y};
    }
}

enum Product { kGram, kSquare, kApply, kLast };

// Both operands of a tile go from memory to LDS as they lie, sixteen bytes a lane, with no register in between, in stages of 16 or 24 KB:
// four rows of blocks of 32 steps, eight of 16, or twelve of 16.  Up to five stages and two workgroups share a CU's 160 KB: what
// is on its way, about 100 KB per CU, hides a memory latency of more than a microsecond.  A CU takes in some 65 GB/s so, which is what
// bounds small tiles and makes wide ones worth their registers: X of eight [640 x 5760], 1.1 GB in tiles of 128 x 128.
constexpr int kLds = 81920;

// Four values in each of four neighbouring lanes: lane b gets value b of each.  `v` holds the values in pairs.
__device__ __forceinline__ v2u transpose4(v2u v, int lane)
{
    const bool hi = lane & 2, odd = lane & 1;
    unsigned p[4];
#define DOPT_FROM(k)                                                                                             \
    {                                                                                                            \
        const unsigned x = (unsigned)__builtin_amdgcn_mov_dpp((int)v.x, (k) * 0x55, 0xf, 0xf, true);             \
        const unsigned y = (unsigned)__builtin_amdgcn_mov_dpp((int)v.y, (k) * 0x55, 0xf, 0xf, true);             \
        const unsigned z = hi ? y : x;                                                                           \
        p[k] = odd ? z >> 16 : z & 0xffffu;                                                                      \
    }
    DOPT_FROM(0) DOPT_FROM(1) DOPT_FROM(2) DOPT_FROM(3)
#undef DOPT_FROM
    return v2u{p[0] | p[1] << 16, p[2] | p[3] << 16};
}

// A 32 x 32 tile of parts is two blocks, which a wavefront puts together in LDS as they lie in memory (eight bytes a lane straight
// to memory took four times the requests).  `row` runs to 32, `piece` along the columns to 8.
__device__ __forceinline__ void put_part(char *image, int row, int piece, int half, v2u v)
{
    *(v2u *)(image + (piece >> 2) * 2048 + piece_at(row, piece & 3) + 8 * half) = v;
}
__device__ __forceinline__ void store_image(const char *image, char *to, int lane)
{
#pragma unroll
    for (int k = 0; k < 4; k++) *(Global<v4u>)(global(to) + k * 1024 + lane * 16) = *(const v4u *)(image + k * 1024 + lane * 16);
}

// What a lane adds to a 32 x 32 tile of a square product at the end, asked for before it is needed.
struct Old {
    v2u h[4], l[4];
};
__device__ __forceinline__ void load_old(Old &o, const Tile &t, int c, int row0, int col0, int lane)
{
    const Global<const char> at = global((const char *)t.square(c) + block_at(col0, row0, t.sp) + 8 * (lane >> 5));
#pragma unroll
    for (int g = 0; g < 4; g++) {
        o.h[g] = *(Global<const v2u>)(at + (g >> 1) * 2048 + piece_at(lane, 2 * (g & 1)));
        o.l[g] = *(Global<const v2u>)(at + (g >> 1) * 2048 + piece_at(lane, 2 * (g & 1) + 1));
    }
}

// What the last product reads of a matrix, in registers: from the table, every store to w would have it read again.
struct W {
    Global<float> w;
    int s, l, tall, quads;
};

// A 32 x 32 tile of w, as a lane holds it.  Where all of it lies inside, there are no guards: each guarded load is waited for by
// itself.
struct TileOfW {
    int row0, col0;
    bool whole;
    float v[16];
    __device__ __forceinline__ Global<float> first(const W &q, int lane) const
    {
        const int r = row0 + 4 * (lane >> 5), c = col0 + (lane & 31);
        return q.w + (q.tall ? (size_t)c * q.s + r : (size_t)r * q.l + c);
    }
    __device__ __forceinline__ bool in(const W &q, int i, int lane) const { return row0 + acc_row(i, lane) < q.s && col0 + (lane & 31) < q.l; }
    __device__ __forceinline__ void load(const W &q, int lane, int row, int col)
    {
        row0 = row;
        col0 = col;
        whole = row + 32 <= q.s && col + 32 <= q.l;
        const Global<float> at = first(q, lane);
        const size_t step = q.tall ? 1 : (size_t)q.l;
        if (whole && q.quads) {
#pragma unroll
            for (int g = 0; g < 4; g++) {
                const v4f x = *(Global<const v4f>)(at + 8 * g);
#pragma unroll
                for (int e = 0; e < 4; e++) v[4 * g + e] = x[e];
            }
        } else if (whole) {
#pragma unroll
            for (int i = 0; i < 16; i++) v[i] = at[(8 * (i >> 2) + (i & 3)) * step];
        } else {
#pragma unroll
            for (int i = 0; i < 16; i++) v[i] = in(q, i, lane) ? at[(8 * (i >> 2) + (i & 3)) * step] : 0.0f;
        }
    }
    __device__ __forceinline__ void update(const W &q, int lane, float keep, float by, const v16f &acc)
    {
        const Global<float> at = first(q, lane);
        const size_t step = q.tall ? 1 : (size_t)q.l;
#pragma unroll
        for (int i = 0; i < 16; i++) v[i] = keep * v[i] - by * acc[i];
        if (whole && q.quads) {
#pragma unroll
            for (int g = 0; g < 4; g++) *(Global<v4f>)(at + 8 * g) = v4f{v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]};
        } else if (whole) {
#pragma unroll
            for (int i = 0; i < 16; i++) at[(8 * (i >> 2) + (i & 3)) * step] = v[i];
        } else {
#pragma unroll
            for (int i = 0; i < 16; i++)
                if (in(q, i, lane)) at[(8 * (i >> 2) + (i & 3)) * step] = v[i];
        }
    }
};

// The end of a 32 x 32 tile of a product at (row0, col0): a lane holds column `col` and rows r .. r + 3 of each of four groups.
// Values are stored row by row along the columns of the transpose ("across": four neighbouring values of the lane) and, exchanged
// between four lanes, along the rows.  `images`: 8 KB of LDS of the wavefront's own.
template <int kProduct>
__device__ __forceinline__ void finish(const Tile &t, const SquareOp &op, int turn, const v16f &acc, const Old &old, int row0, int col0, int lane,
                                       char *images)
{
    constexpr bool kSq = kProduct == kGram || kProduct == kSquare;
    if (kSq && row0 < col0) return;   // the other half of a tile on the diagonal stores this one
    const int c = lane & 31, col = col0 + c, half = lane >> 5;
#pragma unroll
    for (int g = 0; g < 4; g++) {
        const int r = 8 * g + 4 * half;
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = acc[4 * g + e] * op.alpha;
        if (kProduct == kSquare) {
            float o[4];
            join4(old.h[g], old.l[g], o);
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] += op.beta * o[e] + (row0 + r + e == col ? op.gamma : 0.0f);
        }
        v2u h, l;
        split4(v, h, l);
        put_part(images, c, 2 * g, half, h);
        put_part(images, c, 2 * g + 1, half, l);
        put_part(images + 4096, r + (lane & 3), 2 * (c >> 3), (c >> 2) & 1, transpose4(h, lane));
        put_part(images + 4096, r + (lane & 3), 2 * (c >> 3) + 1, (c >> 2) & 1, transpose4(l, lane));
    }
    char *const along = kSq ? t.square(op.d) : t.along(turn ^ 1), *const across = kSq ? t.square(op.d) : t.across(turn ^ 1);
    store_image(images, across + block_at(col0, row0, t.sp), lane);
    if (!kSq || row0 != col0) store_image(images + 4096, along + block_at(row0, col0, kSq ? t.sp : t.lp), lane);
}

// The sums of a 32 x 32 tile as four quads per lane.
__device__ __forceinline__ v4f quad_of(const v16f &a, int g) { return v4f{a[4 * g], a[4 * g + 1], a[4 * g + 2], a[4 * g + 3]}; }
__device__ __forceinline__ void set_quad(v16f &a, int g, v4f v)
{
    a[4 * g] = v.x;
    a[4 * g + 1] = v.y;
    a[4 * g + 2] = v.z;
    a[4 * g + 3] = v.w;
}

// What a wavefront does with its MI x NI tiles of 32 x 32 at (row0, col0).
template <int kProduct, int MI, int NI>
__device__ __forceinline__ void finish_all(const Matrix *jobs, const Tile &t, const Step &st, const SquareOp &op, int turn, const v16f (&acc)[MI][NI],
                                           int row0, int col0, int w, int lane, char *images)
{
    if (kProduct == kGram && t.slot >= 0) {
        const Global<v4f> to = (Global<v4f>)global(jobs[t.job].partial) + ((size_t)t.slot * 1024 + w * MI * NI * 256 + lane);
#pragma unroll
        for (int k = 0; k < MI * NI; k++)
#pragma unroll
            for (int g = 0; g < 4; g++) to[(k * 4 + g) * 64] = quad_of(acc[k / NI][k % NI], g);
        return;
    }
    if constexpr (kProduct == kLast) {
        const Matrix &m = jobs[t.job];
        const W q{global(m.w), m.s, m.l, m.tall, m.quads};
        const float by = st.by * m.wide * op.alpha;
        TileOfW a, b;   // one is updated while the next one arrives
        a.load(q, lane, row0, col0);
#pragma unroll
        for (int k = 0; k < MI * NI; k += 2) {
            if (k + 1 < MI * NI) b.load(q, lane, row0 + (k + 1) / NI * 32, col0 + (k + 1) % NI * 32);
            a.update(q, lane, st.keep, by, acc[k / NI][k % NI]);
            if (k + 2 < MI * NI) a.load(q, lane, row0 + (k + 2) / NI * 32, col0 + (k + 2) % NI * 32);
            if (k + 1 < MI * NI) b.update(q, lane, st.keep, by, acc[(k + 1) / NI % MI][(k + 1) % NI]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < MI; i++)
#pragma unroll
            for (int j = 0; j < NI; j++) {
                if (kProduct == kApply && col0 + 32 * j >= t.lp) continue;   // the end of X inside a tile
                Old old;
                if (kProduct == kSquare) load_old(old, t, op.c, row0 + 32 * i, col0 + 32 * j, lane);
                finish<kProduct>(t, op, turn, acc[i][j], old, row0 + 32 * i, col0 + 32 * j, lane, images);
            }
    }
}

template <int kProduct>
__global__ __launch_bounds__(kBlock, 2) void muon_product_k(const Matrix *jobs, const Tile *tiles, Step st, SquareOps ops, int turn)
{
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const Tile t = tiles[blockIdx.x];
    if (t.job < 0) return;
    const SquareOp op = ops.op[blockIdx.y];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), wm = w >> 1, wn = w & 1;
    const char *const left = kProduct == kGram ? t.along(turn) : t.square(op.l);
    const char *const right = kProduct == kGram ? t.along(turn) : kProduct == kSquare ? t.square(op.r) : t.across(turn);
    const int steps = kProduct == kGram ? t.lp : t.sp;   // of a row of both
    const size_t row_of_blocks = (size_t)steps * 128, from = (size_t)t.from * 4096;
    char *const images = lds + w * 8192;
    if (t.kind == kSmall) {   // four rows of blocks, one for each wavefront to bring; 32 steps a stage
        const char *const src = (w < 2 ? left + (size_t)(t.i * 2 + w) * row_of_blocks : right + (size_t)(t.j * 2 + w - 2) * row_of_blocks) + from;
        v16f acc[1][1];
        zero_acc(acc);
        pipeline<5, 16384, 4, 2, 2>(   // (two blocks of steps at a time)
            lds, t.to - t.from, [&](int k, char *to) { bring(src + (size_t)k * 4096, 4, lane, to + w * 4096); },
            [&](const char *now, Side<2> &a, Side<2> &b) {
                a.read(now + wm * 4096, lane);
                b.read(now + 8192 + wn * 4096, lane);
            },
            [&](const Side<2> &a, const Side<2> &b) {
#pragma unroll
                for (int s = 0; s < 2; s++) acc[0][0] = product(a.h[s], a.l[s], b.h[s], b.l[s], acc[0][0]);
            });
        finish_all<kProduct>(jobs, t, st, op, turn, acc, t.i * 64 + wm * 32, t.j * 64 + wn * 32, w, lane, images);
        return;
    }
    if constexpr (kProduct == kGram || kProduct == kSquare) {   // eight rows of blocks, two for each wavefront; 16 steps a stage
        const char *const src =
            (w < 2 ? left + (size_t)(t.i * 4 + 2 * w) * row_of_blocks : right + (size_t)(t.j * 4 + 2 * w - 4) * row_of_blocks) + from;
        v16f acc[2][2];
        zero_acc(acc);
        pipeline<5, 16384, 4, 2, 2>(
            lds, 2 * (t.to - t.from),
            [&](int k, char *to) {
                bring(src + (size_t)k * 2048, 2, lane, to + w * 4096);
                bring(src + row_of_blocks + (size_t)k * 2048, 2, lane, to + w * 4096 + 2048);
            },
            [&](const char *now, Side<2> &a, Side<2> &b) {
                a.read(now + wm * 4096, lane);
                b.read(now + 8192 + wn * 4096, lane);
            },
            [&](const Side<2> &a, const Side<2> &b) { multiply(a, b, acc); });
        finish_all<kProduct>(jobs, t, st, op, turn, acc, t.i * 128 + wm * 64, t.j * 128 + wn * 64, w, lane, images);
    } else {   // four rows of blocks on the left, eight on the right (the last one again where X ends), three for each wavefront
        const int last = t.lp / 32 - 1;
        const char *src[3];
#pragma unroll
        for (int b = 0; b < 3; b++) {
            const int r = 3 * w + b;
            src[b] = (r < 4 ? left + (size_t)(t.i * 4 + r) * row_of_blocks : right + (size_t)min(t.j * 8 + r - 4, last) * row_of_blocks) + from;
        }
        v16f acc[2][4];
        zero_acc(acc);
        pipeline<3, 24576, 6, 2, 4>(
            lds, 2 * (t.to - t.from),
            [&](int k, char *to) {
#pragma unroll
                for (int b = 0; b < 3; b++) bring(src[b] + (size_t)k * 2048, 2, lane, to + (3 * w + b) * 2048);
            },
            [&](const char *now, Side<2> &a, Side<4> &b) {
                a.read(now + wm * 4096, lane);
                b.read(now + 8192 + wn * 8192, lane);
            },
            [&](const Side<2> &a, const Side<4> &b) { multiply(a, b, acc); });
        finish_all<kProduct>(jobs, t, st, op, turn, acc, t.i * 128 + wm * 64, t.j * 256 + wn * 128, w, lane, images);
    }
}

// Adds the parts of 64 x 64 values of A, in their order.
__global__ __launch_bounds__(kBlock) void muon_meet_k(const Matrix *jobs, const Tile *tiles, SquareOps ops)
{
    __shared__ __attribute__((aligned(16))) char images[4 * 8192];
    const Tile t = tiles[blockIdx.x];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const Global<const v4f> from = (Global<const v4f>)global((const float4 *)jobs[t.job].partial) + ((size_t)t.slot * 1024 + w * 256 + lane);
    const size_t step = t.kind == kSmall ? 1024 : 4096;
    v16f sum;
#pragma unroll
    for (int g = 0; g < 4; g++) set_quad(sum, g, v4f{0.0f, 0.0f, 0.0f, 0.0f});
    for (int p = 0; p < t.parts; p++)
#pragma unroll
        for (int g = 0; g < 4; g++) set_quad(sum, g, quad_of(sum, g) + from[p * step + g * 64]);
    finish<kGram>(t, ops.op[0], 0, sum, Old{}, t.i * 64 + (w >> 1) * 32, t.j * 64 + (w & 1) * 32, lane, images + w * 8192);
}

// The square products of a group of iterations for matrices whose shorter side is at most 64: everything in one workgroup's LDS, a
// product and a barrier after the other, where thirteen launches of a tile each took 3.6 us.  Adds the parts of A first; the
// last product goes to memory.
constexpr int kChainOps = 16;
struct Chain {
    SquareOp op[kChainOps];
    int n, a, q;   // how many; where A goes, and which one is wanted
};
__global__ __launch_bounds__(kBlock) void muon_chain_k(const Matrix *jobs, const Tile *tiles, Chain ch)
{
    extern __shared__ __attribute__((aligned(16))) char lds[];   // kSquares matrices of 16 KB: four blocks along, two down
    const Tile t = tiles[blockIdx.x];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), wm = w >> 1, wn = w & 1;
    const int c = lane & 31, half = lane >> 5;
    // (row, col) lies in blocks 4 (row / 32) + col / 16; what is below the diagonal is stored twice, what is above not formed
    auto store = [&](char *to, const v16f &acc, float alpha, float beta, const char *old, float gamma) {
        if (wm < wn) return;
        char *const across = to + wn * 8192 + wm * 4096, *const along = to + wm * 8192 + wn * 4096;
        const char *const at = old + wn * 8192 + wm * 4096;
#pragma unroll
        for (int g = 0; g < 4; g++) {
            const int r = 8 * g + 4 * half, place = (g >> 1) * 2048 + 8 * half;
            const int hp = piece_at(c, 2 * (g & 1)), lp = piece_at(c, 2 * (g & 1) + 1);
            float o[4], v[4];
            join4(*(const v2u *)(at + place + hp), *(const v2u *)(at + place + lp), o);
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] = acc[4 * g + e] * alpha + (beta * o[e] + (wm == wn && r + e == c ? gamma : 0.0f));
            v2u h, l;
            split4(v, h, l);
            put_part(across, c, 2 * g, half, h);
            put_part(across, c, 2 * g + 1, half, l);
            if (wm == wn) continue;
            put_part(along, r + (lane & 3), 2 * (c >> 3), (c >> 2) & 1, transpose4(h, lane));
            put_part(along, r + (lane & 3), 2 * (c >> 3) + 1, (c >> 2) & 1, transpose4(l, lane));
        }
    };
    {   // A: the sum of its parts
        const Global<const v4f> from = (Global<const v4f>)global((const float4 *)jobs[t.job].partial) + ((size_t)t.slot * 1024 + w * 256 + lane);
        v16f sum;
#pragma unroll
        for (int g = 0; g < 4; g++) set_quad(sum, g, v4f{0.0f, 0.0f, 0.0f, 0.0f});
        for (int p = 0; p < t.parts; p++)
#pragma unroll
            for (int g = 0; g < 4; g++) set_quad(sum, g, quad_of(sum, g) + from[p * 1024 + g * 64]);
        // (beta is zero: what is read beside it only has to be a number)
        for (int i = threadIdx.x; i < kSquares * 1024; i += kBlock) ((v4u *)lds)[i] = v4u{0, 0, 0, 0};
        meet();
        store(lds + ch.a * 16384, sum, ch.op[0].gamma, 0.0f, lds + ch.a * 16384, 0.0f);
    }
    for (int k = 1; k < ch.n; k++) {
        meet();
        const SquareOp op = ch.op[k];
        v16f acc[1][1];
        zero_acc(acc);
        if (wm >= wn) {
#pragma unroll
            for (int s = 0; s < 4; s++)
                multiply(lds + op.l * 16384 + wm * 8192 + s * 2048, lds + op.r * 16384 + wn * 8192 + s * 2048, lane, acc);
        }
        store(lds + op.d * 16384, acc[0][0], op.alpha, op.beta, lds + op.c * 16384, op.gamma);
    }
    meet();
    const Global<char> to = global(t.square(ch.q));
#pragma unroll
    for (int i = 0; i < 4; i++) *(Global<v4u>)(to + (i * kBlock + threadIdx.x) * 16) = *(const v4u *)(lds + ch.q * 16384 + (i * kBlock + threadIdx.x) * 16);
}

// No iterations: w moves along X itself.
__global__ __launch_bounds__(kBlock) void muon_plain_k(const Matrix *jobs, const Tile *chunks, Step st)
{
    const Tile t = chunks[blockIdx.x];
    const Matrix q = jobs[t.job];
    const size_t n = (size_t)q.rows * q.cols, from = (size_t)t.i * kChunk, to = min(from + kChunk, n);
    const float by = st.by * q.wide * (1.0f / kUp);
    for (size_t i = from + threadIdx.x; i < to; i += kBlock) {
        const int r = (int)(i / q.cols), c = (int)(i % q.cols), piece = 2 * (c >> 3 & 1);
        const char *const at = (q.tall ? t.across(0) : t.along(0)) + block_at(r, c, q.tall ? q.sp : q.lp) + 2 * (c & 7);
        const float x = (float)*(const _Float16 *)(at + piece_at(r, piece)) + (float)*(const _Float16 *)(at + piece_at(r, piece + 1));
        q.w[i] = st.keep * q.w[i] - by * x;
    }
}

// Tiles in the order in which the workgroups are handed out: each of the eight XCDs gets neighbouring tiles (they share
// operands in its L2) of about an eighth of the whole cost, the costliest first.
std::vector<Tile> deal(const std::vector<Tile> &tiles, const std::vector<double> &cost)
{
    double total = 0, sum = 0;
    for (double c : cost) total += c;
    std::vector<std::vector<size_t>> xcd(8);
    for (size_t i = 0; i < tiles.size(); i++) {
        xcd[std::min<size_t>(7, (size_t)((sum + cost[i] / 2) / total * 8))].push_back(i);
        sum += cost[i];
    }
    size_t most = 0;
    for (auto &x : xcd) {
        std::stable_sort(x.begin(), x.end(), [&](size_t a, size_t b) { return cost[a] > cost[b]; });
        most = std::max(most, x.size());
    }
    std::vector<Tile> out;
    Tile nothing{};
    nothing.job = -1;
    for (size_t k = 0; k < most; k++)
        for (auto &x : xcd) out.push_back(k < x.size() ? tiles[x[k]] : nothing);
    return out;
}

void release(Handle *h)
{
    dopt_hip_free(h->memory);
    delete h;
}

int build(Handle *h)
{
    size_t bytes = 0;
    auto take = [&](size_t n) { const size_t at = bytes; bytes += ceil_div(n, (size_t)256) * 256; return at; };
    std::vector<size_t> x_at, sq_at, partial_at, parts_at;
    size_t all = 0, longest = 0, mids = 0;   // stages of all tiles of A, of one; 128 x 128 tiles of square matrices
    h->small = true;
    for (Matrix &q : h->jobs) {
        q.tall = q.rows > q.cols;
        q.s = std::min(q.rows, q.cols);
        q.l = std::max(q.rows, q.cols);
        const int side = q.s <= 64 ? 64 : 128;
        q.sp = (int)ceil_div((size_t)q.s, (size_t)side) * side;
        q.lp = (int)ceil_div((size_t)q.l, (size_t)side) * side;
        q.quads = q.tall && q.cols % 4 == 0 && aligned16(q.w);
        q.wide = std::sqrt(std::max(1.0f, (float)q.rows / (float)q.cols));
        q.nparts = (int)ceil_div((size_t)q.rows * q.cols, kChunk);
        const size_t t = q.sp / side, tiles = t * (t + 1) / 2;
        const size_t stages = (size_t)(q.lp / 32) * (side / 64);   // (one of a 128 x 128 tile is 16 steps)
        all += tiles * stages;
        longest = std::max(longest, stages);
        mids += side == 128 ? tiles : 0;
        h->small = h->small && side == 64;
    }
    // A's reduction is cut so that three workgroups for every two CUs have about the same to do (us for VGG-16's matrices and for eight of
    // [640 x 5760]: one for each CU 456 and 785, three for two 449 and 776, two 468 and 809).  Where one workgroup adds the
    // parts for its whole chain there are sixteen at most: eight of [64 x 8192] take 110 us, in sixty-four parts each 140.
    const size_t part = std::max(h->small ? std::max((size_t)4, longest / 16) : (size_t)32, ceil_div(all * 2, (size_t)num_cus() * 3));
    auto cuts_of = [&](const Matrix &q) { return (int)ceil_div((size_t)q.lp / 32 * (q.sp == 64 ? 1 : 2), part); };
    // 64 x 64 tiles spread a short product over more CUs, 128 x 128 tiles take half the operands' traffic (whole updates, us, in the former
    // and the latter: one [512 x 512] 207 and 343, eight [640 x 5760] 827 and 929, eight [1024 x 1024], 288 of the large
    // tiles, 901 and 874, two [2048 x 2048] 1555 and 1449).
    const bool mid_squares = mids >= (size_t)num_cus();
    for (const Matrix &q : h->jobs) {
        const size_t side = q.sp == 64 ? 64 : 128, t = q.sp / side, cuts = cuts_of(q);
        x_at.push_back(take((size_t)q.sp * q.lp * 4 * 4));
        sq_at.push_back(take((size_t)q.sp * q.sp * 4 * kSquares));
        partial_at.push_back(take(cuts > 1 || h->small ? cuts * t * (t + 1) / 2 * side * side * sizeof(float) : 0));
        parts_at.push_back(take((size_t)q.nparts * sizeof(double)));
    }
    const size_t tables_at = bytes;
    std::vector<Tile> chunks, scales, grams, meets, squares, wides;
    std::vector<double> cgram, csq, cwide;
    for (size_t k = 0; k < h->jobs.size(); k++) {   // (addresses are offsets until the memory is there)
        const Matrix &q = h->jobs[k];
        const bool small = q.sp == 64;
        const int side = small ? 64 : 128, deep = q.lp / 32, cuts = cuts_of(q);
        const int rp = q.tall ? q.lp : q.sp, cp = q.tall ? q.sp : q.lp;
        Tile t{(char *)sq_at[k], (char *)x_at[k], q.sp, q.lp, (int)k, 0, 0, kSmall, 0, q.sp / 32, -1, 0};
        auto at = [&](int i, int j) { t.i = i; t.j = j; return t; };
        for (int i = 0; i < q.nparts; i++) chunks.push_back(at(i, 0));
        for (int i = 0; i < rp / 64; i++)
            for (int j = 0; j < cp / 64; j++) scales.push_back(at(i, j));
        t.kind = mid_squares && !small ? kMid : kSmall;
        for (int i = 0; i < q.sp / (t.kind == kMid ? 128 : 64); i++)
            for (int j = 0; j <= i; j++) {
                squares.push_back(at(i, j));
                csq.push_back((double)(q.sp + 256) * (t.kind == kMid ? 2 : 1));
            }
        t.kind = small ? kSmall : kMid;
        int slots = 0;
        for (int i = 0; i < q.sp / side; i++)
            for (int j = 0; j <= i; j++) {
                Tile g = at(i, j);
                if (cuts > 1 || h->small) {   // its quarters of 64 x 64, on and below the diagonal
                    g.parts = cuts;
                    for (int p = 0; p < (small ? 1 : 4); p++) {
                        g.slot = slots + p;
                        g.i = small ? i : 2 * i + p / 2;
                        g.j = small ? j : 2 * j + p % 2;
                        if (g.i >= g.j) meets.push_back(g);
                    }
                    g = at(i, j);
                }
                for (int c = 0; c < cuts; c++) {
                    g.from = (int)((size_t)deep * c / cuts);
                    g.to = (int)((size_t)deep * (c + 1) / cuts);
                    if (cuts > 1 || h->small) {
                        g.slot = slots;
                        slots += small ? 1 : 4;
                    }
                    grams.push_back(g);
                    cgram.push_back((double)(g.to - g.from) * (small ? 1 : 2) + 8);
                }
            }
        t.kind = small ? kSmall : kWide;
        for (int j = 0; j < (int)ceil_div((size_t)q.lp, (size_t)(small ? 64 : 256)); j++)
            for (int i = 0; i < q.sp / side; i++) {
                wides.push_back(at(i, j));
                cwide.push_back((double)(q.sp + 256) * (small ? 1 : 4));
            }
    }
    grams = deal(grams, cgram);
    squares = deal(squares, csq);
    wides = deal(wides, cwide);
    struct Table {
        std::vector<Tile> *tiles;
        Tile **device;
        unsigned *n;
        size_t at;
    } tables[] = {{&chunks, &h->chunks, &h->nchunks, 0}, {&scales, &h->scales, &h->nscales, 0},    {&grams, &h->grams, &h->ngrams, 0},
                  {&meets, &h->meets, &h->nmeets, 0},    {&squares, &h->squares, &h->nsquares, 0}, {&wides, &h->wides, &h->nwides, 0}};
    for (Table &t : tables) t.at = take(t.tiles->size() * sizeof(Tile));
    const size_t jobs_at = take(h->jobs.size() * sizeof(Matrix));
    if (int rc = scratch_alloc(&h->memory, bytes)) return rc;
    char *const base = (char *)h->memory;
    for (size_t k = 0; k < h->jobs.size(); k++) {
        h->jobs[k].partial = (float4 *)(base + partial_at[k]);
        h->jobs[k].parts = (double *)(base + parts_at[k]);
    }
    // the tables and the matrices lie one after the other: one copy
    std::vector<char> host(bytes - tables_at);
    for (Table &t : tables) {
        for (Tile &q : *t.tiles) {
            q.sq = base + (size_t)q.sq;
            q.x = base + (size_t)q.x;
        }
        *t.device = (Tile *)(base + t.at);
        *t.n = (unsigned)t.tiles->size();
        if (!t.tiles->empty()) memcpy(host.data() + (t.at - tables_at), t.tiles->data(), t.tiles->size() * sizeof(Tile));
    }
    h->d_jobs = (Matrix *)(base + jobs_at);
    memcpy(host.data() + (jobs_at - tables_at), h->jobs.data(), h->jobs.size() * sizeof(Matrix));
    return dopt_hip_copy_h2d(base + tables_at, host.data(), host.size());
}

template <int kProduct>
int launch(const Handle *h, unsigned blocks, unsigned products, const Tile *tiles, const Step &st, const SquareOps &ops, int turn)
{
    static bool raised = false;   // above 64 KB of dynamic LDS a kernel has to be told once
    if (!raised) DOPT_HIP_CHECK(hipFuncSetAttribute((const void *)muon_product_k<kProduct>, hipFuncAttributeMaxDynamicSharedMemorySize, kLds));
    raised = true;
    hipLaunchKernelGGL(muon_product_k<kProduct>, dim3(blocks, products), dim3(kBlock), kLds, stream(), h->d_jobs, tiles, st, ops, turn);
    DOPT_LAUNCH_CHECK();
    return DOPT_HIP_OK;
}

// Which of the square matrices hold something that is still read, and the powers of two that they are held times.
struct Buffers {
    bool used[kSquares] = {};
    int bits[kSquares] = {};
    int take(int b)
    {
        int i = 0;
        while (used[i]) i++;
        used[i] = true;
        bits[i] = b;
        return i;
    }
    void drop(int i) { used[i] = false; }
    // d = by l r + beta c + gamma I
    SquareOp op(float by, int l, int r, float beta, int c, float gamma, int d) const
    {
        return SquareOp{l, r, d, c, std::ldexp(by, bits[d] - bits[l] - bits[r]), std::ldexp(beta, bits[d] - bits[c]), std::ldexp(gamma, bits[d])};
    }
};

// The square products of `count` iterations, in their order: f(operations, how many of them do not wait for each other).  Returns where
// Q is left.
template <class F>
int squares_of(int count, Buffers &b, int a, F &&f, int *q_out)
{
    SquareOps ops{};
    int q = -1;
    for (int k = 0; k < count; k++) {
        const int p = b.take(kScaleBits);
        ops.op[0] = b.op(kC, a, a, kB, a, kA, p);   // P
        if (int rc = f(ops, 1)) return rc;
        unsigned n = 0;
        const int before = q;
        if (q >= 0) {   // Q <- P Q
            const int next = b.take(kScaleBitsQ);
            ops.op[n++] = b.op(1.0f, p, q, 0.0f, q, 0.0f, next);
            q = next;
        } else {
            q = p;
        }
        if (k + 1 < count) {   // A <- P A P
            const int t = b.take(kScaleBits);
            ops.op[n++] = b.op(1.0f, p, a, 0.0f, a, 0.0f, t);
            if (int rc = f(ops, n)) return rc;
            const int next = b.take(kScaleBits);
            ops.op[0] = b.op(1.0f, t, p, 0.0f, a, 0.0f, next);
            if (int rc = f(ops, 1)) return rc;
            b.drop(a);
            b.drop(t);
            a = next;
        } else if (n) {
            if (int rc = f(ops, n)) return rc;
        }
        if (before >= 0) {
            b.drop(before);
            b.drop(p);
        }
    }
    *q_out = q;
    return DOPT_HIP_OK;
}

// `count` iterations on X[turn]: into X[turn ^ 1], or into w.
int iterate(const Handle *h, const Step &st, int count, int turn, bool last)
{
    Buffers b;
    const int a = b.take(kScaleBits);
    int q = a;
    SquareOps ops{};
    const float alpha = std::ldexp(1.0f, -kScaleBits);
    ops.op[0] = SquareOp{0, 0, a, 0, alpha, 0.0f, 0.0f};
    if (int rc = launch<kGram>(h, h->ngrams, 1, h->grams, st, ops, turn)) return rc;
    if (h->small) {
        Chain ch{};
        ch.a = a;
        ch.op[ch.n++].gamma = alpha;
        static_assert(1 + 3 * kGroup + (kGroup - 1) <= kChainOps, "an iteration has up to four products");
        if (int rc = squares_of(
                count, b, a,
                [&](const SquareOps &o, unsigned n) {
                    for (unsigned i = 0; i < n; i++) ch.op[ch.n++] = o.op[i];
                    return (int)DOPT_HIP_OK;
                },
                &q))
            return rc;
        ch.q = q;
        static bool raised = false;
        if (!raised) DOPT_HIP_CHECK(hipFuncSetAttribute((const void *)muon_chain_k, hipFuncAttributeMaxDynamicSharedMemorySize, kSquares * 16384));
        raised = true;
        hipLaunchKernelGGL(muon_chain_k, dim3(h->nmeets), dim3(kBlock), kSquares * 16384, stream(), h->d_jobs, h->meets, ch);
        DOPT_LAUNCH_CHECK();
    } else {
        if (h->nmeets) {
            hipLaunchKernelGGL(muon_meet_k, dim3(h->nmeets), dim3(kBlock), 0, stream(), h->d_jobs, h->meets, ops);
            DOPT_LAUNCH_CHECK();
        }
        if (int rc = squares_of(
                count, b, a, [&](const SquareOps &o, unsigned n) { return launch<kSquare>(h, h->nsquares, n, h->squares, st, o, turn); }, &q))
            return rc;
    }
    ops.op[0] = SquareOp{q, 0, 0, 0, std::ldexp(1.0f, (last ? -kScaleBits : 0) - b.bits[q]), 0.0f, 0.0f};
    return last ? launch<kLast>(h, h->nwides, 1, h->wides, st, ops, turn) : launch<kApply>(h, h->nwides, 1, h->wides, st, ops, turn);
}

}  // namespace

extern "C" {

int dopt_hip_muon_create(int nmatrices, const dopt_hip_matrix_ref *refs, void **handle)
{
    DOPT_REQUIRE(handle != nullptr, "dopt_hip_muon_create: handle is null");
    *handle = nullptr;
    DOPT_REQUIRE(nmatrices >= 0 && (nmatrices == 0 || refs), "dopt_hip_muon_create: bad list of matrices");
    for (int i = 0; i < nmatrices; i++) {
        const dopt_hip_matrix_ref &r = refs[i];
        DOPT_REQUIRE(r.rows <= ((size_t)1 << 28) && r.cols <= ((size_t)1 << 28) && r.rows * r.cols <= ((size_t)1 << 28) &&
                         std::min(r.rows, r.cols) <= 16384,
                     "dopt_hip_muon_create: matrix %d is too large", i);
        const size_t n = r.rows * r.cols;
        DOPT_REQUIRE(n == 0 || (r.w && r.g && r.m), "dopt_hip_muon_create: matrix %d has a null w, g or m", i);
        // all matrices are updated at the same time: what one writes nobody else may read or write
        const size_t bytes = n * sizeof(float);
        for (int j = 0; j <= i; j++) {
            const dopt_hip_matrix_ref &q = refs[j];
            const size_t k = q.rows * q.cols * sizeof(float);
            const void *written[] = {r.w, r.m}, *theirs[] = {q.w, q.m, q.g};
            bool shared = overlaps(r.g, bytes, q.w, k) || overlaps(r.g, bytes, q.m, k);
            for (int a = 0; a < 2; a++)
                for (int b = 0; b < 3; b++) shared = shared || ((i != j || a != b) && overlaps(written[a], bytes, theirs[b], k));
            DOPT_REQUIRE(!shared, "dopt_hip_muon_create: matrices %d and %d share memory that is written", j, i);
        }
    }
    DOPT_ENSURE_INIT();
    Handle *h = new (std::nothrow) Handle();
    if (!h) return fail(DOPT_HIP_ERR_OOM, "dopt_hip_muon_create: out of host memory");
    int rc;
    try {
        for (int i = 0; i < nmatrices; i++) {
            const dopt_hip_matrix_ref &r = refs[i];
            if (r.rows * r.cols == 0) continue;
            Matrix q{};
            q.w = r.w;
            q.g = r.g;
            q.m = r.m;
            q.rows = (int)r.rows;
            q.cols = (int)r.cols;
            h->jobs.push_back(q);
        }
        rc = h->jobs.empty() ? DOPT_HIP_OK : build(h);
    } catch (const std::bad_alloc &) {
        rc = fail(DOPT_HIP_ERR_OOM, "dopt_hip_muon_create: out of host memory");
    }
    if (rc) {
        release(h);
        return rc;
    }
    *handle = h;
    return DOPT_HIP_OK;
}

int dopt_hip_muon_destroy(void *handle)
{
    if (handle) release((Handle *)handle);
    return DOPT_HIP_OK;
}

int dopt_hip_muon_step(void *handle, float lr, float mu, int nesterov, float decay, int iterations)
{
    DOPT_REQUIRE(handle != nullptr, "dopt_hip_muon_step: handle is null");
    DOPT_REQUIRE(iterations >= 0 && iterations <= 100, "dopt_hip_muon_step: %d iterations", iterations);
    const Handle *const h = (const Handle *)handle;
    if (h->jobs.empty()) return DOPT_HIP_OK;
    const Step st{mu, lr, 1.0f - lr * decay, nesterov != 0};
    hipLaunchKernelGGL(muon_momentum_k, dim3(h->nchunks), dim3(kBlock), 0, stream(), h->d_jobs, h->chunks, st);
    hipLaunchKernelGGL(muon_scale_k, dim3(h->nscales), dim3(kBlock), 0, stream(), h->d_jobs, h->scales, st);
    DOPT_LAUNCH_CHECK();
    if (iterations == 0) {
        hipLaunchKernelGGL(muon_plain_k, dim3(h->nchunks), dim3(kBlock), 0, stream(), h->d_jobs, h->chunks, st);
        DOPT_LAUNCH_CHECK();
    }
    const int groups = (iterations + kGroup - 1) / kGroup;
    for (int k = 0, done = 0; k < groups; k++) {
        const int count = (iterations - done + groups - k - 1) / (groups - k);   // the longer groups first
        if (int rc = iterate(h, st, count, k & 1, k + 1 == groups)) return rc;
        done += count;
    }
    return DOPT_HIP_OK;
}

}  // extern "C"
