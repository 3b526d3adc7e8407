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
// still weak; all five at once would make it 1e-2.
//
// The products run on the fp16 matrix instruction with every value as the sum of two fp16 numbers, h = fp16(v) and
// l = fp16(v - h), of the three products h h + h l + l h that matter, in fp32 sums.  Two parts hold 22 bits, and l l is 2^-24 of
// h h on average: together half a bit more than fp32 rounds away from each product, with random signs.  fp16's small range does
// no harm here, where no value is large: |X| <= 1 by its scaling and the iteration keeps singular values below 1.21, so entries
// of X stay under 1.21, of A under 1.47, of P under 3.45 and of Q under 41, and are held times 2^13 (Q: 2^10); what lies below
// 2^-14 of fp16 loses bits only against 2^-34 of the largest entry possible.  That is half the matrix work of three bf16 parts,
// which the products of sgemm.hip need for operands of any size, and a value takes the four bytes that it takes in fp32.
//
// Operands lie row by row along the reduction in pieces of eight values: their h parts (16 bytes), then their l parts.  The square
// matrices are symmetric, so all products are of that form once X is kept both as it is and transposed.
#include <algorithm>
#include <cmath>
#include <new>
#include <vector>

#include "common.h"
#include "mfma_core.h"

namespace {

using namespace dopt;

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v4h __attribute__((ext_vector_type(4)));
using lds_ptr = __attribute__((address_space(3))) void *;
using glb_ptr = __attribute__((address_space(1))) const void *;

constexpr int kBlock = 256;
constexpr size_t kChunk = 8192;   // values per workgroup of the momentum's pass
constexpr float kA = 3.4445f, kB = -4.7750f, kC = 2.0315f, kEps = 1e-7f;
constexpr int kScaleBits = 13, kScaleBitsQ = 10, kSquares = 6, kGroup = 3;
constexpr float kUp = 0x1p13f;

struct Matrix {
    float *w;
    const float *g;
    float *m;
    char *x[2], *xt[2];           // X and its transpose before and after a group of iterations
    char *sq[kSquares];           // the square matrices
    float4 *partial;              // sums of parts of A's reduction
    double *parts;                // the momentum's pass: sums of squares
    int rows, cols;               // as w lies
    int s, l;                     // the shorter and the longer side: X is [s][l]
    int sp, lp;                   // ... in whole tiles
    int nparts, tall;             // tall: X is w transposed
    float wide;                   // sqrt(max(1, rows / cols))
};

struct Tile {
    int job, i, j, big;    // job < 0: nothing to do
    int from, to;          // the part of the reduction, in 64 steps
    int slot, parts;       // slot >= 0: where its sums wait for those of the other parts
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
};

__device__ __forceinline__ float step_value(float g, float m, const Step &st) { return st.nesterov ? g + st.mu * m : m; }

// Bound by memory: reads g and m, writes m.
__global__ __launch_bounds__(kBlock) void muon_momentum_k(const Matrix *jobs, const Tile *chunks, Step st)
{
    const Tile t = chunks[blockIdx.x];
    const Matrix &q = jobs[t.job];
    const size_t n = (size_t)q.rows * q.cols, from = (size_t)t.i * kChunk, to = min(from + kChunk, n);
    const float *const g = q.g;
    float *const m = q.m;
    double s = 0.0;
    if ((((uintptr_t)g | (uintptr_t)m) & 15) == 0) {
        constexpr int kQuads = kChunk / kBlock / 4;
        const size_t whole = from + (to - from) / 4 * 4;
        float4 a[kQuads], b[kQuads];
#pragma unroll
        for (int u = 0; u < kQuads; u++) {
            const size_t i = from + ((size_t)u * kBlock + threadIdx.x) * 4;
            if (i < whole) {
                a[u] = *(const float4 *)(m + i);
                b[u] = *(const float4 *)(g + i);
            }
        }
#pragma unroll
        for (int u = 0; u < kQuads; u++) {
            const size_t i = from + ((size_t)u * kBlock + threadIdx.x) * 4;
            if (i < whole) {
                float4 v = make_float4(st.mu * a[u].x + b[u].x, st.mu * a[u].y + b[u].y, st.mu * a[u].z + b[u].z, st.mu * a[u].w + b[u].w);
                *(float4 *)(m + i) = v;
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
    if (threadIdx.x == 0) q.parts[t.i] = (red[0] + red[1]) + (red[2] + red[3]);
}

// Four values, already times kUp, as their h and l parts.
__device__ __forceinline__ void split4(const float *v, uint2 &h, uint2 &l)
{
    v4h a, b;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        a[e] = (_Float16)v[e];
        b[e] = (_Float16)(v[e] - (float)a[e]);
    }
    h = __builtin_bit_cast(uint2, a);
    l = __builtin_bit_cast(uint2, b);
}

__device__ __forceinline__ void join4(uint2 h, uint2 l, float *v)
{
    const v4h a = __builtin_bit_cast(v4h, h), b = __builtin_bit_cast(v4h, l);
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] = (float)a[e] + (float)b[e];
}

// X = u / (|u| + eps), as it is and transposed, a 64 x 64 tile of w's layout per workgroup; zero outside.
__global__ __launch_bounds__(kBlock) void muon_scale_k(const Matrix *jobs, const Tile *tiles, Step st)
{
    __shared__ double red[kBlock / 64];
    __shared__ float tile[64][65];
    const Tile t = tiles[blockIdx.x];
    const Matrix &q = jobs[t.job];
    double s = 0.0;
    for (int i = threadIdx.x; i < q.nparts; i += kBlock) s += q.parts[i];
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    float v[16];
#pragma unroll
    for (int u = 0; u < 16; u++) {
        const int r = t.i * 64 + (int)(threadIdx.x >> 6) + 4 * u, c = t.j * 64 + (int)(threadIdx.x & 63);
        const size_t at = (size_t)r * q.cols + c;
        v[u] = r < q.rows && c < q.cols ? step_value(q.g[at], q.m[at], st) : 0.0f;
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
    char *const along = q.tall ? q.xt[0] : q.x[0], *const across = q.tall ? q.x[0] : q.xt[0];
    const int along_p = q.tall ? q.sp : q.lp, across_p = q.tall ? q.lp : q.sp;   // values per row
#pragma unroll
    for (int u = 0; u < 2; u++) {
        const int r = (int)(threadIdx.x >> 3) + 32 * u, c = (int)(threadIdx.x & 7) * 8;
        float p[8], o[8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            p[e] = tile[r][c + e];
            o[e] = tile[c + e][r];
        }
        uint2 h0, l0, h1, l1;
        split4(p, h0, l0);
        split4(p + 4, h1, l1);
        char *at = along + ((size_t)(t.i * 64 + r) * along_p + t.j * 64 + c) * 4;
        *(v4u *)at = v4u{h0.x, h0.y, h1.x, h1.y};
        *(v4u *)(at + 16) = v4u{l0.x, l0.y, l1.x, l1.y};
        split4(o, h0, l0);
        split4(o + 4, h1, l1);
        at = across + ((size_t)(t.j * 64 + r) * across_p + t.i * 64 + c) * 4;
        *(v4u *)at = v4u{h0.x, h0.y, h1.x, h1.y};
        *(v4u *)(at + 16) = v4u{l0.x, l0.y, l1.x, l1.y};
    }
}

enum Product { kGram, kSquare, kApply, kLast };

// Rows of both operands of a tile go from memory to LDS as they lie, sixteen bytes a lane, with no register in between; piece p
// of a row's 128 or 256 bytes lies at place p ^ (row mod pieces), so that lanes which read the same piece of neighbouring rows
// touch different banks (the lanes fetch accordingly: inside a row's line the order is theirs to choose).
constexpr int kStage = 32768;

// 8 KB of rows from `src`, kLine bytes of each: a wavefront's share of a stage.
template <int kLine>
__device__ __forceinline__ void stage(const char *src, size_t pitch, int lane, char *lds)
{
    constexpr int kPieces = kLine / 16, kRows = 64 / kPieces;   // rows per instruction
    const int row = lane / kPieces, place = lane % kPieces;
#pragma unroll
    for (int q = 0; q < 8; q++) {
        const int piece = place ^ ((q * kRows + row) % kPieces);
        __builtin_amdgcn_global_load_lds((glb_ptr)(src + (size_t)(q * kRows + row) * pitch + piece * 16), (lds_ptr)(lds + q * 1024), 16, 0, 0);
    }
}

template <int kLine>
__device__ __forceinline__ v8h fragment(const char *lds, int row, int piece)
{
    return *(const v8h *)(lds + row * kLine + ((piece ^ (row % (kLine / 16))) * 16));
}

// acc[i][j] += rows 32 i of A times rows 32 j of B over sixteen steps, whose first piece is `piece`.
template <int kLine>
__device__ __forceinline__ void multiply(const char *A, const char *B, int arow, int brow, int piece, v16f (&acc)[2][2])
{
    v8h ah[2], al[2], bh[2], bl[2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
        ah[i] = fragment<kLine>(A, arow + 32 * i, piece);
        al[i] = fragment<kLine>(A, arow + 32 * i, piece + 1);
        bh[i] = fragment<kLine>(B, brow + 32 * i, piece);
        bl[i] = fragment<kLine>(B, brow + 32 * i, piece + 1);
    }
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
        for (int j = 0; j < 2; j++) {
            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(al[i], bh[j], acc[i][j], 0, 0, 0);
            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah[i], bl[j], acc[i][j], 0, 0, 0);
            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah[i], bh[j], acc[i][j], 0, 0, 0);
        }
}

// Between reads and writes of the same LDS by different wavefronts.  The empty statement keeps the reads in front of the barrier: without
// it the compiler moved those of `red` below, which ended in a branch behind the barrier, into that branch.
__device__ __forceinline__ void meet()
{
    asm volatile("" ::: "memory");
    __syncthreads();
}

// Stage k of `steps` is in LDS, for everyone, and the stage before it has been read by everyone.  Each wavefront waits for its own
// loads (eight a stage, of which the stages behind k may be under way) and meets the others; lgkmcnt: its fragments have left
// the stage that is filled next.
template <int kStages>
__device__ __forceinline__ void arrive(int k, int steps)
{
    const int behind = min(steps - 1 - k, kStages - 2);
    if (behind >= 2) asm volatile("s_waitcnt vmcnt(16) lgkmcnt(0)" ::: "memory");
    else if (behind == 1) asm volatile("s_waitcnt vmcnt(8) lgkmcnt(0)" ::: "memory");
    else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// f(stage in LDS) for each of `steps` stages, kStages - 1 of which are on their way ahead.
template <int kLine, int kStages, class F>
__device__ __forceinline__ void pipeline(const char *src, size_t pitch, int lane, int w, char *lds, int steps, F &&f)
{
    static_assert(kStages >= 2 && kStages <= 4, "arrive() counts up to two stages ahead");
    char *const mine = lds + w * (kStage / 4);
#pragma unroll
    for (int k = 0; k < kStages - 1; k++)
        if (k < steps) stage<kLine>(src + (size_t)k * kLine, pitch, lane, mine + k * kStage);
    int at = 0, fill = kStages - 1;
    for (int k = 0; k < steps; k++) {
        arrive<kStages>(k, steps);
        if (k + kStages - 1 < steps) stage<kLine>(src + (size_t)(k + kStages - 1) * kLine, pitch, lane, mine + fill * kStage);
        f(lds + at * kStage);
        fill = at;
        at = at + 1 == kStages ? 0 : at + 1;
    }
    meet();   // the last stage has been read
}

// Four values in each of four neighbouring lanes: lane b gets value b of each.  `v` holds the values in pairs.
__device__ __forceinline__ uint2 transpose4(uint2 v, int lane)
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
    return make_uint2(p[0] | p[1] << 16, p[2] | p[3] << 16);
}

// A 32 x 32 tile of parts, 128 bytes a row, that a wavefront puts together in LDS and stores in whole lines (eight bytes a lane
// straight to memory took four times the requests).  The sixteen-byte pieces of a row lie at place piece ^ (row mod 8).
__device__ __forceinline__ void put_part(char *image, int row, int piece, int half, uint2 v)
{
    *(uint2 *)(image + row * 128 + ((piece ^ (row & 7)) * 16) + 8 * half) = v;
}
__device__ __forceinline__ void store_image(const char *image, char *to, size_t pitch, int lane)
{
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const int row = 8 * k + (lane >> 3), place = lane & 7;
        *(v4u *)(to + row * pitch + ((place ^ (row & 7)) * 16)) = *(const v4u *)(image + row * 128 + place * 16);
    }
}

// The values of c that a lane adds to a square product at the end: asked for before the product.
struct Old {
    uint2 h[4], l[4];
};
__device__ __forceinline__ void load_old(Old &o, const Matrix &q, int c, int row0, int col0, int lane)
{
    const char *const at = q.sq[c] + (size_t)(col0 + (lane & 31)) * q.sp * 4 + (size_t)row0 * 4 + 8 * (lane >> 5);
#pragma unroll
    for (int g = 0; g < 4; g++) {
        o.h[g] = *(const uint2 *)(at + 32 * g);
        o.l[g] = *(const uint2 *)(at + 32 * g + 16);
    }
}

// The end of a 32 x 32 tile of a product at (row0, col0): a lane holds column `col` and rows r .. r + 3 of each of four groups.
// Values are stored row by row along the columns of the transpose ("across": four neighbouring values of the lane) and, exchanged
// between four lanes, along the rows.  `images`: 8 KB of LDS of the wavefront's own.
template <int kProduct>
__device__ __forceinline__ void finish(const Matrix &q, const Step &st, const SquareOp &op, int turn, const v16f &acc, const Old &old, int row0,
                                       int col0, int lane, char *images)
{
    constexpr bool kSq = kProduct == kGram || kProduct == kSquare;
    if (kSq && row0 < col0) return;   // the other half of a tile on the diagonal stores this one
    const int c = lane & 31, col = col0 + c, half = lane >> 5;
    if (kProduct == kLast) {
        const float by = st.by * q.wide * op.alpha;
        if (col >= q.l) return;
#pragma unroll
        for (int g = 0; g < 4; g++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int r = row0 + 8 * g + 4 * half + e;
                if (r < q.s) {
                    float *const w = q.w + (q.tall ? (size_t)col * q.s + r : (size_t)r * q.l + col);
                    *w = st.keep * *w - by * acc[4 * g + e];
                }
            }
        return;
    }
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
        uint2 h, l;
        split4(v, h, l);
        put_part(images, c, 2 * g, half, h);
        put_part(images, c, 2 * g + 1, half, l);
        put_part(images + 4096, r + (lane & 3), 2 * (c >> 3), (c >> 2) & 1, transpose4(h, lane));
        put_part(images + 4096, r + (lane & 3), 2 * (c >> 3) + 1, (c >> 2) & 1, transpose4(l, lane));
    }
    char *const along = kSq ? q.sq[op.d] : q.x[turn ^ 1], *const across = kSq ? q.sq[op.d] : q.xt[turn ^ 1];
    const size_t along_p = (size_t)(kSq ? q.sp : q.lp) * 4, across_p = (size_t)q.sp * 4;   // bytes per row
    store_image(images, across + (size_t)col0 * across_p + (size_t)row0 * 4, across_p, lane);
    if (!kSq || row0 != col0) store_image(images + 4096, along + (size_t)row0 * along_p + (size_t)col0 * 4, along_p, lane);
}

// The sums of a 32 x 32 tile as four quads per lane.
__device__ __forceinline__ float4 quad_of(const v16f &a, int g) { return make_float4(a[4 * g], a[4 * g + 1], a[4 * g + 2], a[4 * g + 3]); }
__device__ __forceinline__ void set_quad(v16f &a, int g, float4 v)
{
    a[4 * g] = v.x;
    a[4 * g + 1] = v.y;
    a[4 * g + 2] = v.z;
    a[4 * g + 3] = v.w;
}

// Big tiles: 128 x 128, four wavefronts of 64 x 64 each, 32 steps a stage.  Small ones: 64 x 64, each of four wavefronts multiplies
// the whole tile over its quarter of a stage's 64 steps, which takes half of what four tiles of 32 x 32 would read from LDS; their
// sums meet in LDS, in the wavefronts' order.
template <int kProduct, int kStages>
__global__ __launch_bounds__(kBlock, kStages > 2 ? 1 : 2) void muon_product_k(const Matrix *jobs, const Tile *tiles, Step st, SquareOps ops, int turn)
{
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const Tile t = tiles[blockIdx.x];
    if (t.job < 0) return;
    const SquareOp op = ops.op[blockIdx.y];
    const Matrix &q = jobs[t.job];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), l32 = lane & 31, kh = lane >> 5;
    const char *const left = kProduct == kGram ? q.x[turn] : q.sq[op.l];
    const char *const right = kProduct == kGram ? q.x[turn] : kProduct == kSquare ? q.sq[op.r] : q.xt[turn];
    const size_t pitch = (size_t)(kProduct == kGram ? q.lp : q.sp) * 4;   // of both
    const int side = t.big ? 128 : 64;
    // the first two wavefronts bring the left operand's rows, the others the right one's
    const char *const src = (w < 2 ? left + (size_t)(t.i * side + w * (side / 2)) * pitch : right + (size_t)(t.j * side + (w - 2) * (side / 2)) * pitch) +
                            (size_t)t.from * 256;
    char *const images = lds + w * 8192;
    v16f acc[2][2];
    zero_acc(acc);
    if (t.big) {
        const int r0 = t.i * 128 + (w >> 1) * 64, c0 = t.j * 128 + (w & 1) * 64;
        pipeline<128, kStages>(src, pitch, lane, w, lds, 2 * (t.to - t.from), [&](const char *now) {
#pragma unroll
            for (int s = 0; s < 2; s++) multiply<128>(now, now + kStage / 2, (w >> 1) * 64 + l32, (w & 1) * 64 + l32, 4 * s + 2 * kh, acc);
        });
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int j = 0; j < 2; j++) {
                Old old;
                if (kProduct == kSquare) load_old(old, q, op.c, r0 + 32 * i, c0 + 32 * j, lane);
                finish<kProduct>(q, st, op, turn, acc[i][j], old, r0 + 32 * i, c0 + 32 * j, lane, images);
            }
        return;
    }
    const int row0 = t.i * 64 + (w >> 1) * 32, col0 = t.j * 64 + (w & 1) * 32;
    Old old;
    if (kProduct == kSquare) load_old(old, q, op.c, row0, col0, lane);
    pipeline<256, kStages>(src, pitch, lane, w, lds, t.to - t.from,
                           [&](const char *now) { multiply<256>(now, now + kStage / 2, l32, l32, 4 * w + 2 * kh, acc); });
    float4 *const red = (float4 *)lds;   // [wavefront][tile][quad of values][lane]
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
            for (int g = 0; g < 4; g++) red[((w * 4 + i * 2 + j) * 4 + g) * 64 + lane] = quad_of(acc[i][j], g);
    meet();
    v16f sum;
#pragma unroll
    for (int g = 0; g < 4; g++) {
        float4 v = red[(w * 4 + g) * 64 + lane];
#pragma unroll
        for (int o = 1; o < 4; o++) {
            const float4 p = red[((o * 4 + w) * 4 + g) * 64 + lane];
            v = make_float4(v.x + p.x, v.y + p.y, v.z + p.z, v.w + p.w);
        }
        set_quad(sum, g, v);
    }
    if (kProduct == kGram && t.slot >= 0) {
#pragma unroll
        for (int g = 0; g < 4; g++) q.partial[(((size_t)t.slot * 4 + w) * 4 + g) * 64 + lane] = quad_of(sum, g);
        return;
    }
    meet();   // the sums have been read
    finish<kProduct>(q, st, op, turn, sum, old, row0, col0, lane, images);
}

// Adds the parts of a tile of A, in their order.
__global__ __launch_bounds__(kBlock) void muon_meet_k(const Matrix *jobs, const Tile *tiles, Step st, SquareOps ops)
{
    __shared__ __attribute__((aligned(16))) char images[4 * 8192];
    const Tile t = tiles[blockIdx.x];
    const Matrix &q = jobs[t.job];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    v16f sum;
#pragma unroll
    for (int g = 0; g < 4; g++) {
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int p = 0; p < t.parts; p++) {
            const float4 o = q.partial[(((size_t)(t.slot + p) * 4 + w) * 4 + g) * 64 + lane];
            v = make_float4(v.x + o.x, v.y + o.y, v.z + o.z, v.w + o.w);
        }
        set_quad(sum, g, v);
    }
    finish<kGram>(q, st, ops.op[0], 0, sum, Old{}, t.i * 64 + (w >> 1) * 32, t.j * 64 + (w & 1) * 32, lane, images + w * 8192);
}

// No iterations: w moves along X itself.
__global__ __launch_bounds__(kBlock) void muon_plain_k(const Matrix *jobs, const Tile *chunks, Step st)
{
    const Tile t = chunks[blockIdx.x];
    const Matrix &q = jobs[t.job];
    const size_t n = (size_t)q.rows * q.cols, from = (size_t)t.i * kChunk, to = min(from + kChunk, n);
    const float by = st.by * q.wide * (1.0f / kUp);
    for (size_t i = from + threadIdx.x; i < to; i += kBlock) {
        const size_t r = i / q.cols, c = i % q.cols;
        const char *const at = (q.tall ? q.xt[0] : q.x[0]) + (r * (q.tall ? q.sp : q.lp) + c / 8 * 8) * 4 + c % 8 * 2;
        const float x = (float)*(const _Float16 *)at + (float)*(const _Float16 *)(at + 16);
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
    for (size_t k = 0; k < most; k++)
        for (auto &x : xcd) out.push_back(k < x.size() ? tiles[x[k]] : Tile{-1, 0, 0, 0, 0, 0, -1, 0});
    return out;
}

int put(const void *host, size_t bytes, void *to) { return bytes ? dopt_hip_copy_h2d(to, host, bytes) : DOPT_HIP_OK; }

void release(Handle *h)
{
    dopt_hip_free(h->memory);
    delete h;
}

int build(Handle *h)
{
    std::vector<Tile> chunks, scales, grams, meets, squares, wides;
    std::vector<double> cgram, csq, cwide;
    size_t bytes = 0;
    auto take = [&](size_t n) { const size_t at = bytes; bytes += ceil_div(n, (size_t)256) * 256; return at; };
    std::vector<size_t> at;
    constexpr int kBuffers = 4 + kSquares + 2;
    size_t all = 0;   // 64-step stages of all tiles of A
    for (Matrix &q : h->jobs) {
        q.tall = q.rows > q.cols;
        q.s = std::min(q.rows, q.cols);
        q.l = std::max(q.rows, q.cols);
        const int side = q.s <= 64 ? 64 : 128;
        q.sp = (int)ceil_div((size_t)q.s, (size_t)side) * side;
        q.lp = (int)ceil_div((size_t)q.l, (size_t)side) * side;
        q.wide = std::sqrt(std::max(1.0f, (float)q.rows / (float)q.cols));
        q.nparts = (int)ceil_div((size_t)q.rows * q.cols, kChunk);
        const size_t t = q.sp / 64;
        all += t * (t + 1) / 2 * (q.lp / 64);
    }
    // A's reduction is cut where its tiles alone would not give every CU its share
    const size_t part = std::max((size_t)16, ceil_div(all * 2, (size_t)num_cus() * 3));
    for (size_t k = 0; k < h->jobs.size(); k++) {
        Matrix &q = h->jobs[k];
        const int job = (int)k, side = q.s <= 64 ? 64 : 128, big = side == 128, deep = q.lp / 64;
        const int rp = q.tall ? q.lp : q.sp, cp = q.tall ? q.sp : q.lp, cuts = (int)ceil_div((size_t)deep, part);
        for (int i = 0; i < q.nparts; i++) chunks.push_back(Tile{job, i, 0, 0, 0, 0, -1, 0});
        for (int i = 0; i < rp / 64; i++)
            for (int j = 0; j < cp / 64; j++) scales.push_back(Tile{job, i, j, 0, 0, 0, -1, 0});
        int slots = 0;
        for (int i = 0; i < q.sp / 64; i++)
            for (int j = 0; j <= i; j++) {
                squares.push_back(Tile{job, i, j, 0, 0, q.sp / 64, -1, 0});
                csq.push_back((double)q.sp + 512);
                if (cuts > 1) meets.push_back(Tile{job, i, j, 0, 0, 0, slots, cuts});
                for (int c = 0; c < cuts; c++) {
                    const int from = deep * c / cuts, to = deep * (c + 1) / cuts;
                    grams.push_back(Tile{job, i, j, 0, from, to, cuts > 1 ? slots++ : -1, 0});
                    cgram.push_back((double)(to - from) + 8);
                }
            }
        for (int j = 0; j < q.lp / side; j++)
            for (int i = 0; i < q.sp / side; i++) {
                wides.push_back(Tile{job, i, j, big, 0, q.sp / 64, -1, 0});
                cwide.push_back((double)q.sp + 256);
            }
        const size_t x = (size_t)q.sp * q.lp * 4, a = (size_t)q.sp * q.sp * 4;
        for (int i = 0; i < 4; i++) at.push_back(take(x));
        for (int i = 0; i < kSquares; i++) at.push_back(take(a));
        at.push_back(take((size_t)slots * 64 * 64 * sizeof(float)));
        at.push_back(take((size_t)q.nparts * sizeof(double)));
    }
    grams = deal(grams, cgram);
    squares = deal(squares, csq);
    wides = deal(wides, cwide);
    struct Table {
        std::vector<Tile> *tiles;
        Tile **device;
        unsigned *n;
    } tables[] = {{&chunks, &h->chunks, &h->nchunks}, {&scales, &h->scales, &h->nscales},    {&grams, &h->grams, &h->ngrams},
                  {&meets, &h->meets, &h->nmeets},    {&squares, &h->squares, &h->nsquares}, {&wides, &h->wides, &h->nwides}};
    std::vector<size_t> table_at;
    for (Table &t : tables) table_at.push_back(take(t.tiles->size() * sizeof(Tile)));
    const size_t jobs_at = take(h->jobs.size() * sizeof(Matrix));
    if (int rc = scratch_alloc(&h->memory, bytes)) return rc;
    char *const base = (char *)h->memory;
    for (size_t k = 0; k < h->jobs.size(); k++) {
        Matrix &q = h->jobs[k];
        const size_t *const p = &at[kBuffers * k];
        for (int i = 0; i < 2; i++) {
            q.x[i] = base + p[i];
            q.xt[i] = base + p[2 + i];
        }
        for (int i = 0; i < kSquares; i++) q.sq[i] = base + p[4 + i];
        q.partial = (float4 *)(base + p[4 + kSquares]);
        q.parts = (double *)(base + p[5 + kSquares]);
    }
    for (size_t i = 0; i < table_at.size(); i++) {
        *tables[i].device = (Tile *)(base + table_at[i]);
        *tables[i].n = (unsigned)tables[i].tiles->size();
        if (int rc = put(tables[i].tiles->data(), tables[i].tiles->size() * sizeof(Tile), *tables[i].device)) return rc;
    }
    h->d_jobs = (Matrix *)(base + jobs_at);
    return put(h->jobs.data(), h->jobs.size() * sizeof(Matrix), h->d_jobs);
}

template <int kProduct, int kStages>
int launch_deep(const Handle *h, dim3 grid, const Tile *tiles, const Step &st, const SquareOps &ops, int turn)
{
    static bool raised = false;   // above 64 KB of dynamic LDS a kernel has to be told once
    if (!raised && kStages > 2)
        DOPT_HIP_CHECK(hipFuncSetAttribute((const void *)muon_product_k<kProduct, kStages>, hipFuncAttributeMaxDynamicSharedMemorySize,
                                           kStages * kStage));
    raised = true;
    hipLaunchKernelGGL((muon_product_k<kProduct, kStages>), grid, dim3(kBlock), kStages * kStage, stream(), h->d_jobs, tiles, st, ops, turn);
    DOPT_LAUNCH_CHECK();
    return DOPT_HIP_OK;
}

template <int kProduct>
int launch(const Handle *h, unsigned blocks, unsigned products, const Tile *tiles, const Step &st, const SquareOps &ops, int turn)
{
    const dim3 grid(blocks, products);
    return blocks * products <= (unsigned)num_cus() ? launch_deep<kProduct, 4>(h, grid, tiles, st, ops, turn)
                                                    : launch_deep<kProduct, 2>(h, grid, tiles, st, ops, turn);
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

// `count` iterations on X[turn]: into X[turn ^ 1], or into w.
int iterate(const Handle *h, const Step &st, int count, int turn, bool last)
{
    Buffers b;
    auto squares = [&](const SquareOps &ops, unsigned n) { return launch<kSquare>(h, h->nsquares, n, h->squares, st, ops, turn); };
    int a = b.take(kScaleBits), q = -1;
    SquareOps ops{};
    ops.op[0] = SquareOp{0, 0, a, 0, std::ldexp(1.0f, -kScaleBits), 0.0f, 0.0f};
    if (int rc = launch<kGram>(h, h->ngrams, 1, h->grams, st, ops, turn)) return rc;
    if (h->nmeets) {
        hipLaunchKernelGGL(muon_meet_k, dim3(h->nmeets), dim3(kBlock), 0, stream(), h->d_jobs, h->meets, st, ops);
        DOPT_LAUNCH_CHECK();
    }
    for (int k = 0; k < count; k++) {
        const int p = b.take(kScaleBits);
        ops.op[0] = b.op(kC, a, a, kB, a, kA, p);   // P
        if (int rc = squares(ops, 1)) return rc;
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
            if (int rc = squares(ops, n)) return rc;
            const int next = b.take(kScaleBits);
            ops.op[0] = b.op(1.0f, t, p, 0.0f, a, 0.0f, next);
            if (int rc = squares(ops, 1)) return rc;
            b.drop(a);
            b.drop(t);
            a = next;
        } else if (n) {
            if (int rc = squares(ops, n)) return rc;
        }
        if (before >= 0) {
            b.drop(before);
            b.drop(p);
        }
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
