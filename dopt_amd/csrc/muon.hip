// Updates that treat a weight as a matrix: the momentum's orthogonalised form takes the place of the momentum.
// No counterpart in the reference, whose rules are elementwise (online/source/dopt/online/{sgd,adam,amsgrad}.d).
//
//     m' = mu m + g,  u = g + mu m' (nesterov) or m',  X = u / (|u| + 1e-7) in the 2-norm of all values
//     `iterations` times, on the side of fewer rows:  A = X X^T,  X' = a X + (b A + c A A) X
//     w' = (1 - lr decay) w - lr sqrt(max(1, rows / cols)) X
//
// All matrices of a handle go through each step in the same launches: momentum and norm, scaling, and three products per
// iteration, so a network of twenty layers takes seventeen launches and not hundreds.
//
// The products run on the fp16 matrix instruction with every value as the sum of two fp16 numbers, h = fp16(v) and
// l = fp16(v - h), of the three products h h + h l + l h that matter, in fp32 sums.  Two parts hold 22 bits, and l l is 2^-24 of
// h h on average: together half a bit more than fp32 rounds away from each product, with random signs.  fp16's small range does
// no harm here, where no value is: |X| <= 1 by its scaling and the iteration keeps singular values below 1.21, so entries of X,
// A and B = b A + c A A stay under 1.21, 1.47 and 2.81 and are held times 2^13; what lies below 2^-14 of fp16 loses bits only
// against 2^-38 of the largest entry possible.  That is half the matrix work of three bf16 parts, which the products of
// sgemm.hip need for operands of any size, and a value takes the four bytes that it takes in fp32.
//
// Operands lie row by row along the reduction in pieces of eight values: their h parts (16 bytes), then their l parts.  A and B
// are symmetric, so all three products are of that form once X is kept both as it is and transposed: A = X . X, B = A . A,
// X' = B . X^T; of A and B the tiles on and below the diagonal are formed and stored twice.
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
constexpr float kUp = 0x1p13f, kDown = 0x1p-13f, kDownProduct = 0x1p-26f;

struct Matrix {
    float *w;
    const float *g;
    float *m;
    char *x[2], *xt[2], *a, *b;   // X and its transpose before and after an iteration, A, B
    double *parts;                // the momentum's pass: sums of squares
    int rows, cols;               // as w lies
    int s, l;                     // the shorter and the longer side: X is [s][l]
    int sp, lp;                   // ... in whole tiles
    int nparts, tall;             // tall: X is w transposed
    float wide;                   // sqrt(max(1, rows / cols))
};

struct Tile {
    int job, i, j, big;   // job < 0: nothing to do
};

struct Step {
    float mu, by, keep;
    int nesterov;
};

struct Handle {
    std::vector<Matrix> jobs;
    void *memory = nullptr;
    Matrix *d_jobs = nullptr;
    Tile *chunks = nullptr, *scales = nullptr, *squares = nullptr, *wides = nullptr;   // device
    unsigned nchunks = 0, nscales = 0, nsquares = 0, nwides = 0;
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

enum Product { kGram, kPoly, kApply, kLast };

// Rows of both operands of a tile go from memory to LDS as they lie, sixteen bytes a lane, with no register in between; piece p
// of a row's 128 or 256 bytes lies at place p ^ (row mod pieces), so that lanes which read the same piece of neighbouring rows
// touch different banks (the lanes fetch accordingly: inside a row's line the order is theirs to choose).  Two stages of 32 KB:
// one is multiplied while the next one arrives, and two workgroups share a CU.
constexpr int kStage = 32768;

// `rows` rows from `src` (bytes), of the reduction's bytes [k, k + kLine); a wavefront brings 8 KB.
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

// Waits for this wavefront's loads into LDS and meets the others.
__device__ __forceinline__ void arrive()
{
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");   // (lgkmcnt: its fragments have left the stage that is filled next)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
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

// The end of a 32 x 32 tile of a product at (row0, col0): a lane holds column `col` and rows r .. r + 3 of each of four groups.
// Values are stored row by row along the columns of the transpose ("across": four neighbouring values of the lane) and, exchanged
// between four lanes, along the rows.
template <int kProduct>
__device__ __forceinline__ void finish(const Matrix &q, const Step &st, int turn, const v16f &acc, int row0, int col0, int lane)
{
    if (kProduct < kApply && row0 < col0) return;   // the other half of a tile on the diagonal stores this one
    const int col = col0 + (lane & 31), half = lane >> 5;
    const size_t along_p = (size_t)(kProduct < kApply ? q.sp : q.lp) * 4, across_p = (size_t)q.sp * 4;   // bytes per row
    char *const along = kProduct == kGram ? q.a : kProduct == kPoly ? q.b : q.x[turn ^ 1];
    char *const across = kProduct == kGram ? q.a : kProduct == kPoly ? q.b : q.xt[turn ^ 1];
    const char *const old = kProduct == kPoly ? q.a : q.xt[turn];
#pragma unroll
    for (int g = 0; g < 4; g++) {
        const int r = row0 + 8 * g + 4 * half;
        const size_t at = (size_t)col * across_p + (size_t)(row0 + 8 * g) * 4 + 8 * half;
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = acc[4 * g + e] * (kProduct == kPoly ? kC * kDown : kDown);   // times kUp once
        if (kProduct != kGram) {
            float o[4];
            join4(*(const uint2 *)(old + at), *(const uint2 *)(old + at + 16), o);
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] += (kProduct == kPoly ? kB : kA) * o[e];
        }
        if (kProduct == kLast) {
            const float by = st.by * q.wide * kDown;
            if (q.tall) {
                if (col < q.l) {
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        if (r + e < q.s) {
                            float *const w = q.w + (size_t)col * q.s + r + e;
                            *w = st.keep * *w - by * v[e];
                        }
                }
            } else if (col < q.l) {
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (r + e < q.s) {
                        float *const w = q.w + (size_t)(r + e) * q.l + col;
                        *w = st.keep * *w - by * v[e];
                    }
            }
            continue;
        }
        uint2 h, l;
        split4(v, h, l);
        *(uint2 *)(across + at) = h;
        *(uint2 *)(across + at + 16) = l;
        if (kProduct < kApply && row0 == col0) continue;   // a tile on the diagonal is its own transpose
        const size_t to = (size_t)(r + (lane & 3)) * along_p + (size_t)(col >> 3) * 32 + ((col >> 2) & 1) * 8;
        *(uint2 *)(along + to) = transpose4(h, lane);
        *(uint2 *)(along + to + 16) = transpose4(l, lane);
    }
}

// Big tiles: 128 x 128, four wavefronts of 64 x 64 each, 32 steps a stage.  Small ones: 64 x 64, each of four wavefronts multiplies
// the whole tile over its quarter of a stage's 64 steps, which takes half of what four tiles of 32 x 32 would read from LDS; their
// sums meet in LDS, in the wavefronts' order.
template <int kProduct>
__global__ __launch_bounds__(kBlock, 2) void muon_product_k(const Matrix *jobs, const Tile *tiles, Step st, int turn)
{
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const Tile t = tiles[blockIdx.x];
    if (t.job < 0) return;
    const Matrix &q = jobs[t.job];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), l32 = lane & 31, kh = lane >> 5;
    const char *const left = kProduct == kGram ? q.x[turn] : kProduct == kPoly ? q.a : q.b;
    const char *const right = kProduct == kGram ? q.x[turn] : kProduct == kPoly ? q.a : q.xt[turn];
    const size_t pitch = (size_t)(kProduct == kGram ? q.lp : q.sp) * 4;   // of both
    const int side = t.big ? 128 : 64;
    // the first two wavefronts bring the left operand's rows, the others the right one's
    const char *src = (w < 2 ? left + (size_t)(t.i * side + w * (side / 2)) * pitch : right + (size_t)(t.j * side + (w - 2) * (side / 2)) * pitch);
    char *const mine = lds + w * (kStage / 4);
    v16f acc[2][2];
    zero_acc(acc);
    if (t.big) {
        const int steps = (int)(pitch / 128);
        stage<128>(src, pitch, lane, mine);
        for (int k = 0; k < steps; k++) {
            arrive();
            if (k + 1 < steps) stage<128>(src + (size_t)(k + 1) * 128, pitch, lane, mine + ((k + 1) & 1) * kStage);
            const char *const now = lds + (k & 1) * kStage;
#pragma unroll
            for (int s = 0; s < 2; s++)
                multiply<128>(now, now + kStage / 2, (w >> 1) * 64 + l32, (w & 1) * 64 + l32, 4 * s + 2 * kh, acc);
        }
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int j = 0; j < 2; j++)
                finish<kProduct>(q, st, turn, acc[i][j], t.i * 128 + (w >> 1) * 64 + 32 * i, t.j * 128 + (w & 1) * 64 + 32 * j, lane);
    } else {
        const int steps = (int)(pitch / 256);
        stage<256>(src, pitch, lane, mine);
        for (int k = 0; k < steps; k++) {
            arrive();
            if (k + 1 < steps) stage<256>(src + (size_t)(k + 1) * 256, pitch, lane, mine + ((k + 1) & 1) * kStage);
            const char *const now = lds + (k & 1) * kStage;
            multiply<256>(now, now + kStage / 2, l32, l32, 4 * w + 2 * kh, acc);
        }
        __syncthreads();   // the last stage has been read
        float4 *const red = (float4 *)lds;   // [wavefront][tile][quad of values][lane]
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
                for (int g = 0; g < 4; g++)
                    red[((w * 4 + i * 2 + j) * 4 + g) * 64 + lane] =
                        make_float4(acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]);
        __syncthreads();
        v16f sum;
#pragma unroll
        for (int g = 0; g < 4; g++) {
            float4 v = red[(w * 4 + g) * 64 + lane];
#pragma unroll
            for (int o = 1; o < 4; o++) {
                const float4 p = red[((o * 4 + w) * 4 + g) * 64 + lane];
                v = make_float4(v.x + p.x, v.y + p.y, v.z + p.z, v.w + p.w);
            }
            sum[4 * g] = v.x;
            sum[4 * g + 1] = v.y;
            sum[4 * g + 2] = v.z;
            sum[4 * g + 3] = v.w;
        }
        finish<kProduct>(q, st, turn, sum, t.i * 64 + (w >> 1) * 32, t.j * 64 + (w & 1) * 32, lane);
    }
}

// No iterations: w moves along X itself.
__global__ __launch_bounds__(kBlock) void muon_plain_k(const Matrix *jobs, const Tile *chunks, Step st)
{
    const Tile t = chunks[blockIdx.x];
    const Matrix &q = jobs[t.job];
    const size_t n = (size_t)q.rows * q.cols, from = (size_t)t.i * kChunk, to = min(from + kChunk, n);
    const float by = st.by * q.wide * kDown;
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
        for (auto &x : xcd) out.push_back(k < x.size() ? tiles[x[k]] : Tile{-1, 0, 0, 0});
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
    std::vector<Tile> chunks, scales, squares, wides;
    std::vector<double> csq, cwide;
    size_t bytes = 0;
    auto take = [&](size_t n) { const size_t at = bytes; bytes += ceil_div(n, (size_t)256) * 256; return at; };
    std::vector<size_t> at;
    for (size_t k = 0; k < h->jobs.size(); k++) {
        Matrix &q = h->jobs[k];
        q.tall = q.rows > q.cols;
        q.s = std::min(q.rows, q.cols);
        q.l = std::max(q.rows, q.cols);
        const int side = q.s <= 64 ? 64 : 128;
        q.sp = (int)ceil_div((size_t)q.s, (size_t)side) * side;
        q.lp = (int)ceil_div((size_t)q.l, (size_t)side) * side;
        q.wide = std::sqrt(std::max(1.0f, (float)q.rows / (float)q.cols));
        q.nparts = (int)ceil_div((size_t)q.rows * q.cols, kChunk);
        const size_t x = (size_t)q.sp * q.lp * 4, a = (size_t)q.sp * q.sp * 4;
        for (size_t n : {x, x, x, x, a, a, (size_t)q.nparts * sizeof(double)}) at.push_back(take(n));
        const int job = (int)k;
        for (int i = 0; i < q.nparts; i++) chunks.push_back(Tile{job, i, 0, 0});
        const int rp = q.tall ? q.lp : q.sp, cp = q.tall ? q.sp : q.lp;
        for (int i = 0; i < rp / 64; i++)
            for (int j = 0; j < cp / 64; j++) scales.push_back(Tile{job, i, j, 0});
        for (int i = 0; i < q.sp / 64; i++)
            for (int j = 0; j <= i; j++) {
                squares.push_back(Tile{job, i, j, 0});
                csq.push_back((double)q.lp + 512);
            }
        const int big = side == 128;
        for (int j = 0; j < q.lp / side; j++)
            for (int i = 0; i < q.sp / side; i++) {
                wides.push_back(Tile{job, i, j, big});
                cwide.push_back((double)q.sp + 256);
            }
    }
    squares = deal(squares, csq);
    wides = deal(wides, cwide);
    h->nchunks = (unsigned)chunks.size();
    h->nscales = (unsigned)scales.size();
    h->nsquares = (unsigned)squares.size();
    h->nwides = (unsigned)wides.size();
    const size_t jobs_at = take(h->jobs.size() * sizeof(Matrix)), chunks_at = take(chunks.size() * sizeof(Tile)),
                 scales_at = take(scales.size() * sizeof(Tile)), squares_at = take(squares.size() * sizeof(Tile)),
                 wides_at = take(wides.size() * sizeof(Tile));
    if (int rc = scratch_alloc(&h->memory, bytes)) return rc;
    char *const base = (char *)h->memory;
    for (size_t k = 0; k < h->jobs.size(); k++) {
        Matrix &q = h->jobs[k];
        const size_t *const p = &at[7 * k];
        q.x[0] = base + p[0];
        q.x[1] = base + p[1];
        q.xt[0] = base + p[2];
        q.xt[1] = base + p[3];
        q.a = base + p[4];
        q.b = base + p[5];
        q.parts = (double *)(base + p[6]);
    }
    h->d_jobs = (Matrix *)(base + jobs_at);
    h->chunks = (Tile *)(base + chunks_at);
    h->scales = (Tile *)(base + scales_at);
    h->squares = (Tile *)(base + squares_at);
    h->wides = (Tile *)(base + wides_at);
    int rc = put(h->jobs.data(), h->jobs.size() * sizeof(Matrix), h->d_jobs);
    if (!rc) rc = put(chunks.data(), chunks.size() * sizeof(Tile), h->chunks);
    if (!rc) rc = put(scales.data(), scales.size() * sizeof(Tile), h->scales);
    if (!rc) rc = put(squares.data(), squares.size() * sizeof(Tile), h->squares);
    if (!rc) rc = put(wides.data(), wides.size() * sizeof(Tile), h->wides);
    return rc;
}

template <int kProduct>
int launch(const Handle *h, unsigned blocks, const Tile *tiles, const Step &st, int turn)
{
    hipLaunchKernelGGL(muon_product_k<kProduct>, dim3(blocks), dim3(kBlock), 2 * kStage, stream(), h->d_jobs, tiles, st, turn);
    DOPT_LAUNCH_CHECK();
    return DOPT_HIP_OK;
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
    for (int it = 0; it < iterations; it++) {
        const int turn = it & 1;
        if (int rc = launch<kGram>(h, h->nsquares, h->squares, st, turn)) return rc;
        if (int rc = launch<kPoly>(h, h->nsquares, h->squares, st, turn)) return rc;
        if (int rc = it + 1 < iterations ? launch<kApply>(h, h->nwides, h->wides, st, turn) : launch<kLast>(h, h->nwides, h->wides, st, turn))
            return rc;
    }
    return DOPT_HIP_OK;
}

}  // extern "C"
