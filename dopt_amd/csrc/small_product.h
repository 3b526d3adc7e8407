// Products of small outputs on the fp32 matrix instruction, straight from memory: sgemm.hip's, and those of groups of rows.
#pragma once

#include "dense.h"
#include "mfma_core.h"

namespace dopt {

// Small outputs (a dense layer at batch 128: 128 x 512 values from a 512-deep reduction).  The tile
// engine above would run four blocks plus a reduction launch; here one block owns a 32 x 32 tile of
// C, its eight wavefronts each take an eighth of K straight from memory into MFMA operands (no LDS
// staging: nothing is reused inside a 32-wide tile), and the eight partial tiles are summed through
// LDS in wavefront order.  Per step of 8 reductions a lane holds four k values for its row of A and
// four for its column of B; v_mfma_f32_32x32x2 number e pairs element e of lanes 0-31 (k = 8q + e)
// with element e of lanes 32-63 (k = 8q + 4 + e) - any pairing works as long as A and B agree.
//
// X is "k-contiguous" when element (r, k) sits at X[r * ld + k] (A as given, B transposed), else
// "r-contiguous" at X[k * ld + r].
//
// Loads go through buffer resources (an element outside the matrix or past the end of the wavefront's share of K
// comes from kOobOffset and reads as zero: no branch) and kSmallDepth steps are in flight per wavefront: with one
// step of prefetch every step waited a full memory latency, eight of them in a row for a 512-deep reduction -
// most of such a kernel's duration.  The order of the sums is that of the steps, whatever is in flight.
constexpr int kSmallWaves = 8, kSmallDepth = 4;

// The lane's four reductions kk .. kk + 3 of row / column r.  `base`: byte offset of (r, reduction 0), or kOobOffset
// when r lies outside the matrix; `pitch`: bytes between consecutive reductions of an r-contiguous operand.
// A k-contiguous operand is loaded as one 16-byte piece whatever its alignment (see Stage3): word by word, each load touched a
// line per row, and [29 x 2146] x [2146 x 2424], B stored [2424][2146], took 49 us instead of 20.
template <bool kKContig>
__device__ __forceinline__ void small_load(__amdgpu_buffer_rsrc_t rs, unsigned base, unsigned pitch, int kk, int k_end,
                                           float (&v)[4])
{
    if (kKContig) {
        const float4 q = buffer_load_f32x4(rs, kk < k_end ? base + (unsigned)kk * 4u : kOobOffset, 0);
        v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
    } else {
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = buffer_load_f32(rs, kk + e < k_end ? base + (unsigned)(kk + e) * pitch : kOobOffset, 0);
    }
}

// What the last pieces of a k-contiguous operand hold past the end of the reduction counts as zero.  kCut: a reduction of no
// multiple of four, whose last pieces do.
template <bool kKContig, bool kCut>
__device__ __forceinline__ float small_value(const float (&v)[4], int e, int kk, int k_end)
{
    return kKContig && kCut && e > 0 ? (kk + e < k_end ? v[e] : 0.0f) : v[e];
}

// kCut: a k-contiguous operand's rows are no whole quads.  kLong: a wavefront's share of the reduction may be longer than kSmallPart; each
// such part has an accumulator of its own then.
constexpr int kSmallPart = 1024;
template <bool kTA, bool kTB, bool kCut, class E = NoEpilogue, bool kLong = false>
__device__ __forceinline__ void sgemm_small_body(int M, int N, int K, int lda, int ldb, int kslice, const float *A,
                                                 const float *B, float *C, const float *colbias, int bias_shift,
                                                 const float *rowvec, int relu, const float *mask, int bx, int by, int k0, int k1,
                                                 float (*red)[32 * 33], const E &ep = E{})
{
    const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, r = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);   // the same in every lane: loop bounds stay scalar
    const int m0 = by * 32, n0 = bx * 32;
    const int row = m0 + r, col = n0 + r;
    const int k_begin = k0 + wave * kslice, k_end = min(k1, k_begin + kslice);   // the block's part of the reduction: [k0, k1)
    const __amdgpu_buffer_rsrc_t rsa = make_rsrc(A, (size_t)M * K * sizeof(float)), rsb = make_rsrc(B, (size_t)K * N * sizeof(float));
    // A is k-contiguous as given, B when it is read transposed
    const unsigned abase = row < M ? (kTA ? (unsigned)row * 4u : (unsigned)row * (unsigned)lda * 4u) : kOobOffset;
    const unsigned bbase = col < N ? (kTB ? (unsigned)col * (unsigned)ldb * 4u : (unsigned)col * 4u) : kOobOffset;
    const unsigned apitch = (unsigned)lda * 4u, bpitch = (unsigned)ldb * 4u;

    v16f acc;
#pragma unroll
    for (int v = 0; v < 16; v++) acc[v] = 0.0f;
    float a[kSmallDepth][4], b[kSmallDepth][4];
    const int nsteps = k_begin < k_end ? (k_end - k_begin + 7) / 8 : 0;
#pragma unroll
    for (int j = 0; j < kSmallDepth; j++) {   // steps past the end fetch nothing
        small_load<!kTA>(rsa, abase, apitch, k_begin + 8 * j + 4 * half, k_end, a[j]);
        small_load<kTB>(rsb, bbase, bpitch, k_begin + 8 * j + 4 * half, k_end, b[j]);
        __builtin_amdgcn_sched_barrier(0);   // in this order: the first step's operands are waited for first
    }
    auto value_a = [&](int j, int s, int e) { return small_value<!kTA, kCut>(a[j], e, k_begin + 8 * (s + j) + 4 * half, k_end); };
    auto value_b = [&](int j, int s, int e) { return small_value<kTB, kCut>(b[j], e, k_begin + 8 * (s + j) + 4 * half, k_end); };
    // Whole rounds of kSmallDepth steps without a branch inside (a branch per step made the compiler wait for every
    // load in flight at the top of the loop), then the steps left over, whose operands are in their registers or on
    // their way already.
    const int whole = nsteps / kSmallDepth * kSmallDepth;
    auto rounds = [&](int from, int to) {
        for (int s = from; s < to; s += kSmallDepth) {
#pragma unroll
            for (int j = 0; j < kSmallDepth; j++) {
#pragma unroll
                for (int e = 0; e < 4; e++) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(value_a(j, s, e), value_b(j, s, e), acc, 0, 0, 0);
                const int kk = k_begin + 8 * (s + j + kSmallDepth) + 4 * half;   // this register set's next step
                small_load<!kTA>(rsa, abase, apitch, kk, k_end, a[j]);
                small_load<kTB>(rsb, bbase, bpitch, kk, k_end, b[j]);
                __builtin_amdgcn_sched_barrier(0);   // keep each refill behind its own step: sunk to the loop's end, all of them are waited for at once
            }
        }
    };
    v16f parts = {};
    if constexpr (kLong) {
        constexpr int kPart = kSmallPart / 8;   // steps
        for (int s = 0; s < whole; s += kPart) {
            rounds(s, min(whole, s + kPart));
            parts += acc;
            acc = v16f{};
        }
    } else {
        rounds(0, whole);
    }
#pragma unroll
    for (int j = 0; j < kSmallDepth - 1; j++)
        if (whole + j < nsteps) {
#pragma unroll
            for (int e = 0; e < 4; e++) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(value_a(j, whole, e), value_b(j, whole, e), acc, 0, 0, 0);
        }
#pragma unroll
    for (int v = 0; v < 16; v++) red[wave][acc_row(v, lane) * 33 + r] = kLong ? parts[v] + acc[v] : acc[v];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const int idx = tid + i * 64 * kSmallWaves, rr = idx >> 5, cc = idx & 31;
        float sum = red[0][rr * 33 + cc];
#pragma unroll
        for (int w = 1; w < kSmallWaves; w++) sum += red[w][rr * 33 + cc];
        if (m0 + rr < M && n0 + cc < N) {
            if constexpr (E::kOn) sum = ep(sum, (size_t)(m0 + rr) * N + n0 + cc);
            if (colbias) {   // one value per group of 2^bias_shift columns, times the row's factor when there is one
                float add = colbias[(n0 + cc) >> bias_shift];
                if (rowvec) add = __fmul_rn(rowvec[m0 + rr], add);   // rounded on its own, as the separate product is
                sum += add;
            }
            if (relu) sum = sum < 0.0f ? 0.0f : sum;
            if (mask) sum = mask[(size_t)(m0 + rr) * N + n0 + cc] > 0.0f ? sum : 0.0f;   // reluGrad(product, ., mask)
            C[(size_t)(m0 + rr) * N + n0 + cc] = sum;
        }
    }
}

}  // namespace dopt
