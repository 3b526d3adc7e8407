// Products of fp32 values as two fp16 parts each: h = fp16(v) and l = fp16(v - h), 22 bits in four bytes, and the three products h h + h l + l h
// on the fp16 matrix instruction, in fp32 sums.  The caller scales its values into fp16's range, and bounds how many steps are added in one accumulator: all three
// products go there, and the instruction rounds down what lies below its guard bits.
//
// Operands run along the reduction.  They lie in blocks of 32 rows by 16 steps, 2 KB one after the other along a row of blocks; a row of a
// block is 64 bytes, h and l parts of eight values (16 bytes each) and of the next eight.  Inside a row the four pieces lie at
// place piece ^ (row / 4 mod 4), in memory as in LDS, so that lanes which read the same piece of neighbouring rows touch
// different banks.
#pragma once

#include <hip/hip_runtime.h>

#include "mfma_core.h"

namespace dopt {

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v4h __attribute__((ext_vector_type(4)));
using lds_ptr = __attribute__((address_space(3))) void *;
using glb_ptr = __attribute__((address_space(1))) const void *;
// Addresses that come out of a table: the compiler does not see that they are global memory's, and a flat access waits for LDS too.
template <class T>
using Global = __attribute__((address_space(1))) T *;
template <class T>
__device__ __forceinline__ Global<T> global(T *p)
{
    return (Global<T>)p;
}
typedef float v4f __attribute__((ext_vector_type(4)));
typedef unsigned v2u __attribute__((ext_vector_type(2)));

// Four values as their h and l parts.
__device__ __forceinline__ void split4(const float *v, v2u &h, v2u &l)
{
    v4h a, b;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        a[e] = (_Float16)v[e];
        b[e] = (_Float16)(v[e] - (float)a[e]);
    }
    h = __builtin_bit_cast(v2u, a);
    l = __builtin_bit_cast(v2u, b);
}

__device__ __forceinline__ void join4(v2u h, v2u l, float *v)
{
    const v4h a = __builtin_bit_cast(v4h, h), b = __builtin_bit_cast(v4h, l);
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] = (float)a[e] + (float)b[e];
}

// Where a row's piece lies in its block, and where the block of (row, step) lies in a matrix of `steps` steps.
__device__ __forceinline__ int piece_at(int row, int piece) { return (row & 31) * 64 + ((piece ^ ((row >> 2) & 3)) * 16); }
__device__ __forceinline__ size_t block_at(int row, int step, int steps) { return ((size_t)(row >> 5) * (steps >> 4) + (step >> 4)) * 2048; }

// Both operands of a tile go from memory to LDS as they lie, sixteen bytes a lane, with no register in between.
__device__ __forceinline__ void bring(const char *src, int kilobytes, int lane, char *lds)
{
#pragma unroll
    for (int q = 0; q < kilobytes; q++)
        __builtin_amdgcn_global_load_lds((glb_ptr)(src + q * 1024 + lane * 16), (lds_ptr)(lds + q * 1024), 16, 0, 0);
}

__device__ __forceinline__ v8h fragment(const char *block, int row, int piece) { return *(const v8h *)(block + piece_at(row, piece)); }

// Blocks of a wavefront's side of a product, as its lanes hold them.
template <int N>
struct Side {
    v8h h[N], l[N];
    __device__ __forceinline__ void read(const char *blocks, int lane)
    {
        const int row = lane & 31, piece = 2 * (lane >> 5);
#pragma unroll
        for (int i = 0; i < N; i++) {
            h[i] = fragment(blocks + 2048 * i, row, piece);
            l[i] = fragment(blocks + 2048 * i, row, piece + 1);
        }
    }
};

__device__ __forceinline__ v16f product(v8h ah, v8h al, v8h bh, v8h bl, v16f acc)
{
    acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(al, bh, acc, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah, bl, acc, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(ah, bh, acc, 0, 0, 0);
}

// acc[i][j] += block i of a times block j of b.
template <int MI, int NI>
__device__ __forceinline__ void multiply(const Side<MI> &a, const Side<NI> &b, v16f (&acc)[MI][NI])
{
#pragma unroll
    for (int i = 0; i < MI; i++)
#pragma unroll
        for (int j = 0; j < NI; j++) acc[i][j] = product(a.h[i], a.l[i], b.h[j], b.l[j], acc[i][j]);
}
template <int MI, int NI>
__device__ __forceinline__ void multiply(const char *A, const char *B, int lane, v16f (&acc)[MI][NI])
{
    Side<MI> a;
    Side<NI> b;
    a.read(A, lane);
    b.read(B, lane);
    multiply(a, b, acc);
}

// Between reads and writes of the same LDS by different wavefronts.  The empty statement keeps the reads in front of the barrier: without
// it the compiler moved reads whose values were used in a branch behind the barrier into that branch.
__device__ __forceinline__ void meet()
{
    asm volatile("" ::: "memory");
    __syncthreads();
}

// The wavefront's fragments have left LDS, and all but the last `kLoads` loads that it has asked for are there.
template <int kLoads>
__device__ __forceinline__ void settled()
{
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(kLoads) : "memory");
}

// multiply(a, b) for each of `steps` stages, which bring(k, stage in LDS) asks for, kLoads loads of a wavefront each, and of which
// read(stage in LDS, a, b) takes the wavefront's blocks.  While a stage is multiplied the next one is read into other
// registers; kStages - 1 further ones are on their way.  Once a wavefront's own part of stage k + 1 is there it meets the others: then
// all of it is, and stage k has been read by everyone.
template <int kStages, int kStage, int kLoads, int MI, int NI, class B, class R, class M>
__device__ __forceinline__ void pipeline(char *lds, int steps, B &&bring_stage, R &&read, M &&multiply_blocks)
{
    static_assert(kStages >= 3 && kStages <= 5 && kStages * kStage <= 163840, "one to three stages may be under way behind the next one");
    auto arrived = [&](int behind) {   // all loads but those of the last `behind` stages asked for
        if (kStages > 4 && behind >= 3) settled<3 * kLoads>();
        else if (kStages > 3 && behind >= 2) settled<2 * kLoads>();
        else if (behind >= 1) settled<kLoads>();
        else settled<0>();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
#pragma unroll
    for (int k = 0; k < kStages - 1; k++)
        if (k < steps) bring_stage(k, lds + k * kStage);
    int at = 0, fill = kStages - 1;   // where the stage that was read last lies, and the next one asked for
    arrived(min(steps - 1, kStages - 2));
    Side<MI> a0, a1;
    Side<NI> b0, b1;
    read(lds, a0, b0);
    if (kStages - 1 < steps) bring_stage(kStages - 1, lds + fill * kStage);
    auto one = [&](int k, const Side<MI> &a, const Side<NI> &b, Side<MI> &next_a, Side<NI> &next_b) {
        if (k + 1 < steps) {
            arrived(min(steps - 2 - k, kStages - 2));
            fill = at;
            at = at + 1 == kStages ? 0 : at + 1;
            read(lds + at * kStage, next_a, next_b);
            if (k + kStages < steps) bring_stage(k + kStages, lds + fill * kStage);
        }
        multiply_blocks(a, b);
    };
    for (int k = 0; k < steps; k += 2) {
        one(k, a0, b0, a1, b1);
        if (k + 1 < steps) one(k + 1, a1, b1, a0, b0);
    }
    meet();   // the last stage has been read
}

}  // namespace dopt
