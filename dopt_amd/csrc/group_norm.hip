// Group norm with an activation behind it, forward and backward, for [N, C, inner] and channels-last [N, inner, C] tensors.
// No counterpart in the reference, whose only norm is over the batch (cuda/source/dopt/cuda/nnet/cudnn7.d:547-654); the packed
// results follow its batch norm's (core/source/dopt/core/ops/nnet.d:222-235).
//
//     z = (x - mean) rstd scale[c] + bias[c],  y = act(z);  mean, biased variance of a group: C / G channels x inner values
//     dz = dy act'(z),  dbias[c] = sum dz,  dscale[c] = sum dz xhat,
//     dx = rstd (dz scale[c] - s1 - xhat s2),  s1, s2 the group's means of dz scale and dz scale xhat
//
// All of it is bound by memory: 8 bytes a value forward, 12 backward.  A group of an [N, C, inner] tensor lies in one piece, and up to
// 32768 values of it (of the gradient 16384 of both tensors) stay in the registers of one workgroup, which so reads and writes everything
// once.  Longer groups are parted: a first launch leaves each part's statistics (or sums), a second one joins them and reads the part again.
// Channels-last groups lie in pieces of C / G values; those of 8 to 64 channels, a power of two, are held likewise (gradients where that is
// faster, see held_for), otherwise workgroups take runs of pixels with all their channels, in two launches.  Means are taken before variances everywhere - of a part in registers, then
// of the parts - so nothing cancels however far from zero the values lie; sums of any length are taken in pieces or keep what their roundings leave out.
// No atomics: every sum has one order.
//
// Measured: [128, 160, 32 x 32] in 32 groups 34 us (168 MB, 4.9 TB/s), its like of 320 channels of 16 x 16 backward 35 us (126 MB), of
// which the sums over samples take 5; channels last [37, 29 x 33, 200] in 25 groups 15.4 us (57 MB; in two launches by runs 25),
// [64, 32 x 32, 128] in 16 groups backward 33 us by runs (101 MB; two passes over x and dy, the second from the last cache);
// one sample of [64, 8 x 8] 5.5 us, a launch.
#include <algorithm>
#include <type_traits>

#include "activation.h"
#include "common.h"

namespace {

using namespace dopt;

constexpr int kBlock = 256;
constexpr int kPiece = 8192;   // values of a part
constexpr int kRuns = 64;      // runs of pixels of a channels-last sample, at most

typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v4f_any __attribute__((ext_vector_type(4), aligned(4)));   // sixteen bytes wherever they start

__device__ __forceinline__ v4f load4(const float *p) { return *(const v4f_any *)p; }
__device__ __forceinline__ void store4(float *p, v4f v) { *(v4f_any *)p = v; }

// Between reads and writes of the same LDS by different wavefronts; the empty statement keeps reads in front of it that are used behind
// it in a branch.
__device__ __forceinline__ void meet()
{
    asm volatile("" ::: "memory");
    __syncthreads();
}

// A launch counts its threads in 32 bits along each side of its grid: more workgroups than this go into rows of as many.
constexpr unsigned kGridRow = 1 << 20;
__device__ __forceinline__ size_t block_id() { return (size_t)blockIdx.y * kGridRow + blockIdx.x; }
dim3 grid_of(size_t blocks)
{
    return blocks <= kGridRow ? dim3((unsigned)blocks) : dim3(kGridRow, (unsigned)ceil_div(blocks, (size_t)kGridRow));
}

template <int kControl>
__device__ __forceinline__ float plus_moved(float v)
{
    return v + __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), kControl, 0xf, 0xf, true));
}

// The sum over groups of `lanes` (a power of two, the same in all lanes) lanes, in all of them: with the neighbour, the other pair, the
// other quad (each of whose lanes holds its sum by now: the mirrored lane's does), the other eight, sixteen and thirty-two.
__device__ __forceinline__ float lanes_sum(float v, int lanes)
{
    if (lanes >= 2) v = plus_moved<0xB1>(v);
    if (lanes >= 4) v = plus_moved<0x4E>(v);
    if (lanes >= 8) v = plus_moved<0x141>(v);
    if (lanes >= 16) v = plus_moved<0x140>(v);
    if (lanes >= 32) v += __shfl_xor(v, 16, 64);
    if (lanes >= 64) v += __shfl_xor(v, 32, 64);
    return v;
}

// The sum over a workgroup of whole wavefronts, in every thread; red: 16 values.
__device__ __forceinline__ float block_sum(float v, float *red)
{
    v = lanes_sum(v, 64);
    const int waves = blockDim.x >> 6;
    if (waves == 1) return v;
    meet();   // the last sum has been read
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    meet();
    float s = red[0];
    for (int i = 1; i < waves; i++) s += red[i];
    return s;
}

// A sum of any length with what its roundings have left out (Kahan): many equal values are rounded the same way again and again, 135168 of
// 0.1 to a mean that is 1e-3 off.
struct LongSum {
    float sum = 0.0f, over = 0.0f;
    __device__ __forceinline__ void add(float v)
    {
        const float more = v - over, next = sum + more;
        over = __builtin_fabsf(next) <= 3.402823466e38f ? (next - sum) - more : 0.0f;   // (infinity stays one)
        sum = next;
    }
};

// What a workgroup holds of a group: `channels` of them from the group's channel c0 on, `len` values of each from `i0` on, P lanes to a
// channel; a thread has channels row, row + rows, .. (kC of them) and quads lane, lane + P, .. (kQ) of each.
struct Part {
    size_t base;      // of the group's first value
    size_t inner;
    int c0, channels, len, P, rows;
    size_t i0;
    int row, lane;    // of the thread
};

struct Where {
    size_t at;    // offset of a quad's first value
    int c;        // its channel in the group
    int first;    // the quad's values from `first` on are its own (4: none)
};

// A channel's last quad begins where it ends with the channel; the values that it shares with the quad before are that one's.  What lies
// beyond the last quad or channel repeats it, so that nothing is guarded but the sums.
__device__ __forceinline__ Where where(const Part &p, int ci, int qi)
{
    const int c = p.row + ci * p.rows, q = p.lane + qi * p.P;
    const int start = min(4 * q, p.len - 4);
    Where w;
    w.c = p.c0 + min(c, p.channels - 1);
    w.at = p.base + (size_t)w.c * p.inner + p.i0 + start;
    w.first = c < p.channels && p.row < p.rows ? min(4 * q - start, 4) : 4;
    return w;
}

__device__ __forceinline__ float own_sum(v4f v, int first)
{
    return ((first <= 0 ? v.x : 0.0f) + (first <= 1 ? v.y : 0.0f)) + ((first <= 2 ? v.z : 0.0f) + (first <= 3 ? v.w : 0.0f));
}

struct Sizes {
    size_t C, inner;
    int Cg, G;
    int pieces;            // of a channel
    int per;               // channels of a part
    int parts;             // of a group
    int P, rows;
    size_t blocks;         // of a launch
};

__device__ __forceinline__ Part part_of(const Sizes &s, size_t n, int g, int k)
{
    Part p;
    p.inner = s.inner;
    p.base = (n * s.C + (size_t)g * s.Cg) * s.inner;
    p.c0 = k / s.pieces * s.per;
    p.channels = min(s.per, s.Cg - p.c0);
    const size_t piece = k % s.pieces;
    p.i0 = s.inner * piece / s.pieces;
    p.len = (int)(s.inner * (piece + 1) / s.pieces - p.i0);
    p.P = s.P;
    p.rows = s.rows;
    p.row = (int)threadIdx.x / s.P;
    p.lane = (int)threadIdx.x - p.row * s.P;
    return p;
}

template <int kC, int kQ>
__device__ __forceinline__ void load_part(const Part &p, const float *x, v4f (&v)[kC][kQ])
{
#pragma unroll
    for (int ci = 0; ci < kC; ci++)
#pragma unroll
        for (int qi = 0; qi < kQ; qi++) v[ci][qi] = load4(x + where(p, ci, qi).at);
}

// Mean and sum of squared differences from it of what the workgroup holds.
template <int kC, int kQ>
__device__ __forceinline__ void moments(const Part &p, const v4f (&v)[kC][kQ], float *red, float &mean, float &m2)
{
    float s = 0.0f;
#pragma unroll
    for (int ci = 0; ci < kC; ci++)
#pragma unroll
        for (int qi = 0; qi < kQ; qi++) s += own_sum(v[ci][qi], where(p, ci, qi).first);
    mean = block_sum(s, red) / ((float)p.channels * (float)p.len);
    float q = 0.0f;
#pragma unroll
    for (int ci = 0; ci < kC; ci++)
#pragma unroll
        for (int qi = 0; qi < kQ; qi++) {
            const v4f d = v[ci][qi] - mean;
            q += own_sum(d * d, where(p, ci, qi).first);
        }
    m2 = block_sum(q, red);
}


// Joins `parts` parts' means and sums of squared differences; count(i) values are in part i.  For a whole workgroup.
template <class F>
__device__ __forceinline__ void join(const float2 *parts, int n, float total, F &&count, float *red, float &mean, float &m2)
{
    const float pivot = parts[0].x;   // equal means give that mean
    float s = 0.0f;
    for (int i = threadIdx.x; i < n; i += blockDim.x) s += (parts[i].x - pivot) * (count(i) / total);
    mean = pivot + block_sum(s, red);
    float q = 0.0f;
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
        const float d = parts[i].x - mean;
        q += parts[i].y + count(i) * (d * d);
    }
    m2 = block_sum(q, red);
}

// ------------------------------------------------------------------------------- [N, C, inner], inner of 4 and more

enum Mode { kWhole, kFirst, kSecond };   // a group in one workgroup; the two launches over parts

// `stats`: of each part (mean, sum of squared differences).
template <int kC, int kQ, int kMode>
__global__ __launch_bounds__(1024) void gn_fwd_k(Sizes s, float eps, int act, const float *x, const float *scale, const float *bias, float *y,
                                                 float *means, float *rstds, float2 *stats)
{
    __shared__ float red[16];
    const size_t block = block_id(), group = kMode == kWhole ? block : block / s.parts;
    if (block >= s.blocks) return;
    const int k = kMode == kWhole ? 0 : (int)(block % s.parts), g = (int)(group % s.G);
    const Part p = part_of(s, group / s.G, g, k);
    v4f v[kC][kQ];
    load_part(p, x, v);
    float mean, m2;
    if (kMode != kSecond) moments(p, v, red, mean, m2);
    if (kMode == kFirst) {
        if (threadIdx.x == 0) stats[block] = make_float2(mean, m2);
        return;
    }
    const float total = (float)s.Cg * (float)s.inner;
    if (kMode == kSecond)
        join(
            stats + group * s.parts, s.parts, total,
            [&](int i) {
                const Part o = part_of(s, 0, 0, i);
                return (float)o.channels * (float)o.len;
            },
            red, mean, m2);
    const float rstd = 1.0f / sqrtf(m2 / total + eps);
    if (threadIdx.x == 0 && k == 0) {
        means[group] = mean;
        rstds[group] = rstd;
    }
    with_activation(act, [&](auto kind) {
#pragma unroll
        for (int ci = 0; ci < kC; ci++) {
            const size_t c = (size_t)g * s.Cg + where(p, ci, 0).c;
            const float a = rstd * scale[c], b = bias[c];
#pragma unroll
            for (int qi = 0; qi < kQ; qi++) {
                v4f o;
#pragma unroll
                for (int e = 0; e < 4; e++) o[e] = act_value<kind.value>((v[ci][qi][e] - mean) * a + b);
                store4(y + where(p, ci, qi).at, o);
            }
        }
    });
}

// `sums`: of dz and dz xhat over each piece of each channel.
template <int kC, int kQ, int kMode>
__global__ __launch_bounds__(1024) void gn_bwd_k(Sizes s, int act, const float *dy, const float *x, const float *scale, const float *bias,
                                                 const float *means, const float *rstds, float2 *sums, float *dx)
{
    __shared__ float red[16];
    __shared__ float2 waves[kC * 16];
    const size_t block = block_id(), group = kMode == kWhole ? block : block / s.parts, n = group / s.G;
    if (block >= s.blocks) return;
    const int k = kMode == kWhole ? 0 : (int)(block % s.parts), g = (int)(group % s.G);
    const Part p = part_of(s, n, g, k);
    v4f v[kC][kQ], d[kC][kQ];
    load_part(p, x, v);
    load_part(p, dy, d);
    const float mean = means[group], rstd = rstds[group];
    with_activation(act, [&](auto kind) {
#pragma unroll
        for (int ci = 0; ci < kC; ci++) {
            const size_t c = (size_t)g * s.Cg + where(p, ci, 0).c;
            const float a = scale[c], b = bias[c];
#pragma unroll
            for (int qi = 0; qi < kQ; qi++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    v[ci][qi][e] = (v[ci][qi][e] - mean) * rstd;
                    d[ci][qi][e] = act_grad<kind.value>(d[ci][qi][e], v[ci][qi][e] * a + b);
                }
        }
    });
    float s1 = 0.0f, s2 = 0.0f;
    if (kMode != kSecond) {   // a channel's sums: along its lanes, and where it has several wavefronts, over those
        const int lanes = min(p.P, 64);
        float2 own[kC];
#pragma unroll
        for (int ci = 0; ci < kC; ci++) {
            float t = 0.0f, q = 0.0f;
#pragma unroll
            for (int qi = 0; qi < kQ; qi++) {
                const int first = where(p, ci, qi).first;
                t += own_sum(d[ci][qi], first);
                q += own_sum(d[ci][qi] * v[ci][qi], first);
            }
            own[ci] = make_float2(lanes_sum(t, lanes), lanes_sum(q, lanes));
            if (p.P > 64 && (threadIdx.x & 63) == 0) waves[ci * 16 + (threadIdx.x >> 6)] = own[ci];
        }
        if (p.P > 64) meet();
        const int row = p.row;
        const bool leads = p.lane == 0 && row < p.rows;
#pragma unroll
        for (int ci = 0; ci < kC; ci++) {
            const int c = row + ci * p.rows;
            if (!leads || c >= p.channels) continue;
            if (p.P > 64) {
                own[ci] = waves[ci * 16 + (threadIdx.x >> 6)];
                for (int i = 1; i < p.P / 64; i++) {
                    const float2 o = waves[ci * 16 + (threadIdx.x >> 6) + i];
                    own[ci] = make_float2(own[ci].x + o.x, own[ci].y + o.y);
                }
            }
            const size_t in_all = (size_t)g * s.Cg + p.c0 + c;
            sums[(n * s.C + in_all) * s.pieces + k % s.pieces] = own[ci];
            const float a = scale[in_all];
            s1 += a * own[ci].x;
            s2 += a * own[ci].y;
        }
        if (kMode == kFirst) return;
    } else {
        const float2 *const of = sums + (n * s.C + (size_t)g * s.Cg) * s.pieces;
        for (size_t i = threadIdx.x; i < (size_t)s.Cg * s.pieces; i += blockDim.x) {
            const float a = scale[(size_t)g * s.Cg + i / s.pieces];
            s1 += a * of[i].x;
            s2 += a * of[i].y;
        }
    }
    const float total = (float)s.Cg * (float)s.inner;
    s1 = block_sum(s1, red) / total;
    s2 = block_sum(s2, red) / total;
#pragma unroll
    for (int ci = 0; ci < kC; ci++) {
        const float a = scale[(size_t)g * s.Cg + where(p, ci, 0).c];
#pragma unroll
        for (int qi = 0; qi < kQ; qi++) {
            v4f o;
#pragma unroll
            for (int e = 0; e < 4; e++) o[e] = rstd * (d[ci][qi][e] * a - s1 - v[ci][qi][e] * s2);
            store4(dx + where(p, ci, qi).at, o);
        }
    }
}

// Adds `rows` rows of sums, C channels of `pieces` each: eight channels of a workgroup by thirty-two lanes.  red: kFoldRed values of LDS.
constexpr int kFoldRed = 32 * 9;
struct Fold {
    size_t rows, C;
    int pieces;
    const float2 *sums;
    float *dscale, *dbias;
};
__device__ __forceinline__ void fold(const Fold &f, size_t block, float2 *red)
{
    const int col = threadIdx.x & 7, lane = threadIdx.x >> 3;
    const size_t c = block * 8 + col;
    LongSum sum_x, sum_y;
    if (c < f.C) {
#pragma unroll 8
        for (size_t i = lane; i < f.rows * f.pieces; i += 32) {
            const float2 v = f.pieces == 1 ? f.sums[i * f.C + c] : f.sums[(i / f.pieces * f.C + c) * f.pieces + i % f.pieces];
            sum_x.add(v.x);
            sum_y.add(v.y);
        }
    }
    float s = sum_x.sum, q = sum_y.sum;
    red[lane * 9 + col] = make_float2(s, q);
    meet();
    if (lane == 0 && c < f.C) {
        for (int i = 1; i < 32; i++) {
            s += red[i * 9 + col].x;
            q += red[i * 9 + col].y;
        }
        f.dbias[c] = s;
        f.dscale[c] = q;
    }
}
__global__ __launch_bounds__(kBlock) void gn_fold_k(Fold f)
{
    __shared__ float2 red[kFoldRed];
    fold(f, block_id(), red);
}

// ------------------------------------------------------------------------------- [N, inner, C]

// V channels to a thread (four where C is a multiple of four), C / V threads to a pixel, as many pixels at once as 256 threads take; more
// channels than that are taken one run of 256 V after the other.
struct Rows {
    size_t C, inner;
    int Cg, G, S;       // S: runs of pixels of a sample
    int U, R;           // threads to a pixel, pixels at once
    size_t runs;        // of all samples
    int per_group, per_channel;   // lanes that join what a workgroup's threads have of one, powers of two
};

template <int V>
struct Vec {
    typedef float type __attribute__((ext_vector_type(V)));
};
template <>
struct Vec<1> {
    typedef float type;
};
template <int V>
__device__ __forceinline__ float &lane_of(typename Vec<V>::type &v, int e)
{
    return ((float *)&v)[e];
}

struct Run {
    size_t n, at;    // the sample, its first value
    size_t p0;       // pixels from p0 on
    int count, k;
};
__device__ __forceinline__ Run run_of(const Rows &r)
{
    Run u;
    u.n = block_id() / r.S;
    u.k = (int)(block_id() % r.S);
    u.p0 = r.inner * u.k / r.S;
    u.count = (int)(r.inner * (u.k + 1) / r.S - u.p0);
    u.at = (u.n * r.inner + u.p0) * r.C;
    return u;
}
__device__ __forceinline__ int pixels_in(const Rows &r, int i) { return (int)(r.inner * (i + 1) / r.S - r.inner * i / r.S); }

// Statistics of a run of pixels, group by group: eight pixels at a time in registers, joined per channel, then per group.
// (Few groups have many lanes each: [64, 32 x 32, 64] in one group takes 17.5 us, with eight lanes 71; [215, 63 x 51, 4] in two 16 and 42.)
template <int V>
__global__ __launch_bounds__(kBlock) void gn_last_stats_k(Rows r, const float *x, float2 *stats)
{
    extern __shared__ float2 entry[];   // [pixel lane][channel]: mean, sum of squared differences
    typedef typename Vec<V>::type vec __attribute__((aligned(4)));
    if (block_id() >= r.runs) return;
    const Run run = run_of(r);
    const int row = r.R > 1 ? threadIdx.x / r.U : 0, u0 = r.R > 1 ? threadIdx.x % r.U : threadIdx.x;
    const int mine = row < r.R && row < run.count ? (run.count - row + r.R - 1) / r.R : 0;
    for (int u = u0; u < r.U && row < r.R; u += kBlock) {
        const float *const at = x + run.at + (size_t)row * r.C + (size_t)u * V;
        const size_t step = (size_t)r.R * r.C;
        float mean[V], m2[V];
#pragma unroll
        for (int e = 0; e < V; e++) mean[e] = m2[e] = 0.0f;
        int j = 0;
        for (; j + 8 <= mine; j += 8) {
            vec v[8];
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = *(const vec *)(at + (size_t)(j + i) * step);
            const float share = 8.0f / (float)(j + 8), weight = (float)j * share;
#pragma unroll
            for (int e = 0; e < V; e++) {
                float m = 0.0f, q = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; i++) m += lane_of<V>(v[i], e);
                m *= 0.125f;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float d = lane_of<V>(v[i], e) - m;
                    q += d * d;
                }
                const float d = m - mean[e];
                mean[e] += d * share;
                m2[e] += q + d * d * weight;
            }
        }
        for (; j < mine; j++) {
            vec v = *(const vec *)(at + (size_t)j * step);
            const float share = 1.0f / (float)(j + 1);
#pragma unroll
            for (int e = 0; e < V; e++) {
                const float d = lane_of<V>(v, e) - mean[e];
                mean[e] += d * share;
                m2[e] += d * d * ((float)j * share);
            }
        }
#pragma unroll
        for (int e = 0; e < V; e++) entry[(size_t)row * r.C + (size_t)u * V + e] = make_float2(mean[e], m2[e]);
    }
    meet();
    const int rows = min(r.R, run.count), n = rows * r.Cg, lane = threadIdx.x & (r.per_group - 1);
    const float total = (float)run.count * (float)r.Cg;
    auto held = [&](int row) { return (float)((run.count - row + r.R - 1) / r.R); };
    for (int g = threadIdx.x / r.per_group; g < r.G; g += kBlock / r.per_group) {
        const float pivot = entry[g * r.Cg].x;
        float m = 0.0f, q = 0.0f;
        for (int i = lane; i < n; i += r.per_group) m += (entry[(size_t)(i / r.Cg) * r.C + g * r.Cg + i % r.Cg].x - pivot) * (held(i / r.Cg) / total);
        m = pivot + lanes_sum(m, r.per_group);
        for (int i = lane; i < n; i += r.per_group) {
            const float2 o = entry[(size_t)(i / r.Cg) * r.C + g * r.Cg + i % r.Cg];
            const float d = o.x - m;
            q += o.y + held(i / r.Cg) * (d * d);
        }
        q = lanes_sum(q, r.per_group);
        if (lane == 0) stats[block_id() * r.G + g] = make_float2(m, q);
    }
}

// What a thread needs of its channels: y = act((x - mean) a + b).
template <int V>
struct Channels {
    float mean[V], a[V], b[V];
};

template <int V>
__global__ __launch_bounds__(kBlock) void gn_last_apply_k(Rows r, float eps, int act, const float *x, const float *scale, const float *bias, float *y,
                                                          float *means, float *rstds, const float2 *stats)
{
    extern __shared__ float2 entry[];   // [group]: mean, rstd
    typedef typename Vec<V>::type vec __attribute__((aligned(4)));
    if (block_id() >= r.runs) return;
    const Run run = run_of(r);
    const int lane = threadIdx.x & 7;
    for (int g = threadIdx.x >> 3; g < r.G; g += kBlock / 8) {   // a group's runs by eight lanes, eight runs to a lane
        const float2 *const of = stats + run.n * r.S * r.G + g;
        const float all = (float)r.inner;
        float2 part[kRuns / 8];
        float w[kRuns / 8];
#pragma unroll
        for (int i = 0; i < kRuns / 8; i++) part[i] = of[(size_t)min(lane + 8 * i, r.S - 1) * r.G];
#pragma unroll
        for (int i = 0; i < kRuns / 8; i++) w[i] = lane + 8 * i < r.S ? (float)pixels_in(r, lane + 8 * i) : 0.0f;
        const float pivot = __shfl(part[0].x, 0, 8);   // equal means give that mean
        float m = 0.0f, q = 0.0f;
#pragma unroll
        for (int i = 0; i < kRuns / 8; i++) m += (part[i].x - pivot) * (w[i] / all);
        m = pivot + lanes_sum(m, 8);
#pragma unroll
        for (int i = 0; i < kRuns / 8; i++) {
            const float d = part[i].x - m;
            q += (w[i] > 0.0f ? part[i].y : 0.0f) + w[i] * (float)r.Cg * (d * d);
        }
        const float rstd = 1.0f / sqrtf(lanes_sum(q, 8) / (all * (float)r.Cg) + eps);
        if (lane == 0) {
            entry[g] = make_float2(m, rstd);
            if (run.k == 0) {
                means[run.n * r.G + g] = m;
                rstds[run.n * r.G + g] = rstd;
            }
        }
    }
    meet();
    const int row = r.R > 1 ? threadIdx.x / r.U : 0, u0 = r.R > 1 ? threadIdx.x % r.U : threadIdx.x;
    if (row >= r.R) return;
    with_activation(act, [&](auto kind) {
        for (int u = u0; u < r.U; u += kBlock) {
            Channels<V> ch;
#pragma unroll
            for (int e = 0; e < V; e++) {
                const int c = u * V + e;
                const float2 o = entry[c / r.Cg];
                ch.mean[e] = o.x;
                ch.a[e] = o.y * scale[c];
                ch.b[e] = bias[c];
            }
            const size_t first = run.at + (size_t)row * r.C + (size_t)u * V, step = (size_t)r.R * r.C;
            auto one = [&](vec v) {
                vec o;
#pragma unroll
                for (int e = 0; e < V; e++) lane_of<V>(o, e) = act_value<kind.value>((lane_of<V>(v, e) - ch.mean[e]) * ch.a[e] + ch.b[e]);
                return o;
            };
            const int mine = row < run.count ? (run.count - row + r.R - 1) / r.R : 0;
            int j = 0;
            for (; j + 4 <= mine; j += 4) {
                vec v[4];
#pragma unroll
                for (int i = 0; i < 4; i++) v[i] = *(const vec *)(x + first + (size_t)(j + i) * step);
#pragma unroll
                for (int i = 0; i < 4; i++) *(vec *)(y + first + (size_t)(j + i) * step) = one(v[i]);
            }
            for (; j < mine; j++) *(vec *)(y + first + (size_t)j * step) = one(*(const vec *)(x + first + (size_t)j * step));
        }
    });
}

// kDx = false: sums of dz and dz xhat over a run of pixels, per channel (sums) and, times scale, per group (gsums).  kDx: dx.
template <int V, bool kDx>
__global__ __launch_bounds__(kBlock) void gn_last_grad_k(Rows r, int act, const float *dy, const float *x, const float *scale, const float *bias,
                                                         const float *means, const float *rstds, float2 *sums, float2 *gsums, float *dx,
                                                         Fold f)
{
    extern __shared__ float2 entry[];   // kDx: [group]: s1, s2, or the fold's; else [pixel lane][channel]
    typedef typename Vec<V>::type vec __attribute__((aligned(4)));
    if (block_id() >= r.runs) {   // the sums over all runs wait for nothing that this launch does: they ride behind it
        if (kDx) fold(f, block_id() - r.runs, entry);
        return;
    }
    const Run run = run_of(r);
    if (kDx) {
        const float total = (float)r.inner * (float)r.Cg;
        const int lane = threadIdx.x & 7;
        for (int g = threadIdx.x >> 3; g < r.G; g += kBlock / 8) {
            float s = 0.0f, q = 0.0f;
            float2 part[kRuns / 8];
#pragma unroll
            for (int i = 0; i < kRuns / 8; i++) part[i] = gsums[(run.n * r.S + min(lane + 8 * i, r.S - 1)) * r.G + g];
#pragma unroll
            for (int i = 0; i < kRuns / 8; i++) {
                s += lane + 8 * i < r.S ? part[i].x : 0.0f;
                q += lane + 8 * i < r.S ? part[i].y : 0.0f;
            }
            s = lanes_sum(s, 8);
            q = lanes_sum(q, 8);
            if (lane == 0) entry[g] = make_float2(s / total, q / total);
        }
        meet();
    }
    const int row = r.R > 1 ? threadIdx.x / r.U : 0, u0 = r.R > 1 ? threadIdx.x % r.U : threadIdx.x;
    const int mine = row < r.R && row < run.count ? (run.count - row + r.R - 1) / r.R : 0;
    with_activation(act, [&](auto kind) {
        for (int u = u0; u < r.U && row < r.R; u += kBlock) {
            float mean[V], rstd[V], a[V], b[V], s[V], q[V], all_s[V], all_q[V];
#pragma unroll
            for (int e = 0; e < V; e++) {
                const int c = u * V + e, g = c / r.Cg;
                mean[e] = means[run.n * r.G + g];
                rstd[e] = rstds[run.n * r.G + g];
                a[e] = scale[c];
                b[e] = bias[c];
                s[e] = kDx ? entry[g].x : 0.0f;
                q[e] = kDx ? entry[g].y : 0.0f;
                all_s[e] = all_q[e] = 0.0f;
            }
            const size_t first = run.at + (size_t)row * r.C + (size_t)u * V, step = (size_t)r.R * r.C;
            auto one = [&](vec v, vec d, size_t at) {
                vec o;
#pragma unroll
                for (int e = 0; e < V; e++) {
                    const float xhat = (lane_of<V>(v, e) - mean[e]) * rstd[e];
                    const float dz = act_grad<kind.value>(lane_of<V>(d, e), xhat * a[e] + b[e]);
                    if (kDx) {
                        lane_of<V>(o, e) = rstd[e] * (dz * a[e] - s[e] - xhat * q[e]);
                    } else {
                        s[e] += dz;
                        q[e] += dz * xhat;
                    }
                }
                if (kDx) *(vec *)(dx + at) = o;
            };
            auto put_aside = [&]() {
#pragma unroll
                for (int e = 0; e < V; e++) {
                    all_s[e] += s[e];
                    all_q[e] += q[e];
                    s[e] = q[e] = 0.0f;
                }
            };
            int j = 0;
            for (; j + 4 <= mine; j += 4) {
                if (!kDx && (j & 63) == 0) put_aside();   // sums of 64 values each, so that many like ones do not round the same way for long
                vec v[4], d[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    v[i] = *(const vec *)(x + first + (size_t)(j + i) * step);
                    d[i] = *(const vec *)(dy + first + (size_t)(j + i) * step);
                }
#pragma unroll
                for (int i = 0; i < 4; i++) one(v[i], d[i], first + (size_t)(j + i) * step);
            }
            for (; j < mine; j++) {
                const size_t at = first + (size_t)j * step;
                one(*(const vec *)(x + at), *(const vec *)(dy + at), at);
            }
            if (!kDx) {
                put_aside();
#pragma unroll
                for (int e = 0; e < V; e++) entry[(size_t)row * r.C + (size_t)u * V + e] = make_float2(all_s[e], all_q[e]);
            }
        }
    });
    if (kDx) return;
    meet();
    const int part = threadIdx.x & (r.per_channel - 1);
    for (size_t c = threadIdx.x / r.per_channel; c < r.C; c += kBlock / r.per_channel) {
        float2 t = make_float2(0.0f, 0.0f);
        for (int i = part; i < r.R; i += r.per_channel) {
            const float2 o = entry[(size_t)i * r.C + c];
            t = make_float2(t.x + o.x, t.y + o.y);
        }
        t = make_float2(lanes_sum(t.x, r.per_channel), lanes_sum(t.y, r.per_channel));
        if (part) continue;
        sums[block_id() * r.C + c] = t;
        const float a = scale[c];
        entry[c] = make_float2(a * t.x, a * t.y);
    }
    meet();
    const int lane = threadIdx.x & 7;
    for (int g = threadIdx.x >> 3; g < r.G; g += kBlock / 8) {
        float s = 0.0f, q = 0.0f;
        for (int i = lane; i < r.Cg; i += 8) {
            s += entry[(size_t)g * r.Cg + i].x;
            q += entry[(size_t)g * r.Cg + i].y;
        }
        s = lanes_sum(s, 8);
        q = lanes_sum(q, 8);
        if (lane == 0) gsums[block_id() * r.G + g] = make_float2(s, q);
    }
}

// ------------------------------------------------------------------------------- [N, inner, C], a group in one workgroup

// Groups of 8 to 64 channels, a power of two of them: `1 << bits` threads to a pixel's quads, and the group's values in registers as above.
// A pixel's piece may be less than a line of 128 bytes, which then belongs to several groups: blocks of one XCD, whose L2
// holds it meanwhile, take groups that lie side by side.
struct Held {
    size_t C, inner;
    int Cg, G, bits;
    unsigned groups, per;   // all of them, an XCD's
};
__device__ __forceinline__ size_t held_group(const Held &h) { return (block_id() & 7) * h.per + (block_id() >> 3); }

template <int kQ>
__global__ __launch_bounds__(1024) void gn_held_fwd_k(Held h, float eps, int act, const float *x, const float *scale, const float *bias, float *y,
                                                      float *means, float *rstds)
{
    __shared__ float red[16];
    const size_t group = held_group(h);
    if (block_id() >= 8 * (size_t)h.per || group >= h.groups) return;
    const int quad = threadIdx.x & ((1 << h.bits) - 1), row = threadIdx.x >> h.bits, rows = blockDim.x >> h.bits, last = (int)h.inner - 1;
    const int c = (int)(group % h.G) * h.Cg + 4 * quad;
    const size_t base = group / h.G * h.inner * h.C + c;
    v4f v[kQ];
#pragma unroll
    for (int i = 0; i < kQ; i++) v[i] = load4(x + base + (size_t)min(row + i * rows, last) * h.C);
    const v4f a0 = load4(scale + c), b = load4(bias + c);
    const float total = (float)h.Cg * (float)h.inner;
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < kQ; i++) s += own_sum(v[i], row + i * rows <= last ? 0 : 4);
    const float mean = block_sum(s, red) / total;
    float q = 0.0f;
#pragma unroll
    for (int i = 0; i < kQ; i++) {
        const v4f d = v[i] - mean;
        q += own_sum(d * d, row + i * rows <= last ? 0 : 4);
    }
    const float rstd = 1.0f / sqrtf(block_sum(q, red) / total + eps);
    if (threadIdx.x == 0) {
        means[group] = mean;
        rstds[group] = rstd;
    }
    const v4f a = rstd * a0;
    with_activation(act, [&](auto kind) {
#pragma unroll
        for (int i = 0; i < kQ; i++) {
            v4f o;
#pragma unroll
            for (int e = 0; e < 4; e++) o[e] = act_value<kind.value>((v[i][e] - mean) * a[e] + b[e]);
            if (row + i * rows <= last) store4(y + base + (size_t)(row + i * rows) * h.C, o);
        }
    });
}

// `sums`: of dz and dz xhat over each sample's channels.
template <int kQ>
__global__ __launch_bounds__(1024) void gn_held_bwd_k(Held h, int act, const float *dy, const float *x, const float *scale, const float *bias,
                                                      const float *means, const float *rstds, float2 *sums, float *dx)
{
    __shared__ float red[16];
    __shared__ float2 waves[16][64];
    const size_t group = held_group(h);
    if (block_id() >= 8 * (size_t)h.per || group >= h.groups) return;
    const int quad = threadIdx.x & ((1 << h.bits) - 1), row = threadIdx.x >> h.bits, rows = blockDim.x >> h.bits, last = (int)h.inner - 1;
    const int c = (int)(group % h.G) * h.Cg + 4 * quad;
    const size_t base = group / h.G * h.inner * h.C + c;
    v4f v[kQ], d[kQ];
#pragma unroll
    for (int i = 0; i < kQ; i++) {
        const size_t at = base + (size_t)min(row + i * rows, last) * h.C;
        v[i] = load4(x + at);
        d[i] = load4(dy + at);
    }
    const v4f a = load4(scale + c), b = load4(bias + c);
    const float mean = means[group], rstd = rstds[group];
    v4f t{0.0f, 0.0f, 0.0f, 0.0f}, u = t;
    with_activation(act, [&](auto kind) {
#pragma unroll
        for (int i = 0; i < kQ; i++) {
            const bool own = row + i * rows <= last;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                v[i][e] = (v[i][e] - mean) * rstd;
                d[i][e] = act_grad<kind.value>(d[i][e], v[i][e] * a[e] + b[e]);
                t[e] += own ? d[i][e] : 0.0f;
                u[e] += own ? d[i][e] * v[i][e] : 0.0f;
            }
        }
    });
#pragma unroll
    for (int e = 0; e < 4; e++)   // the wavefront's pixels, then the wavefronts
        for (int m = 32; m >> h.bits; m >>= 1) {
            t[e] += __shfl_xor(t[e], m, 64);
            u[e] += __shfl_xor(u[e], m, 64);
        }
    if ((threadIdx.x & 63) == quad) {
#pragma unroll
        for (int e = 0; e < 4; e++) waves[threadIdx.x >> 6][4 * quad + e] = make_float2(t[e], u[e]);
    }
    meet();
    float s1 = 0.0f, s2 = 0.0f;
    if ((int)threadIdx.x < h.Cg) {
        float2 o = waves[0][threadIdx.x];
        for (unsigned i = 1; i < blockDim.x / 64; i++) o = make_float2(o.x + waves[i][threadIdx.x].x, o.y + waves[i][threadIdx.x].y);
        const size_t at = group % h.G * h.Cg + threadIdx.x;
        sums[group / h.G * h.C + at] = o;
        s1 = scale[at] * o.x;
        s2 = scale[at] * o.y;
    }
    const float total = (float)h.Cg * (float)h.inner;
    s1 = block_sum(s1, red) / total;
    s2 = block_sum(s2, red) / total;
#pragma unroll
    for (int i = 0; i < kQ; i++) {
        v4f o;
#pragma unroll
        for (int e = 0; e < 4; e++) o[e] = rstd * (d[i][e] * a[e] - s1 - v[i][e] * s2);
        if (row + i * rows <= last) store4(dx + base + (size_t)(row + i * rows) * h.C, o);
    }
}

// ------------------------------------------------------------------------------- one value to a channel: rows of a dense layer

constexpr int kRowValues = 16;   // of a lane: groups of up to 1024 channels

// A wavefront per sample and group.
__global__ __launch_bounds__(kBlock) void gn_row_fwd_k(size_t groups, int Cg, int G, float eps, int act, const float *x, const float *scale,
                                                       const float *bias, float *y, float *means, float *rstds)
{
    const size_t group = block_id() * 4 + (threadIdx.x >> 6);
    if (group >= groups) return;
    const int lane = threadIdx.x & 63, c0 = (int)(group % G) * Cg;
    const size_t at = group * Cg;
    float v[kRowValues], s = 0.0f, q = 0.0f;
#pragma unroll
    for (int i = 0; i < kRowValues; i++) {
        if (64 * i >= Cg) break;   // uniform
        v[i] = x[at + min(lane + 64 * i, Cg - 1)];
        s += lane + 64 * i < Cg ? v[i] : 0.0f;
    }
    const float mean = lanes_sum(s, 64) / (float)Cg;
#pragma unroll
    for (int i = 0; i < kRowValues; i++) {
        if (64 * i >= Cg) break;
        const float d = v[i] - mean;
        q += lane + 64 * i < Cg ? d * d : 0.0f;
    }
    const float rstd = 1.0f / sqrtf(lanes_sum(q, 64) / (float)Cg + eps);
    if (lane == 0) {
        means[group] = mean;
        rstds[group] = rstd;
    }
    with_activation(act, [&](auto kind) {
#pragma unroll
        for (int i = 0; i < kRowValues; i++) {
            const int c = lane + 64 * i;
            if (c >= Cg) break;
            y[at + c] = act_value<kind.value>((v[i] - mean) * (rstd * scale[c0 + c]) + bias[c0 + c]);
        }
    });
}

__global__ __launch_bounds__(kBlock) void gn_row_dx_k(size_t groups, int Cg, int G, int act, const float *dy, const float *x, const float *scale,
                                                      const float *bias, const float *means, const float *rstds, float *dx)
{
    const size_t group = block_id() * 4 + (threadIdx.x >> 6);
    if (group >= groups) return;
    const int lane = threadIdx.x & 63, c0 = (int)(group % G) * Cg;
    const size_t at = group * Cg;
    const float mean = means[group], rstd = rstds[group];
    float v[kRowValues], d[kRowValues], s = 0.0f, q = 0.0f;
#pragma unroll
    for (int i = 0; i < kRowValues; i++) {
        if (64 * i >= Cg) break;   // uniform
        const int c = min(lane + 64 * i, Cg - 1);
        v[i] = (x[at + c] - mean) * rstd;
        d[i] = dy[at + c];
    }
    with_activation(act, [&](auto kind) {
#pragma unroll
        for (int i = 0; i < kRowValues; i++) {
            if (64 * i >= Cg) break;
            const int c = min(lane + 64 * i, Cg - 1);
            const float a = scale[c0 + c];
            d[i] = act_grad<kind.value>(d[i], v[i] * a + bias[c0 + c]) * a;
            const bool own = lane + 64 * i < Cg;
            s += own ? d[i] : 0.0f;
            q += own ? d[i] * v[i] : 0.0f;
        }
    });
    const float s1 = lanes_sum(s, 64) / (float)Cg, s2 = lanes_sum(q, 64) / (float)Cg;
#pragma unroll
    for (int i = 0; i < kRowValues; i++) {
        const int c = lane + 64 * i;
        if (c >= Cg) break;
        dx[at + c] = rstd * (d[i] - s1 - v[i] * s2);
    }
}

// Sums over a run of samples, 64 channels by four samples at a time.
__global__ __launch_bounds__(kBlock) void gn_row_sums_k(size_t N, size_t C, int Cg, int G, int S, int act, const float *dy, const float *x,
                                                        const float *scale, const float *bias, const float *means, const float *rstds, float2 *sums)
{
    __shared__ float2 red[4][64];
    const size_t tiles = (C + 63) / 64, c = block_id() % tiles * 64 + (threadIdx.x & 63), run = block_id() / tiles;
    if (run >= (size_t)S) return;
    const size_t from = N * run / S, to = N * (run + 1) / S;
    float s = 0.0f, q = 0.0f;
    if (c < C) {
        const float a = scale[c], b = bias[c];
        const size_t g = c / Cg;
        with_activation(act, [&](auto kind) {
            for (size_t first = from + (threadIdx.x >> 6); first < to; first += 256) {   // (of 64 values each, as below)
                const size_t end = min(first + 256, to);
                float t = 0.0f, u = 0.0f;
#pragma unroll 4
                for (size_t n = first; n < end; n += 4) {
                    const float xhat = (x[n * C + c] - means[n * G + g]) * rstds[n * G + g];
                    const float dz = act_grad<kind.value>(dy[n * C + c], xhat * a + b);
                    t += dz;
                    u += dz * xhat;
                }
                s += t;
                q += u;
            }
        });
    }
    red[threadIdx.x >> 6][threadIdx.x & 63] = make_float2(s, q);
    meet();
    if (threadIdx.x < 64 && c < C) {
        float2 t = red[0][threadIdx.x];
        for (int i = 1; i < 4; i++) t = make_float2(t.x + red[i][threadIdx.x].x, t.y + red[i][threadIdx.x].y);
        sums[run * C + c] = t;
    }
}

// ------------------------------------------------------------------------------- any other shape

// Rows of two and three values, groups of more than 1024 channels of one value, more than 8192 channels last.
struct Place {
    size_t N, C, inner, Cg, G;
    int last;
    __device__ size_t at(size_t n, size_t g, size_t i) const
    {
        if (!last) return (n * C + g * Cg) * inner + i;
        return (n * inner + i / Cg) * C + g * Cg + i % Cg;
    }
    __device__ size_t channel(size_t g, size_t i) const { return g * Cg + (last ? i % Cg : i / inner); }
};

// A workgroup per group.
__global__ __launch_bounds__(kBlock) void gn_any_fwd_k(Place p, float eps, int act, const float *x, const float *scale, const float *bias, float *y,
                                                       float *means, float *rstds)
{
    __shared__ float red[16];
    const size_t group = block_id(), n = group / p.G, g = group % p.G, L = p.Cg * p.inner;
    if (n >= p.N) return;
    LongSum s, q;
    for (size_t i = threadIdx.x; i < L; i += kBlock) s.add(x[p.at(n, g, i)]);
    const float mean = L ? block_sum(s.sum, red) / (float)L : 0.0f;
    for (size_t i = threadIdx.x; i < L; i += kBlock) {
        const float d = x[p.at(n, g, i)] - mean;
        q.add(d * d);
    }
    const float rstd = 1.0f / sqrtf((L ? block_sum(q.sum, red) / (float)L : 0.0f) + eps);
    with_activation(act, [&](auto kind) {
        for (size_t i = threadIdx.x; i < L; i += kBlock) {
            const size_t at = p.at(n, g, i), c = p.channel(g, i);
            y[at] = act_value<kind.value>((x[at] - mean) * (rstd * scale[c]) + bias[c]);
        }
    });
    if (threadIdx.x == 0) {
        means[group] = mean;
        rstds[group] = rstd;
    }
}

// A thread per sample and channel: its sums of dz and dz xhat, of 64 values each and then of those.  ([246, 992, 2] took 250 us by workgroups.)
__global__ __launch_bounds__(kBlock) void gn_any_sums_k(Place p, int act, const float *dy, const float *x, const float *scale, const float *bias,
                                                        const float *means, const float *rstds, float2 *sums)
{
    const size_t i = block_id() * kBlock + threadIdx.x, n = i / p.C, c = i % p.C, g = c / p.Cg;
    if (n >= p.N) return;
    const float mean = means[n * p.G + g], rstd = rstds[n * p.G + g], a = scale[c], b = bias[c];
    const size_t first = p.last ? n * p.inner * p.C + c : i * p.inner, step = p.last ? p.C : 1;
    float s = 0.0f, q = 0.0f;
    with_activation(act, [&](auto kind) {
        for (size_t from = 0; from < p.inner; from += 64) {
            const size_t to = min(from + 64, p.inner);
            float t = 0.0f, u = 0.0f;
#pragma unroll 4
            for (size_t k = from; k < to; k++) {
                const size_t at = first + k * step;
                const float xhat = (x[at] - mean) * rstd, dz = act_grad<kind.value>(dy[at], xhat * a + b);
                t += dz;
                u += dz * xhat;
            }
            s += t;
            q += u;
        }
    });
    sums[i] = make_float2(s, q);
}

// A workgroup per group.
__global__ __launch_bounds__(kBlock) void gn_any_dx_k(Place p, int act, const float *dy, const float *x, const float *scale, const float *bias,
                                                      const float *means, const float *rstds, const float2 *sums, float *dx)
{
    __shared__ float red[16];
    const size_t group = block_id(), n = group / p.G, g = group % p.G, L = p.Cg * p.inner;
    if (n >= p.N) return;
    const float mean = means[group], rstd = rstds[group];
    LongSum t, u;
    for (size_t c = g * p.Cg + threadIdx.x; c < (g + 1) * p.Cg; c += kBlock) {
        const float2 v = sums[n * p.C + c];
        t.add(v.x * scale[c]);
        u.add(v.y * scale[c]);
    }
    const float s1 = block_sum(t.sum, red) / (float)L, s2 = block_sum(u.sum, red) / (float)L;
    with_activation(act, [&](auto kind) {
        for (size_t i = threadIdx.x; i < L; i += kBlock) {
            const size_t at = p.at(n, g, i), c = p.channel(g, i);
            const float xhat = (x[at] - mean) * rstd, a = scale[c];
            const float dz = act_grad<kind.value>(dy[at], xhat * a + bias[c]);
            dx[at] = rstd * (dz * a - s1 - xhat * s2);
        }
    });
}

// ------------------------------------------------------------------------------- which of them

// The most quads that a thread holds of a tensor: 1024 threads leave each 128 registers, of which the gradient's eight quads of both its
// tensors spilled 800 values ([64, 512, 32 x 32] in 16 groups, whole: 361 us, in parts 134).
constexpr int kMost = 8, kMostGrad = 4;

// How a workgroup holds `channels` channels of `len` values, up to `most` quads to a thread: threads (0: it cannot), channels and quads
// of a thread.
struct Hold {
    int threads = 0, c = 1, q = 1, P = 1, rows = 1;
};
Hold hold_for(int channels, size_t len, int most)
{
    Hold best;
    size_t least = 0;
    const size_t quads = ceil_div(len, (size_t)4);
    for (int q = 1; q <= most; q *= 2)
        for (int c = 1; c * q <= most; c *= 2) {
            // lanes to a channel: a power of two, or whole wavefronts ([87, 160, 39 x 28] in 16 groups backward, 273 quads to a channel,
            // 70 us; with 512 lanes, or half of them to spare, 101)
            int P = 1;
            while ((size_t)P * q < quads && P <= 1024) P += P < 64 ? P : 64;
            const int rows = (channels + c - 1) / c, threads = (int)ceil_div((size_t)rows * P, (size_t)64) * 64;
            if (P > 1024 || rows > 1024 || threads > 1024) continue;
            // Places that stay empty cost what full ones do.  Four quads of one tensor to a thread, two of two, and more wavefronts with the
            // registers that this saves: the gradient of [128, 320, 16 x 16] in sixteen groups takes 38.5 us with two, 48.1 with four.
            const size_t cost = (size_t)threads * (c * q * 16 + std::abs(c * q - most / 2) * 4);
            if (best.threads && cost >= least) continue;
            least = cost;
            best.threads = threads;
            best.c = c;
            best.q = q;
            best.P = P;
            best.rows = rows;
        }
    return best;
}

// The [N, C, inner] tensors' workgroups: whole groups, or parts.
struct Split {
    Sizes s;
    Hold h;
    bool whole;
};
Split split_of(size_t N, size_t C, size_t inner, size_t G, int most)
{
    Split r;
    Sizes &s = r.s;
    s.C = C;
    s.inner = inner;
    s.Cg = (int)(C / G);
    s.G = (int)G;
    s.pieces = 1;
    s.per = s.Cg;
    s.parts = 1;
    const size_t L = C / G * inner;
    r.h = L <= (size_t)4096 * most ? hold_for(s.Cg, inner, most) : Hold{};
    // (also where a few of them leave most of the chip idle: sixteen of 32768 values take 8.9 us, in parts 9.2; 128 of them 11.3 and 14.2)
    r.whole = r.h.threads != 0;
    if (!r.whole) {
        s.pieces = (int)ceil_div(inner, (size_t)kPiece);
        s.per = s.pieces > 1 ? 1 : std::max(1, std::min(s.Cg, (int)(kPiece / inner)));
        s.per = (int)ceil_div((size_t)s.Cg, ceil_div((size_t)s.Cg, (size_t)s.per));   // (of about the same size)
        s.parts = s.pieces * (int)ceil_div((size_t)s.Cg, (size_t)s.per);
        r.h = hold_for(s.per, ceil_div(inner, (size_t)s.pieces), most);
    }
    s.P = r.h.P;
    s.rows = r.h.rows;
    s.blocks = N * G * s.parts;
    return r;
}

template <int kMax, class F>
int with_hold(const Hold &h, F &&f)
{
#define DOPT_HOLD(C, Q) \
    if constexpr (C * Q <= kMax) \
        if (h.c == C && h.q == Q) return f(std::integral_constant<int, C>{}, std::integral_constant<int, Q>{});
    DOPT_HOLD(1, 1) DOPT_HOLD(1, 2) DOPT_HOLD(1, 4) DOPT_HOLD(1, 8) DOPT_HOLD(2, 1)
    DOPT_HOLD(2, 2) DOPT_HOLD(2, 4) DOPT_HOLD(4, 1) DOPT_HOLD(4, 2) DOPT_HOLD(8, 1)
#undef DOPT_HOLD
    return fail(DOPT_HIP_ERR_UNSUPPORTED, "group norm: no kernel holds such a group");
}

// Channels-last groups in registers: threads (0: not these), quads of a thread.
struct HeldHold {
    Held h;
    int threads = 0, q = 1;
};
HeldHold held_for(size_t N, size_t C, size_t inner, size_t G, bool grad)
{
    HeldHold r;
    const int most = grad ? kMostGrad : kMost;
    const size_t Cg = C / G;
    if (Cg < 8 || Cg > 64 || (Cg & (Cg - 1)) || Cg * inner > (size_t)4096 * most) return r;
    // The gradient's runs read everything twice, but the second time from a cache of 256 MB, and in whole lines.  In registers [64, 1024, 128]
    // in 16 groups takes 37.8 us, by runs 32.0; four times as many samples 116 and 134; [37, 957, 200] in 25 groups
    // 29.3 and 30.7; [8, 256, 256] in 32 groups 9.2 and 11.0; [8, 2048, 64] in 8 groups 12.3 and 10.7.  Forward, where [64, 1024, 128]
    // takes 16.6 and 23.7 us, registers win throughout.
    const size_t in = 2 * N * C * inner * sizeof(float);
    if (grad && in < (size_t)200 << 20 && (in > (size_t)60 << 20 || Cg * inner > kPiece)) return r;
    r.h = Held{C, inner, (int)Cg, (int)G, 0, (unsigned)(N * G), (unsigned)ceil_div(N * G, (size_t)8)};
    while ((size_t)4 << r.h.bits < Cg) r.h.bits++;
    size_t least = 0;
    for (int q = 1; q <= most; q *= 2) {
        const size_t threads = ceil_div(ceil_div(inner, (size_t)q) << r.h.bits, (size_t)64) * 64;
        if (threads > 1024) continue;
        const size_t cost = threads * (q * 16 + std::abs(q - 4) * 4);   // as in hold_for
        if (r.threads && cost >= least) continue;
        least = cost;
        r.threads = (int)threads;
        r.q = q;
    }
    return r;
}

constexpr size_t kLastChannels = 8192;   // 64 KB of LDS for a run of pixels, which every launch may ask for

Rows rows_of(size_t N, size_t C, size_t inner, size_t G, int V)
{
    Rows r;
    r.C = C;
    r.inner = inner;
    r.Cg = (int)(C / G);
    r.G = (int)G;
    r.U = (int)(C / V);
    r.R = std::max(1, kBlock / r.U);
    const size_t most = std::min((size_t)kRuns, ceil_div(inner, (size_t)r.R * 8));   // (eight pixels to a thread)
    r.S = (int)std::min(most, std::max((size_t)1, ceil_div((size_t)num_cus() * 4, N)));
    r.runs = N * r.S;
    auto lanes = [](size_t n, int least) {   // of 256 threads to each of n
        int l = 64;
        while (l > least && l * n > (size_t)kBlock) l /= 2;
        return l;
    };
    r.per_group = lanes(G, 8);
    r.per_channel = lanes(C, 1);
    return r;
}

template <int kMax, class F>
int with_quads(int q, F &&f)
{
    if (q == 1) return f(std::integral_constant<int, 1>{});
    if (q == 2) return f(std::integral_constant<int, 2>{});
    if (q == 4 || kMax == 4) return f(std::integral_constant<int, 4>{});
    return f(std::integral_constant<int, kMax>{});
}

template <class F>
int with_vec(size_t C, F &&f)
{
    return C % 4 == 0 ? f(std::integral_constant<int, 4>{}) : f(std::integral_constant<int, 1>{});
}

int check(const char *who, size_t N, size_t C, size_t inner, size_t groups, int act)
{
    DOPT_REQUIRE(groups > 0 && C % groups == 0, "%s: %zu channels cannot be parted into %zu groups", who, C, groups);
    DOPT_REQUIRE(known_activation(act), "%s: there is no activation %d", who, act);
    DOPT_REQUIRE(N < ((size_t)1 << 31) && C < ((size_t)1 << 31) && inner < ((size_t)1 << 31) && N * C < ((size_t)1 << 31) &&
                     N * C * inner < ((size_t)1 << 40),
                 "%s: dimensions too large", who);
    return DOPT_HIP_OK;
}

}  // namespace

extern "C" {

int dopt_hip_group_norm(size_t N, size_t C, size_t inner, size_t groups, int channels_last, float eps, int act, const float *x,
                        const float *scale, const float *bias, float *packed)
{
    if (int rc = check("dopt_hip_group_norm", N, C, inner, groups, act)) return rc;
    const size_t total = N * C * inner, G = groups;
    if (N * C == 0) return DOPT_HIP_OK;
    DOPT_REQUIRE(packed && (total == 0 || (x && scale && bias)), "dopt_hip_group_norm: null argument");
    const size_t out = (total + 2 * N * groups) * sizeof(float), per = C * sizeof(float);
    DOPT_REQUIRE(!overlaps(packed, out, x, total * sizeof(float)) && !overlaps(packed, out, scale, per) && !overlaps(packed, out, bias, per),
                 "dopt_hip_group_norm: the result overlaps an operand");
    DOPT_ENSURE_INIT();
    float *const y = packed, *const means = packed + total, *const rstds = means + N * G;
    const bool rows = inner == 1 && C / G <= 64 * kRowValues;
    if (rows) {
        hipLaunchKernelGGL(gn_row_fwd_k, grid_of(ceil_div(N * G, (size_t)4)), dim3(kBlock), 0, stream(), N * G, (int)(C / G), (int)G, eps,
                           act, x, scale, bias, y, means, rstds);
        DOPT_LAUNCH_CHECK();
        return DOPT_HIP_OK;
    }
    const HeldHold held = channels_last && inner > 1 ? held_for(N, C, inner, G, false) : HeldHold{};
    if (held.threads)
        return with_quads<kMost>(held.q, [&](auto q) -> int {
            hipLaunchKernelGGL(gn_held_fwd_k<decltype(q)::value>, grid_of(8 * (size_t)held.h.per), dim3(held.threads), 0, stream(), held.h, eps, act, x, scale,
                               bias, y, means, rstds);
            DOPT_LAUNCH_CHECK();
            return DOPT_HIP_OK;
        });
    if (channels_last && inner > 1 && C <= kLastChannels)
        return with_vec(C, [&](auto v) -> int {
            constexpr int V = decltype(v)::value;
            const Rows r = rows_of(N, C, inner, G, V);
            float2 *const stats = (float2 *)workspace(r.runs * G * sizeof(float2));
            if (!stats) return DOPT_HIP_ERR_OOM;
            const dim3 grid = grid_of(r.runs);
            hipLaunchKernelGGL(gn_last_stats_k<V>, grid, dim3(kBlock), r.R * C * sizeof(float2), stream(), r, x, stats);
            DOPT_LAUNCH_CHECK();
            hipLaunchKernelGGL(gn_last_apply_k<V>, grid, dim3(kBlock), G * sizeof(float2), stream(), r, eps, act, x, scale, bias, y, means, rstds,
                               stats);
            DOPT_LAUNCH_CHECK();
            return DOPT_HIP_OK;
        });
    if (!channels_last && inner >= 4) {
        const Split k = split_of(N, C, inner, G, kMost);
        float2 *stats = nullptr;
        if (!k.whole && !(stats = (float2 *)workspace(N * G * k.s.parts * sizeof(float2)))) return DOPT_HIP_ERR_OOM;
        return with_hold<kMost>(k.h, [&](auto c, auto q) -> int {
            constexpr int kC = decltype(c)::value, kQ = decltype(q)::value;
            const dim3 grid = grid_of(k.s.blocks), block(k.h.threads);
            if (k.whole) {
                hipLaunchKernelGGL((gn_fwd_k<kC, kQ, kWhole>), grid, block, 0, stream(), k.s, eps, act, x, scale, bias, y, means, rstds, stats);
            } else {
                hipLaunchKernelGGL((gn_fwd_k<kC, kQ, kFirst>), grid, block, 0, stream(), k.s, eps, act, x, scale, bias, y, means, rstds, stats);
                DOPT_LAUNCH_CHECK();
                hipLaunchKernelGGL((gn_fwd_k<kC, kQ, kSecond>), grid, block, 0, stream(), k.s, eps, act, x, scale, bias, y, means, rstds, stats);
            }
            DOPT_LAUNCH_CHECK();
            return DOPT_HIP_OK;
        });
    }
    const Place p{N, C, inner, C / G, G, channels_last != 0};
    hipLaunchKernelGGL(gn_any_fwd_k, grid_of(N * G), dim3(kBlock), 0, stream(), p, eps, act, x, scale, bias, y, means, rstds);
    DOPT_LAUNCH_CHECK();
    return DOPT_HIP_OK;
}

int dopt_hip_group_norm_grad(size_t N, size_t C, size_t inner, size_t groups, int channels_last, int act, const float *dy, const float *x,
                             const float *scale, const float *bias, const float *stats, float *packed)
{
    if (int rc = check("dopt_hip_group_norm_grad", N, C, inner, groups, act)) return rc;
    if (C == 0) return DOPT_HIP_OK;
    const size_t total = N * C * inner, G = groups;
    DOPT_REQUIRE(packed && (total == 0 || (dy && x && scale && bias && stats)), "dopt_hip_group_norm_grad: null argument");
    const size_t out = (total + 2 * C) * sizeof(float), per = C * sizeof(float), in = total * sizeof(float);
    DOPT_REQUIRE(!overlaps(packed, out, dy, in) && !overlaps(packed, out, x, in) && !overlaps(packed, out, scale, per) &&
                     !overlaps(packed, out, bias, per) && !overlaps(packed, out, stats, 2 * N * groups * sizeof(float)),
                 "dopt_hip_group_norm_grad: the result overlaps an operand");
    DOPT_ENSURE_INIT();
    float *const dx = packed;
    const float *const means = stats, *const rstds = stats + N * G;
    float2 *sums = nullptr;
    const size_t folds = ceil_div(C, (size_t)8);
    auto fold = [&](size_t rows, int pieces) -> int {
        hipLaunchKernelGGL(gn_fold_k, grid_of(folds), dim3(kBlock), 0, stream(), Fold{rows, C, pieces, sums, packed + total, packed + total + C});
        DOPT_LAUNCH_CHECK();
        return DOPT_HIP_OK;
    };
    if (total == 0) return fold(0, 1);
    if (inner == 1 && C / G <= 64 * kRowValues) {
        const size_t tiles = ceil_div(C, (size_t)64);
        const int S = (int)std::min(std::max((size_t)1, (size_t)num_cus() * 4 / tiles), ceil_div(N, (size_t)32));
        if (!(sums = (float2 *)workspace((size_t)S * C * sizeof(float2)))) return DOPT_HIP_ERR_OOM;
        hipLaunchKernelGGL(gn_row_dx_k, grid_of(ceil_div(N * G, (size_t)4)), dim3(kBlock), 0, stream(), N * G, (int)(C / G), (int)G, act, dy,
                           x, scale, bias, means, rstds, dx);
        DOPT_LAUNCH_CHECK();
        hipLaunchKernelGGL(gn_row_sums_k, grid_of(tiles * S), dim3(kBlock), 0, stream(), N, C, (int)(C / G), (int)G, S, act, dy, x, scale,
                           bias, means, rstds, sums);
        DOPT_LAUNCH_CHECK();
        return fold(S, 1);
    }
    const HeldHold held = channels_last && inner > 1 ? held_for(N, C, inner, G, true) : HeldHold{};
    if (held.threads) {
        if (!(sums = (float2 *)workspace(N * C * sizeof(float2)))) return DOPT_HIP_ERR_OOM;
        if (int rc = with_quads<kMostGrad>(held.q, [&](auto q) -> int {
                hipLaunchKernelGGL(gn_held_bwd_k<decltype(q)::value>, grid_of(8 * (size_t)held.h.per), dim3(held.threads), 0, stream(), held.h, act, dy, x,
                                   scale, bias, means, rstds, sums, dx);
                DOPT_LAUNCH_CHECK();
                return DOPT_HIP_OK;
            }))
            return rc;
        return fold(N, 1);
    }
    if (channels_last && inner > 1 && C <= kLastChannels)
        return with_vec(C, [&](auto v) -> int {
            constexpr int V = decltype(v)::value;
            const Rows r = rows_of(N, C, inner, G, V);
            sums = (float2 *)workspace(r.runs * (C + G) * sizeof(float2));
            if (!sums) return DOPT_HIP_ERR_OOM;
            float2 *const gsums = sums + r.runs * C;
            const Fold f{r.runs, C, 1, sums, packed + total, packed + total + C};
            hipLaunchKernelGGL((gn_last_grad_k<V, false>), grid_of(r.runs), dim3(kBlock), r.R * C * sizeof(float2), stream(), r, act, dy, x, scale, bias,
                               means, rstds, sums, gsums, dx, f);
            DOPT_LAUNCH_CHECK();
            hipLaunchKernelGGL((gn_last_grad_k<V, true>), grid_of(r.runs + folds), dim3(kBlock), std::max(G, (size_t)kFoldRed) * sizeof(float2), stream(), r, act, dy, x, scale, bias,
                               means, rstds, sums, gsums, dx, f);
            DOPT_LAUNCH_CHECK();
            return DOPT_HIP_OK;
        });
    if (!channels_last && inner >= 4) {
        const Split k = split_of(N, C, inner, G, kMostGrad);
        if (!(sums = (float2 *)workspace(N * C * k.s.pieces * sizeof(float2)))) return DOPT_HIP_ERR_OOM;
        if (int rc = with_hold<kMostGrad>(k.h, [&](auto c, auto q) -> int {
                constexpr int kC = decltype(c)::value, kQ = decltype(q)::value;
                const dim3 grid = grid_of(k.s.blocks), block(k.h.threads);
                if (k.whole) {
                    hipLaunchKernelGGL((gn_bwd_k<kC, kQ, kWhole>), grid, block, 0, stream(), k.s, act, dy, x, scale, bias, means, rstds, sums, dx);
                } else {
                    hipLaunchKernelGGL((gn_bwd_k<kC, kQ, kFirst>), grid, block, 0, stream(), k.s, act, dy, x, scale, bias, means, rstds, sums, dx);
                    DOPT_LAUNCH_CHECK();
                    hipLaunchKernelGGL((gn_bwd_k<kC, kQ, kSecond>), grid, block, 0, stream(), k.s, act, dy, x, scale, bias, means, rstds, sums, dx);
                }
                DOPT_LAUNCH_CHECK();
                return DOPT_HIP_OK;
            }))
            return rc;
        return fold(N, k.s.pieces);
    }
    const Place p{N, C, inner, C / G, G, channels_last != 0};
    if (!(sums = (float2 *)workspace(N * C * sizeof(float2)))) return DOPT_HIP_ERR_OOM;
    hipLaunchKernelGGL(gn_any_sums_k, grid_of(ceil_div(N * C, (size_t)kBlock)), dim3(kBlock), 0, stream(), p, act, dy, x, scale, bias, means, rstds, sums);
    DOPT_LAUNCH_CHECK();
    hipLaunchKernelGGL(gn_any_dx_k, grid_of(N * G), dim3(kBlock), 0, stream(), p, act, dy, x, scale, bias, means, rstds, sums, dx);
    DOPT_LAUNCH_CHECK();
    return fold(N, 1);
}

}  // extern "C"
