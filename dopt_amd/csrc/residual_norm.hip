// What lies between two blocks of a residual network: the norm behind the one, its gate, the sum with the stream, and the norm before the
// other, forward and backward, over rows of `cols` values.  No counterpart in the reference, whose only norm is over the batch
// (cuda/source/dopt/cuda/nnet/cudnn7.d:547-654).
//
//     zb = norm(branch),  u = zb ps + pb,  y = s x + gate u,  zy = norm(y),  h = zy qs + qb
//     norm(v) = (v - mean) rstd with rstd = 1 / sqrt(variance + eps), or v rstd with rstd = 1 / sqrt(mean of v^2 + eps)
//
//     e = dh qs,  t = dy + ry (e - mean(e) - zy mean(e zy)),  dx = s t,  dgate = sum over the gate's rows of t u,  du = t gate
//     f = du ps,  dbranch = rb (f - mean(f) - zb mean(f zb))          (no mean(e), mean(f) where a norm takes no mean out)
//     dqs = sum of dh zy,  dqb = sum of dh,  dps = sum of du zb,  dpb = sum of du over all rows
//
// Bound by memory: 16 bytes a value forward, 24 backward.  A row stays in the registers of the team of lanes that has it: 16, 32 or 64 lanes
// of a wavefront for up to 1024 values (256 backward), whole wavefronts for up to 16384, so everything is read and written once; longer rows are
// read several times by a workgroup.  Means come before squared differences from them, so nothing cancels.  Forward a launch has as many workgroups as
// run at a time, so that scales are loaded once by each.  Backward a workgroup of twelve wavefronts, several teams of them where rows are short, takes a
// run of rows with the scales in LDS and the next rows on their way, and adds up the columns in registers: two sums for the branch's three results,
// since dps, dpb and dgate follow from the sums of t zb and of t over a gate's rows.  A second launch adds the runs.  No atomics: every sum has one order.
//
// [16384 x 1024] forward 53 us (5.0 TB/s), backward 88 and 6 for the runs (4.3); [8192 x 4096] forward 99.6 (5.4); [4107 x 1111] with 37 gates backward
// 29 and 6; one row of 512 3.5, a launch; [256 x 1024] backward 14, [1024 x 256] 11: two launches, and the way of a row through both norms.  Rows of more than 8192 values leave a CU one workgroup, whose reads and writes take turns: [1024 x 16384] 92 forward, 174
// backward (2.9 and 2.3 TB/s); beyond 16384 a fifth of the rate is left ([500 x 20000] 114 and 182).
#include <algorithm>
#include <type_traits>

#include "common.h"
#include "mfma_core.h"

namespace {

using namespace dopt;

constexpr int kBlock = 256;          // of teams within a wavefront
constexpr size_t kHeld = 16384;      // values of a row that a workgroup holds at most
constexpr size_t kWholeRows = 16;    // of a gate
constexpr size_t kTeamRows = 128;    // rows that a team adds up at most: sums of more values that are alike are rounded the same way for long
constexpr size_t kMostRuns = (size_t)1 << 22, kMostColumns = (size_t)1 << 24;   // workgroups of a launch, which has fewer than 2^32 threads

typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v4f_any __attribute__((ext_vector_type(4), aligned(4)));   // sixteen bytes wherever they start

// Between reads and writes of the same LDS by different wavefronts; the empty statement keeps reads in front of it that are used behind
// it in a branch.
__device__ __forceinline__ void meet()
{
    asm volatile("" ::: "memory");
    __syncthreads();
}

template <int kControl>
__device__ __forceinline__ float plus_moved(float v)
{
    return v + __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), kControl, 0xf, 0xf, true));
}

// The sum over groups of kLanes lanes, in all of them.
template <int kLanes>
__device__ __forceinline__ float lanes_sum(float v)
{
    v = plus_moved<0xB1>(v);    // the neighbour
    v = plus_moved<0x4E>(v);    // the other pair
    v = plus_moved<0x141>(v);   // the other quad: each of its lanes holds its sum by now
    v = plus_moved<0x140>(v);   // the other eight
    if (kLanes >= 32) v += __shfl_xor(v, 16, 64);
    if (kLanes >= 64) v += __shfl_xor(v, 32, 64);
    return v;
}

struct Norms {
    unsigned rows;
    int cols;
    unsigned per_gate;   // consecutive rows with one gate; 0: there is none
    int post, pre;
    float eps, scale;
    const float *x, *branch, *gate, *ps, *pb, *qs, *qb;
    float *y, *h;
    float *mb, *rb, *my, *ry;    // the rows' statistics
};
struct Grads {
    Norms n;             // y and branch as the forward pass read and left them; statistics as it left them
    const float *dy, *dh;
    float *dx, *db, *dgate;
    float *sums[4];      // by Kind, a row for each run, null where not wanted: scratch, or the result itself where there is one run
    float *gate_sums;    // likewise of the gate, where its rows are several runs
};
enum Kind { kPreScale, kPreBias, kPostScale, kPostBias, kKinds };

// A workgroup's rows: of a gate's rows one of `splits` runs; or, where kWhole, `gates` whole gates.  Its teams take every teams-th row of
// a run, or every teams-th gate.
struct Runs {
    unsigned count, rows, per_gate, splits, gates;
    __device__ __forceinline__ unsigned gate_of(unsigned run) const { return run / splits; }
    __device__ __forceinline__ void range(unsigned run, unsigned &from, unsigned &to) const
    {
        if (gates) {
            from = (unsigned)min((size_t)rows, (size_t)run * gates * per_gate);
            to = (unsigned)min((size_t)rows, from + (size_t)gates * per_gate);
            return;
        }
        const unsigned first = run / splits * per_gate, part = run % splits;
        from = first + (unsigned)((size_t)per_gate * part / splits);
        to = first + (unsigned)((size_t)per_gate * (part + 1) / splits);
    }
};

// A row's values of one thread: quad lane + i * lanes of the row; values beyond its end are zero.
__device__ __forceinline__ v4f load_quad(const float *row, int col, int cols)
{
    if (col + 4 <= cols) return *(const v4f_any *)(row + col);
    v4f v{0.0f, 0.0f, 0.0f, 0.0f};
    if (col < cols) v.x = row[col];
    if (col + 1 < cols) v.y = row[col + 1];
    if (col + 2 < cols) v.z = row[col + 2];
    return v;
}
__device__ __forceinline__ void store_quad(float *row, int col, int cols, v4f v)
{
    if (col + 4 <= cols) {
        *(v4f_any *)(row + col) = v;
        return;
    }
    if (col < cols) row[col] = v.x;
    if (col + 1 < cols) row[col + 1] = v.y;
    if (col + 2 < cols) row[col + 2] = v.z;
}
__device__ __forceinline__ v4f inside(v4f v, int col, int cols)   // zero beyond the row's end
{
    if (col + 4 > cols) {
        if (col >= cols) v.x = 0.0f;
        if (col + 1 >= cols) v.y = 0.0f;
        if (col + 2 >= cols) v.z = 0.0f;
        v.w = 0.0f;
    }
    return v;
}
__device__ __forceinline__ float sum4(v4f v) { return (v.x + v.y) + (v.z + v.w); }
__device__ __forceinline__ v4f splat(float v) { return v4f{v, v, v, v}; }

// The lanes that share a row: kLanes of a wavefront, or (0) `waves` wavefronts of a workgroup, whose teams then sum together.
template <int kLanes>
struct Team {
    static constexpr bool kWide = kLanes == 0;
    float *red;   // of wide teams: twice 32 values
    int waves;
    int turn = 0;
    __device__ __forceinline__ int lanes() const { return kWide ? 64 * waves : kLanes; }
    __device__ __forceinline__ int index() const { return kWide ? (int)threadIdx.x / lanes() : (int)threadIdx.x / (kLanes ? kLanes : 1); }
    __device__ __forceinline__ int lane() const { return kWide ? (int)threadIdx.x - index() * lanes() : (int)threadIdx.x & (kLanes - 1); }
    __device__ __forceinline__ int teams() const { return (int)blockDim.x / lanes(); }
    __device__ __forceinline__ void sum(float &a, float &b)   // both over the team, in all of its lanes
    {
        a = lanes_sum<kWide ? 64 : kLanes>(a);
        b = lanes_sum<kWide ? 64 : kLanes>(b);
        if (!kWide || waves == 1) return;
        float *const r = red + turn * 32;   // two places in turn: a barrier apiece is enough
        turn ^= 1;
        if ((threadIdx.x & 63) == 0) {
            r[threadIdx.x >> 6] = a;
            r[16 + (threadIdx.x >> 6)] = b;
        }
        meet();
        const int first = index() * waves;
        a = r[first];
        b = r[16 + first];
        for (int i = 1; i < waves; i++) {
            a += r[first + i];
            b += r[16 + first + i];
        }
    }
    __device__ __forceinline__ float sum(float a)
    {
        float none = 0.0f;
        sum(a, none);
        return a;
    }
};

// A row's mean (where the norm takes it out) and rstd.
template <int Q, class T>
__device__ __forceinline__ void row_stats(T &team, const v4f (&v)[Q], int kind, int cols, float eps, float &mean, float &rstd)
{
    mean = 0.0f;
    const float n = (float)cols;
    if (kind == DOPT_HIP_NORM_LAYER) {
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < Q; i++) s += sum4(v[i]);
        mean = team.sum(s) / n;
    }
    float q = 0.0f;
#pragma unroll
    for (int i = 0; i < Q; i++) {
        const v4f d = inside(v[i] - splat(mean), 4 * (team.lane() + i * team.lanes()), cols);
        q += sum4(d * d);
    }
    rstd = 1.0f / sqrtf(team.sum(q) / n + eps);
}

template <int Q>
__device__ __forceinline__ void load_row(const float *p, float missing, int lane, int lanes, int cols, v4f (&v)[Q])
{
#pragma unroll
    for (int i = 0; i < Q; i++) v[i] = p ? load_quad(p, 4 * (lane + i * lanes), cols) : splat(missing);
}

// Rows that belong to whole wavefronts go through a buffer resource of the row's bytes: what lies beyond its end reads as zero and is not
// written, dword by dword (measured), without a branch - with branches one wavefront that stuck out of the row held up all of its
// workgroup ([2048 x 7936] took 69 us, [2048 x 8192] 57).
template <bool kWaves, int Q>
__device__ __forceinline__ void fetch_row(const float *p, int lane, int lanes, int cols, v4f (&v)[Q])   // null: zeros
{
    if constexpr (kWaves) {
        const __amdgpu_buffer_rsrc_t row = make_rsrc(p, p ? (size_t)cols * sizeof(float) : 0);
#pragma unroll
        for (int i = 0; i < Q; i++) v[i] = __builtin_bit_cast(v4f, buffer_load_f32x4(row, 16u * (lane + i * lanes), 0));
    } else {
        load_row(p, 0.0f, lane, lanes, cols, v);
    }
}
template <bool kWaves, int Q>
__device__ __forceinline__ void put_row(float *p, int lane, int lanes, int cols, const v4f (&v)[Q])
{
    if constexpr (kWaves) {
        const __amdgpu_buffer_rsrc_t row = make_rsrc(p, (size_t)cols * sizeof(float));
#pragma unroll
        for (int i = 0; i < Q; i++) __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(v4u, v[i]), row, 16 * (lane + i * lanes), 0, 0);
    } else {
#pragma unroll
        for (int i = 0; i < Q; i++) store_quad(p, 4 * (lane + i * lanes), cols, v[i]);
    }
}
// What is the same in all lanes of a team of whole wavefronts, for the scalar registers.
template <bool kWaves>
__device__ __forceinline__ unsigned alike(unsigned v)
{
    return kWaves ? (unsigned)__builtin_amdgcn_readfirstlane((int)v) : v;
}

template <int kLanes, int Q>
__global__ __launch_bounds__(kLanes ? kBlock : 1024) void join_k(Norms n)
{
    constexpr bool kHeldScales = kLanes || Q < 4;   // in registers; else read from the L2 for each row
    constexpr bool kAhead = !kLanes;                // the next row is on its way while one is worked on
    constexpr bool kWaves = kLanes == 0 || kLanes == 64;
    __shared__ float red[64];
    Team<kLanes> team{red, (int)blockDim.x >> 6};
    const int lane = team.lane(), lanes = team.lanes(), cols = n.cols;
    constexpr int H = kHeldScales ? Q : 1;
    v4f ps[H], pb[H], qs[H], qb[H], gate[Q];
    if constexpr (kHeldScales) {
        load_row(n.ps, 1.0f, lane, lanes, cols, ps);
        load_row(n.pb, 0.0f, lane, lanes, cols, pb);
        load_row(n.qs, 1.0f, lane, lanes, cols, qs);
        load_row(n.qb, 0.0f, lane, lanes, cols, qb);
    }
    auto held = [&](const v4f(&v)[H], const float *p, float missing, int i) {
        if constexpr (kHeldScales) return v[i];
        else return p ? load_quad(p, 4 * (lane + i * lanes), cols) : splat(missing);
    };
    const bool one_gate = kHeldScales && (n.per_gate == 0 || n.per_gate == n.rows);
    if (one_gate) load_row(n.gate, 1.0f, lane, lanes, cols, gate);
    const unsigned step = gridDim.x * team.teams();
    const unsigned first = alike<kWaves>(blockIdx.x * team.teams() + team.index());
    auto fetch = [&](unsigned r, v4f(&x)[Q], v4f(&v)[Q]) {
        const size_t at = r * (size_t)cols;
        fetch_row<kWaves>(n.branch ? n.branch + at : nullptr, lane, lanes, cols, v);
        fetch_row<kWaves>(n.x ? n.x + at : nullptr, lane, lanes, cols, x);
    };
    v4f x[Q], v[Q], x_ahead[Q], v_ahead[Q];
    if (kAhead && first < n.rows) fetch(first, x_ahead, v_ahead);
    for (unsigned r = first; r < n.rows; r += step) {
        const size_t at = r * (size_t)cols;
        if (kAhead) {
#pragma unroll
            for (int i = 0; i < Q; i++) {
                x[i] = x_ahead[i];
                v[i] = v_ahead[i];
            }
            if (r + step < n.rows) fetch(r + step, x_ahead, v_ahead);
        } else {
            fetch(r, x, v);
        }
        if (!one_gate) {
            if (n.gate) fetch_row<kWaves>(n.gate + r / n.per_gate * (size_t)cols, lane, lanes, cols, gate);
            else load_row(nullptr, 1.0f, lane, lanes, cols, gate);
        }
        if (n.post) {
            float mean, rstd;
            row_stats(team, v, n.post, cols, n.eps, mean, rstd);
            if (lane == 0 && n.rb) {
                if (n.mb) n.mb[r] = mean;
                n.rb[r] = rstd;
            }
#pragma unroll
            for (int i = 0; i < Q; i++) v[i] = (v[i] - splat(mean)) * splat(rstd) * held(ps, n.ps, 1.0f, i) + held(pb, n.pb, 0.0f, i);
        }
#pragma unroll
        for (int i = 0; i < Q; i++) {
            const int col = 4 * (lane + i * lanes);
            v[i] = inside(splat(n.scale) * x[i] + gate[i] * v[i], col, cols);
        }
        if (n.y) put_row<kWaves>(n.y + at, lane, lanes, cols, v);
        if (!n.pre) continue;
        float mean, rstd;
        row_stats(team, v, n.pre, cols, n.eps, mean, rstd);
        if (lane == 0 && n.ry) {
            if (n.my) n.my[r] = mean;
            n.ry[r] = rstd;
        }
#pragma unroll
        for (int i = 0; i < Q; i++) v[i] = (v[i] - splat(mean)) * splat(rstd) * held(qs, n.qs, 1.0f, i) + held(qb, n.qb, 0.0f, i);
        put_row<kWaves>(n.h + at, lane, lanes, cols, v);
    }
}

struct RowStats {
    float mb, rb, my, ry;
};
__device__ __forceinline__ RowStats stats_of(const Norms &n, unsigned r)
{
    RowStats s{0.0f, 1.0f, 0.0f, 1.0f};
    if (n.post) {
        s.rb = n.rb[r];
        if (n.mb) s.mb = n.mb[r];
    }
    if (n.pre) {
        s.ry = n.ry[r];
        if (n.my) s.my = n.my[r];
    }
    return s;
}

// Adds what the workgroup's teams hold, in team 0.
template <int Q, class T>
__device__ __forceinline__ void join_teams(const T &team, v4f (&acc)[Q], float *lds, int lane, int lanes)
{
    if (team.teams() == 1) return;
    const int width = 4 * lanes * Q;
    meet();
#pragma unroll
    for (int i = 0; i < Q; i++) *(v4f *)(lds + team.index() * width + 4 * (lane + i * lanes)) = acc[i];
    meet();
    if (team.index()) return;
    for (int t = 1; t < team.teams(); t++)
#pragma unroll
        for (int i = 0; i < Q; i++) acc[i] += *(const v4f *)(lds + t * width + 4 * (lane + i * lanes));
}
template <int Q>
__device__ __forceinline__ void store_row(float *to, int lane, int lanes, int cols, const v4f (&v)[Q])
{
#pragma unroll
    for (int i = 0; i < Q; i++) store_quad(to, 4 * (lane + i * lanes), cols, v[i]);
}

// What a thread has of a row.
template <int Q>
struct Row {
    v4f t[Q], e[Q], y[Q], z[Q];
    RowStats s;
};

// Within a gate's rows the sums of t zb and of t are all that the branch's columns need: dps = gate a, dpb = gate b, dgate = ps a + pb b.
// Scales lie in LDS where they fit (kStaged), for the registers' sake.
template <int kLanes, int Q, bool kWhole, int kThreads>
__global__ __launch_bounds__(kThreads) void join_grad_k(Grads g, Runs runs, int waves)
{
    constexpr bool kStaged = kLanes || Q < 4;
    constexpr bool kAhead = kLanes || kThreads <= 768;   // the next row is on its way while one is worked on
    constexpr bool kWaves = kLanes == 0 || kLanes == 64;
    constexpr bool kSumsInLds = !kLanes && Q == 4;               // those of dh: the registers hold the others
    __shared__ float red[64];
    extern __shared__ __attribute__((aligned(16))) float lds[];
    Team<kLanes> team{red, waves};
    const Norms &n = g.n;
    const int lane = team.lane(), lanes = team.lanes(), cols = n.cols, width = 4 * lanes * Q;
    const float over = 1.0f / (float)cols;
    const unsigned run = blockIdx.x;
    unsigned from, to;
    runs.range(run, from, to);
    const float *gate = n.gate ? n.gate + (kWhole ? 0 : runs.gate_of(run)) * (size_t)cols : nullptr;
    if constexpr (kStaged) {
        for (int c = (int)threadIdx.x; c < width; c += (int)blockDim.x) {
            const bool in = c < cols;
            lds[c] = n.qs && in ? n.qs[c] : 1.0f;
            lds[width + c] = n.ps && in ? n.ps[c] : 1.0f;
            if (!kWhole) lds[2 * width + c] = gate && in ? gate[c] : 1.0f;
        }
        meet();
    }
    auto scale = [&](const float *p, int staged, int col) {
        return kStaged ? *(const v4f *)(lds + staged * width + col) : p ? load_quad(p, col, cols) : splat(1.0f);
    };
    auto gates = [&](int col) { return kWhole ? gate ? load_quad(gate, col, cols) : splat(1.0f) : scale(gate, 2, col); };

    constexpr int S = kSumsInLds ? 1 : Q;
    v4f dqs[S], dqb[S], a[Q], b[Q], dps[kWhole ? Q : 1], dpb[kWhole ? Q : 1];
    v4f *const apart = (v4f *)lds + lane;   // dqs and dqb of the thread, where they are in LDS
#pragma unroll
    for (int i = 0; i < Q; i++) {
        a[i] = b[i] = splat(0.0f);
        if constexpr (kSumsInLds) apart[i * lanes] = apart[(Q + i) * lanes] = splat(0.0f);
        else dqs[i] = dqb[i] = splat(0.0f);
    }
    if (kWhole) {
#pragma unroll
        for (int i = 0; i < Q; i++) dps[i] = dpb[i] = splat(0.0f);
    }
    const int teams = team.teams();
    const unsigned mine = alike<kWaves>(team.index());
    unsigned r = kWhole ? from + mine * runs.per_gate : from + mine;   // (beyond the rows by fewer than 2^16: 32 bits hold it)
    unsigned left = runs.per_gate;   // kWhole: rows of this gate that are left
    const unsigned turns = kWhole ? (runs.gates + teams - 1) / teams * runs.per_gate : (to - from + teams - 1) / teams;
    auto fetch = [&](unsigned row, Row<Q> &v) {   // (a team without a row keeps the others company)
        const bool live = row < to;
        const size_t at = live ? row * (size_t)cols : 0;
        fetch_row<kWaves>(live && g.dy ? g.dy + at : nullptr, lane, lanes, cols, v.t);
        fetch_row<kWaves>(live && n.branch && (n.post || gate) ? n.branch + at : nullptr, lane, lanes, cols, v.z);
        if (n.pre) {
            fetch_row<kWaves>(live ? g.dh + at : nullptr, lane, lanes, cols, v.e);
            fetch_row<kWaves>(live ? n.y + at : nullptr, lane, lanes, cols, v.y);
        }
        v.s = RowStats{0.0f, 1.0f, 0.0f, 1.0f};
        if (live) v.s = stats_of(n, row);
    };
    Row<Q> v, ahead;
    if (kAhead && turns) fetch(r, ahead);
    for (unsigned turn = 0; turn < turns; turn++) {
        const bool live = r < to;
        const size_t at = live ? r * (size_t)cols : 0;
        if (kAhead) {
            v = ahead;
            if (turn + 1 < turns) fetch(!kWhole ? r + teams : left > 1 ? r + 1 : r + 1 + (teams - 1) * runs.per_gate, ahead);
        } else {
            fetch(r, v);
        }
        v4f(&t)[Q] = v.t, (&e)[Q] = v.e, (&y)[Q] = v.y, (&z)[Q] = v.z;
        const RowStats s = v.s;
        if (n.pre) {
            float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
            for (int i = 0; i < Q; i++) {
                y[i] = inside((y[i] - splat(s.my)) * splat(s.ry), 4 * (lane + i * lanes), cols);
                if constexpr (kSumsInLds) {
                    apart[i * lanes] += e[i] * y[i];
                    apart[(Q + i) * lanes] += e[i];
                } else {
                    dqb[i] += e[i];
                    dqs[i] += e[i] * y[i];
                }
                e[i] *= scale(n.qs, 0, 4 * (lane + i * lanes));
                s1 += sum4(e[i]);
                s2 += sum4(e[i] * y[i]);
            }
            team.sum(s1, s2);
            s1 = n.pre == DOPT_HIP_NORM_LAYER ? s1 * over : 0.0f;
            s2 *= over;
#pragma unroll
            for (int i = 0; i < Q; i++) t[i] += splat(s.ry) * (e[i] - splat(s1) - y[i] * splat(s2));
        }
#pragma unroll
        for (int i = 0; i < Q; i++) {
            t[i] = inside(t[i], 4 * (lane + i * lanes), cols);
            e[i] = splat(n.scale) * t[i];
        }
        if (g.dx && live) put_row<kWaves>(g.dx + at, lane, lanes, cols, e);
        if (n.branch) {
            if (kWhole && gate) gate = n.gate + (live ? r / runs.per_gate : 0) * (size_t)cols;
            float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
            for (int i = 0; i < Q; i++) {
                const int col = 4 * (lane + i * lanes);
                z[i] = inside((z[i] - splat(s.mb)) * splat(s.rb), col, cols);
                b[i] += t[i];
                a[i] += t[i] * z[i];
                t[i] *= gates(col) * scale(n.ps, 1, col);
                s1 += sum4(t[i]);
                s2 += sum4(t[i] * z[i]);
            }
            if (n.post) {
                team.sum(s1, s2);
                s1 = n.post == DOPT_HIP_NORM_LAYER ? s1 * over : 0.0f;
                s2 *= over;
#pragma unroll
                for (int i = 0; i < Q; i++) t[i] = splat(s.rb) * (t[i] - splat(s1) - z[i] * splat(s2));
            }
            if (g.db && live) put_row<kWaves>(g.db + at, lane, lanes, cols, t);
        }
        r += kWhole ? 1 : teams;
        if (kWhole && --left == 0) {
            left = runs.per_gate;
#pragma unroll
            for (int i = 0; i < Q && live; i++) {
                const int col = 4 * (lane + i * lanes);
                const v4f g4 = gates(col);
                dps[i] += g4 * a[i];
                dpb[i] += g4 * b[i];
                if (g.dgate)
                    store_quad(g.dgate + (r - 1) / runs.per_gate * (size_t)cols, col, cols,
                               scale(n.ps, 1, col) * a[i] + (n.pb ? load_quad(n.pb, col, cols) * b[i] : splat(0.0f)));
                a[i] = b[i] = splat(0.0f);
            }
            r += (teams - 1) * runs.per_gate;
        }
    }
    const size_t place = run * (size_t)cols;
    auto put = [&](v4f(&v)[S], int in_lds, float *sums) {
        if constexpr (kSumsInLds) {   // (a team by itself)
#pragma unroll
            for (int i = 0; i < Q; i++) store_quad(sums, 4 * (lane + i * lanes), cols, apart[(in_lds + i) * lanes]);
        } else {
            join_teams(team, v, lds + 3 * width, lane, lanes);
            if (mine == 0) store_row(sums, lane, lanes, cols, v);
        }
    };
    if (g.sums[kPreScale]) put(dqs, 0, g.sums[kPreScale] + place);
    if (g.sums[kPreBias]) put(dqb, Q, g.sums[kPreBias] + place);
    const bool of_gate = !kWhole && g.dgate;
    if (!g.sums[kPostScale] && !g.sums[kPostBias] && !of_gate) return;
    if (kWhole) {
#pragma unroll
        for (int i = 0; i < Q; i++) {
            a[i] = dps[i];
            b[i] = dpb[i];
        }
    }
    join_teams(team, a, lds + 3 * width, lane, lanes);
    join_teams(team, b, lds + 3 * width, lane, lanes);
    if (mine) return;
#pragma unroll
    for (int i = 0; i < Q; i++) {
        const int col = 4 * (lane + i * lanes);
        const v4f g4 = kWhole ? splat(1.0f) : gates(col);
        if (g.sums[kPostScale]) store_quad(g.sums[kPostScale] + place, col, cols, g4 * a[i]);
        if (g.sums[kPostBias]) store_quad(g.sums[kPostBias] + place, col, cols, g4 * b[i]);
        if (of_gate)
            store_quad((runs.splits == 1 ? g.dgate : g.gate_sums) + place, col, cols,
                       scale(n.ps, 1, col) * a[i] + (n.pb ? load_quad(n.pb, col, cols) * b[i] : splat(0.0f)));
    }
}

// Rows of more than a workgroup holds, a workgroup each, read again for each of what follows from all of a row.
constexpr int kLong = 1024;
__global__ __launch_bounds__(kLong) void join_long_k(Norms n)
{
    __shared__ float red[64];
    Team<0> team{red, kLong / 64};
    const float count = (float)n.cols;
    auto stats = [&](auto &&value, int kind, float &mean, float &rstd) {
        mean = 0.0f;
        if (kind == DOPT_HIP_NORM_LAYER) {
            float all = 0.0f;
            for (int c = threadIdx.x; c < n.cols; c += 64 * kLong) {   // sums of 64 values each
                float s = 0.0f;
                for (int i = c; i < min(n.cols, c + 64 * kLong); i += kLong) s += value(i);
                all += s;
            }
            mean = team.sum(all) / count;
        }
        float all = 0.0f;
        for (int c = threadIdx.x; c < n.cols; c += 64 * kLong) {
            float s = 0.0f;
            for (int i = c; i < min(n.cols, c + 64 * kLong); i += kLong) {
                const float d = value(i) - mean;
                s += d * d;
            }
            all += s;
        }
        rstd = 1.0f / sqrtf(team.sum(all) / count + n.eps);
    };
    for (unsigned r = blockIdx.x; r < n.rows; r += gridDim.x) {
        const size_t at = r * (size_t)n.cols;
        const float *const gate = n.gate ? n.gate + r / n.per_gate * (size_t)n.cols : nullptr;
        float mb = 0.0f, rb = 1.0f;
        if (n.post) stats([&](int c) { return n.branch[at + c]; }, n.post, mb, rb);
        auto y_of = [&](int c) {
            float v = n.branch ? n.branch[at + c] : 0.0f;
            if (n.post) v = (v - mb) * rb * (n.ps ? n.ps[c] : 1.0f) + (n.pb ? n.pb[c] : 0.0f);
            return n.scale * (n.x ? n.x[at + c] : 0.0f) + (gate ? gate[c] : 1.0f) * v;
        };
        float my = 0.0f, ry = 1.0f;
        if (n.pre) stats(y_of, n.pre, my, ry);
        for (int c = threadIdx.x; c < n.cols; c += kLong) {   // (y or h may lie where x or the branch does)
            const float v = y_of(c);
            if (n.y) n.y[at + c] = v;
            if (n.pre) n.h[at + c] = (v - my) * ry * (n.qs ? n.qs[c] : 1.0f) + (n.qb ? n.qb[c] : 0.0f);
        }
        if (threadIdx.x == 0) {
            if (n.post && n.rb) {
                if (n.mb) n.mb[r] = mb;
                n.rb[r] = rb;
            }
            if (n.pre && n.ry) {
                if (n.my) n.my[r] = my;
                n.ry[r] = ry;
            }
        }
    }
}

// ... and their gradients: dx and dbranch, and the rows' four means, for the columns' sums behind it.
struct Means {
    float e, ez, f, fz;
};
__device__ __forceinline__ float stream_grad(const Grads &g, const RowStats &s, const Means &m, size_t i, int c, float &zy)
{
    const Norms &n = g.n;
    const float t = g.dy ? g.dy[i] : 0.0f;
    if (!n.pre) return t;
    zy = (n.y[i] - s.my) * s.ry;
    return t + s.ry * (g.dh[i] * (n.qs ? n.qs[c] : 1.0f) - m.e - zy * m.ez);
}
__global__ __launch_bounds__(kLong) void join_grad_long_k(Grads g, Means *means)
{
    __shared__ float red[64];
    Team<0> team{red, kLong / 64};
    const Norms &n = g.n;
    const float over = 1.0f / (float)n.cols;
    for (unsigned r = blockIdx.x; r < n.rows; r += gridDim.x) {
        const size_t at = r * (size_t)n.cols;
        const float *const gate = n.gate ? n.gate + r / n.per_gate * (size_t)n.cols : nullptr;
        const RowStats s = stats_of(n, r);
        Means m{0.0f, 0.0f, 0.0f, 0.0f};
        auto both = [&](auto &&values, float &a, float &b) {   // sums of 64 values each
            float all_a = 0.0f, all_b = 0.0f;
            for (int c = threadIdx.x; c < n.cols; c += 64 * kLong) {
                float sa = 0.0f, sb = 0.0f;
                for (int i = c; i < min(n.cols, c + 64 * kLong); i += kLong) values(i, sa, sb);
                all_a += sa;
                all_b += sb;
            }
            team.sum(all_a, all_b);
            a = all_a * over;
            b = all_b * over;
        };
        if (n.pre) {
            both(
                [&](int c, float &a, float &b) {
                    const float e = g.dh[at + c] * (n.qs ? n.qs[c] : 1.0f);
                    a += e;
                    b += e * ((n.y[at + c] - s.my) * s.ry);
                },
                m.e, m.ez);
            if (n.pre != DOPT_HIP_NORM_LAYER) m.e = 0.0f;
        }
        float zy;
        auto f_of = [&](int c) {
            return stream_grad(g, s, m, at + c, c, zy) * (gate ? gate[c] : 1.0f) * (n.post && n.ps ? n.ps[c] : 1.0f);
        };
        if (n.branch && n.post) {
            both(
                [&](int c, float &a, float &b) {
                    const float f = f_of(c);
                    a += f;
                    b += f * ((n.branch[at + c] - s.mb) * s.rb);
                },
                m.f, m.fz);
            if (n.post != DOPT_HIP_NORM_LAYER) m.f = 0.0f;
        }
        for (int c = threadIdx.x; c < n.cols; c += kLong) {
            if (g.dx) g.dx[at + c] = n.scale * stream_grad(g, s, m, at + c, c, zy);
            if (g.db) {
                const float f = f_of(c);
                g.db[at + c] = n.post ? s.rb * (f - m.f - (n.branch[at + c] - s.mb) * s.rb * m.fz) : f;
            }
        }
        if (threadIdx.x == 0) means[r] = m;
    }
}
// A thread's column over a run of rows.
__global__ __launch_bounds__(kBlock) void join_columns_k(Grads g, Runs runs, const Means *means)
{
    const Norms &n = g.n;
    const size_t tiles = ((size_t)n.cols + kBlock - 1) / kBlock, run = blockIdx.x / (unsigned)tiles;
    const int c = (int)(blockIdx.x % (unsigned)tiles) * kBlock + (int)threadIdx.x;
    if (c >= n.cols || run >= runs.count) return;
    unsigned from, to;
    runs.range((unsigned)run, from, to);
    float acc[kKinds] = {0.0f, 0.0f, 0.0f, 0.0f}, sum_gate = 0.0f;
    for (unsigned r = from; r < to; r++) {
        const size_t i = r * (size_t)n.cols + c;
        const RowStats s = stats_of(n, r);
        float zy = 0.0f;
        const float t = stream_grad(g, s, means[r], i, c, zy);
        if (n.pre) {
            acc[kPreBias] += g.dh[i];
            acc[kPreScale] += g.dh[i] * zy;
        }
        if (!n.branch) continue;
        const float zb = (n.branch[i] - s.mb) * s.rb;
        sum_gate += t * (zb * (n.ps ? n.ps[c] : 1.0f) + (n.pb ? n.pb[c] : 0.0f));
        const float du = n.gate ? t * n.gate[r / n.per_gate * (size_t)n.cols + c] : t;
        acc[kPostBias] += du;
        acc[kPostScale] += du * zb;
        if (n.gate && runs.gates && g.dgate && (r + 1) % n.per_gate == 0) {
            g.dgate[r / n.per_gate * (size_t)n.cols + c] = sum_gate;
            sum_gate = 0.0f;
        }
    }
    const size_t place = run * (size_t)n.cols + c;
    for (int k = 0; k < kKinds; k++)
        if (g.sums[k]) g.sums[k][place] = acc[k];
    if (n.gate && g.dgate && !runs.gates) (runs.splits == 1 ? g.dgate : g.gate_sums)[place] = sum_gate;
}

// Adds the runs: 32 columns of one result's row by 32 lanes, or of four rows by eight lanes each where there are few runs.
struct Fold {
    struct One {
        const float *from;
        float *to;
        size_t runs, rows;   // of a row of the result; of the result
        int at_once;         // rows of a workgroup
        size_t blocks;       // for 32 columns
    } one[kKinds + 1];
    int n, cols;
    size_t tiles;
};
__global__ __launch_bounds__(1024) void join_fold_k(Fold f)
{
    __shared__ float red[32][33];
    size_t block = blockIdx.x / f.tiles;
    int k = 0;
    while (k + 1 < f.n && block >= f.one[k].blocks) block -= f.one[k++].blocks;
    const Fold::One &o = f.one[k];
    const int lanes = 32 / o.at_once, group = (int)threadIdx.x >> 5, lane = group % lanes;
    const int c = (int)(blockIdx.x % f.tiles) * 32 + (int)(threadIdx.x & 31);
    const size_t row = block * o.at_once + group / lanes;
    const bool in = c < f.cols && row < o.rows;
    float all = 0.0f;
    if (in) {
        const float *const from = o.from + row * o.runs * f.cols + c;
        for (size_t i0 = lane; i0 < o.runs; i0 += 64 * lanes) {   // sums of 64 values each
            float s = 0.0f;
            const size_t end = min(o.runs, i0 + 64 * lanes);
#pragma unroll 8
            for (size_t i = i0; i < end; i += lanes) s += from[i * f.cols];
            all += s;
        }
    }
    red[group][threadIdx.x & 31] = all;
    __syncthreads();
    if (lane || !in) return;
    for (int i = 1; i < lanes; i++) all += red[group + i][threadIdx.x & 31];
    o.to[row * f.cols + c] = all;
}

// Which kernel holds a row: lanes of a wavefront (0: a workgroup) and quads of a lane.
struct Form {
    int lanes, quads;
    unsigned threads;
};
Form form_of(size_t cols, bool back)
{
    const size_t quads = ceil_div(cols, (size_t)4);
    if (quads <= 16) return Form{16, 1, kBlock};
    if (quads <= 32) return Form{32, 1, kBlock};
    if (quads <= 64) return Form{64, 1, kBlock};
    if (quads <= 128 && !back) return Form{64, 2, kBlock};
    if (quads <= 256 && !back) return Form{64, 4, kBlock};   // (of the gradient four quads leave registers for two wavefronts of a SIMD: 105 us for 94)
    // wavefronts in numbers that a CU's four SIMDs share evenly, by themselves or with the teams that a workgroup has of them
    if (quads <= 2048) {
        const unsigned waves = (unsigned)ceil_div(quads, (size_t)128);
        return Form{0, 2, 64 * (waves <= 4 ? waves : waves <= 6 ? 6 : waves <= 8 ? 8 : waves <= 12 ? 12 : 16)};
    }
    return Form{0, 4, quads <= 256 * 12 ? 768u : 1024u};
}
template <bool kBack, class F>
void with_form(const Form &f, F &&call)
{
    auto c = [](auto v) { return v; };
    if (f.lanes == 16) call(c(std::integral_constant<int, 16>{}), c(std::integral_constant<int, 1>{}));
    else if (f.lanes == 32) call(c(std::integral_constant<int, 32>{}), c(std::integral_constant<int, 1>{}));
    else if (f.lanes == 64 && f.quads == 1) call(c(std::integral_constant<int, 64>{}), c(std::integral_constant<int, 1>{}));
    else if (f.lanes == 64) {
        if constexpr (!kBack) {
            if (f.quads == 2) call(c(std::integral_constant<int, 64>{}), c(std::integral_constant<int, 2>{}));
            else call(c(std::integral_constant<int, 64>{}), c(std::integral_constant<int, 4>{}));
        }
    } else if (f.quads == 2) call(c(std::integral_constant<int, 0>{}), c(std::integral_constant<int, 2>{}));
    else call(c(std::integral_constant<int, 0>{}), c(std::integral_constant<int, 4>{}));
}

// How many workgroups of a kernel the chip holds at a time.  The runtime is asked once for each kernel and number of wavefronts, without the LDS that a
// call adds: what that leaves room for is worked out, so that the answer never depends on the calls before.
struct Places {
    int of_cu[17];
    size_t fixed[17];   // bytes of LDS of every launch
};
size_t places_of(Places &known, const void *kernel, unsigned threads, size_t lds)
{
    int &of_cu = known.of_cu[threads / 64];
    size_t &fixed = known.fixed[threads / 64];
    if (!of_cu) {
        hipFuncAttributes a;
        int n = 0;
        if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, (int)threads, 0) != hipSuccess || hipFuncGetAttributes(&a, kernel) != hipSuccess) {
            (void)hipGetLastError();
            n = 1;
            a.sharedSizeBytes = 0;
        }
        fixed = a.sharedSizeBytes;
        of_cu = std::max(1, n);
    }
    const size_t room = (size_t)160 * 1024 / std::max<size_t>(1, fixed + lds);
    return (size_t)num_cus() * std::max<size_t>(1, std::min((size_t)of_cu, room));
}

struct Launch {
    const void *kernel;
    unsigned threads;
    size_t lds, places;
};
template <int kLanes, int Q, bool kWhole, int kThreads>
int grad_launch(unsigned threads, size_t lds, Launch *l)
{
    const auto kernel = join_grad_k<kLanes, Q, kWhole, kThreads>;
    static bool raised = false;
    if (!raised && lds > 65536 - 1024) {
        DOPT_HIP_CHECK(hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, 159 * 1024));
        raised = true;
    }
    static Places known{};
    *l = Launch{(const void *)kernel, threads, lds, places_of(known, (const void *)kernel, threads, lds)};
    return DOPT_HIP_OK;
}

bool known_norm(int kind) { return kind >= DOPT_HIP_NORM_NONE && kind <= DOPT_HIP_NORM_RMS; }

int check(const char *who, const dopt_hip_residual_norm_desc *d, bool branch, const float *gate, const float *ps, const float *pb, const float *qs,
          const float *qb)
{
    DOPT_REQUIRE(d != nullptr, "%s: null argument", who);
    DOPT_REQUIRE(known_norm(d->post) && known_norm(d->pre), "%s: there is no norm %d", who, known_norm(d->post) ? d->pre : d->post);
    DOPT_REQUIRE(d->rows < (size_t)1 << 31 && d->cols < (size_t)1 << 30 && d->rows * d->cols < (size_t)1 << 40, "%s: dimensions too large", who);
    DOPT_REQUIRE(d->gates <= d->rows && (d->gates == 0 || d->rows % d->gates == 0), "%s: %zu rows do not share %zu gates evenly", who, d->rows, d->gates);
    DOPT_REQUIRE((d->gates == 0) == (gate == nullptr) || d->rows == 0, "%s: %zu gates, and %s", who, d->gates, gate ? "an operand for them" : "no operand");
    DOPT_REQUIRE(d->eps >= 0.0f, "%s: eps is %g", who, (double)d->eps);
    DOPT_REQUIRE(d->post || (!ps && !pb), "%s: a scale or bias of a norm that is not there", who);
    DOPT_REQUIRE(d->pre || (!qs && !qb), "%s: a scale or bias of a norm that is not there", who);
    DOPT_REQUIRE(branch || d->rows == 0 || (!d->post && !d->gates), "%s: a norm or gate of a branch that is not there", who);
    return DOPT_HIP_OK;
}

size_t stats_of_norm(int kind) { return kind == DOPT_HIP_NORM_LAYER ? 2 : kind == DOPT_HIP_NORM_RMS ? 1 : 0; }

void place_stats(const dopt_hip_residual_norm_desc *d, float *stats, Norms *n)
{
    if (!stats) return;
    if (d->post == DOPT_HIP_NORM_LAYER) n->mb = stats, stats += d->rows;
    if (d->post) n->rb = stats, stats += d->rows;
    if (d->pre == DOPT_HIP_NORM_LAYER) n->my = stats, stats += d->rows;
    if (d->pre) n->ry = stats;
}

struct Span {
    const void *p;
    size_t bytes;
};

}  // namespace

extern "C" {

int dopt_hip_residual_norm(const dopt_hip_residual_norm_desc *d, const float *x, const float *branch, const float *gate, const float *post_scale,
                           const float *post_bias, const float *pre_scale, const float *pre_bias, float *y, float *h, float *stats)
{
    const char *const who = "dopt_hip_residual_norm";
    if (int rc = check(who, d, branch != nullptr, gate, post_scale, post_bias, pre_scale, pre_bias)) return rc;
    if (d->rows * d->cols == 0) return DOPT_HIP_OK;
    DOPT_REQUIRE(x || branch, "%s: neither a stream nor a branch", who);
    DOPT_REQUIRE((d->pre == 0) == (h == nullptr), "%s: h and the norm that gives it belong together", who);
    DOPT_REQUIRE(y || h, "%s: no result", who);
    const size_t f = sizeof(float), all = d->rows * d->cols * f, row = d->cols * f;
    const Span in[] = {{x, all}, {branch, all}, {gate, d->gates * row}, {post_scale, row}, {post_bias, row}, {pre_scale, row}, {pre_bias, row}};
    const size_t stats_bytes = (stats_of_norm(d->post) + stats_of_norm(d->pre)) * d->rows * f;
    const Span out[] = {{y, all}, {h, all}, {stats, stats_bytes}};
    for (int i = 0; i < 3; i++) {
        for (int k = 0; k < 7; k++)   // (a value of y or h is written by the thread that has read its operands, behind all of the row)
            DOPT_REQUIRE(!overlaps(out[i].p, out[i].bytes, in[k].p, in[k].bytes) || (i < 2 && k < 2 && out[i].p == in[k].p),
                         "%s: a result overlaps an operand", who);
        for (int k = 0; k < i; k++) DOPT_REQUIRE(!overlaps(out[i].p, out[i].bytes, out[k].p, out[k].bytes), "%s: two results overlap", who);
    }
    DOPT_ENSURE_INIT();
    Norms n{};
    n.rows = (unsigned)d->rows;
    n.cols = (int)d->cols;
    n.per_gate = d->gates ? (unsigned)(d->rows / d->gates) : 0;
    n.post = d->post;
    n.pre = d->pre;
    n.eps = d->eps;
    n.scale = d->residual_scale;
    n.x = x;
    n.branch = branch;
    n.gate = gate;
    n.ps = post_scale;
    n.pb = post_bias;
    n.qs = pre_scale;
    n.qb = pre_bias;
    n.y = y;
    n.h = h;
    place_stats(d, stats, &n);
    if (d->cols > kHeld) {
        hipLaunchKernelGGL(join_long_k, dim3((unsigned)std::min(d->rows, (size_t)num_cus() * 8)), dim3(kLong), 0, stream(), n);
    } else {
        const Form form = form_of(d->cols, false);
        const size_t blocks = form.lanes ? ceil_div(d->rows, (size_t)(kBlock / form.lanes)) : d->rows;
        with_form<false>(form, [&](auto lanes, auto quads) {
            const auto kernel = join_k<lanes.value, quads.value>;
            // every workgroup loads the scales once: no more of them than run at a time, and as many rows for each
            static Places known{};
            const size_t rounds = ceil_div(blocks, places_of(known, (const void *)kernel, form.threads, 0));
            hipLaunchKernelGGL(kernel, dim3((unsigned)ceil_div(blocks, rounds)), dim3(form.threads), 0, stream(), n);
        });
    }
    DOPT_LAUNCH_CHECK();
    return DOPT_HIP_OK;
}

int dopt_hip_residual_norm_grad(const dopt_hip_residual_norm_desc *d, const float *dy, const float *dh, const float *y, const float *branch,
                                const float *gate, const float *post_scale, const float *post_bias, const float *pre_scale, const float *stats,
                                float *dx, float *dbranch, float *dgate, float *dpost_scale, float *dpost_bias, float *dpre_scale, float *dpre_bias)
{
    const char *const who = "dopt_hip_residual_norm_grad";
    if (int rc = check(who, d, branch != nullptr, gate, post_scale, post_bias, pre_scale, nullptr)) return rc;
    if (d->cols == 0) return DOPT_HIP_OK;
    const size_t f = sizeof(float), all = d->rows * d->cols * f, row = d->cols * f;
    const size_t stats_bytes = (stats_of_norm(d->post) + stats_of_norm(d->pre)) * d->rows * f;
    DOPT_REQUIRE(d->rows == 0 || (d->pre ? dh && y : dy && !dh), "%s: the gradient of h and y where there is a norm of y, and that of y elsewhere", who);
    DOPT_REQUIRE(d->rows == 0 || stats || !(d->post || d->pre), "%s: the statistics are missing", who);
    DOPT_REQUIRE(branch || d->rows == 0 || !dbranch, "%s: the gradient of a branch that is not there", who);
    DOPT_REQUIRE(d->gates || !dgate, "%s: the gradient of a gate that is not there", who);
    DOPT_REQUIRE(d->post || (!dpost_scale && !dpost_bias), "%s: the gradient of a norm that is not there", who);
    DOPT_REQUIRE(d->pre || (!dpre_scale && !dpre_bias), "%s: the gradient of a norm that is not there", who);
    const Span in[] = {{dy, all}, {dh, all}, {y, all}, {branch, all}, {gate, d->gates * row}, {post_scale, row}, {post_bias, row}, {pre_scale, row},
                       {stats, stats_bytes}};
    const Span out[] = {{dx, all}, {dbranch, all}, {dgate, d->gates * row}, {dpost_scale, row}, {dpost_bias, row}, {dpre_scale, row}, {dpre_bias, row}};
    for (int i = 0; i < 7; i++) {
        for (const Span &s : in) DOPT_REQUIRE(!overlaps(out[i].p, out[i].bytes, s.p, s.bytes), "%s: a result overlaps an operand", who);
        for (int k = 0; k < i; k++) DOPT_REQUIRE(!overlaps(out[i].p, out[i].bytes, out[k].p, out[k].bytes), "%s: two results overlap", who);
    }
    DOPT_ENSURE_INIT();
    Grads g{};
    Norms &n = g.n;
    n.rows = (unsigned)d->rows;
    n.cols = (int)d->cols;
    n.per_gate = d->gates ? (unsigned)(d->rows / d->gates) : 0;
    n.post = d->post;
    n.pre = d->pre;
    n.scale = d->residual_scale;
    n.branch = branch;
    n.gate = gate;
    n.ps = post_scale;
    n.pb = post_bias;
    n.qs = pre_scale;
    n.y = const_cast<float *>(y);
    place_stats(d, const_cast<float *>(stats), &n);
    g.dy = dy;
    g.dh = dh;
    g.dx = dx;
    g.db = dbranch;
    g.dgate = dgate;
    float *const results[kKinds] = {dpre_scale, dpre_bias, dpost_scale, dpost_bias};
    size_t kinds = 0;
    for (const float *r : results) kinds += r != nullptr;

    const bool held = d->cols <= kHeld;
    const Form form = form_of(std::min(d->cols, kHeld), true);
    // Teams of a workgroup: of two wavefronts two, of three four, of six two, so that the SIMDs share them evenly.
    const int waves = (int)form.threads / 64;
    const size_t teams = !held ? 1 : form.lanes ? (size_t)(768 / form.lanes) : waves > 12 ? 1 : 12 / waves;
    const unsigned threads = form.lanes ? 768 : form.threads * (unsigned)teams;
    const size_t width = 4 * (form.lanes ? (size_t)form.lanes : (size_t)form.threads) * form.quads;
    const bool staged = form.lanes || form.quads < 4;
    const size_t lds = (staged ? 3 + (teams > 1 ? teams : 0) : 2) * width * f;   // scales and what teams add, or sums
    Runs runs{0, (unsigned)d->rows, n.per_gate ? n.per_gate : (unsigned)std::max(d->rows, (size_t)1), 1, 0};
    Launch launch{nullptr, kBlock, 0, (size_t)num_cus() * 8};
    // Gates of few rows go to teams as a whole where there are many of them, else to a workgroup each, whose teams share the rows: [1500 x 600]
    // with 100 gates 19.6 us (as a whole 64), [2400 x 1500] with 200 33 (70), [2000 x 700] with 500 28 (27), [8000 x 600] with 1000 71 (51), with 4000 180 (50).
    // So do the gates of any number of rows where a launch has no workgroups for each (a team then adds up a whole gate, of at most 511 rows).
    const size_t column_tiles = ceil_div(d->cols, (size_t)kBlock);
    const bool whole = (runs.per_gate < std::min(kWholeRows, 4 * teams) && d->gates > 2 * (size_t)num_cus()) ||
                       (held ? d->gates >= kMostRuns : d->gates * column_tiles >= kMostColumns);
    if (held) {
        int rc = DOPT_HIP_OK;
        with_form<true>(form, [&](auto lanes, auto quads) {
            auto with = [&](auto most) {
                rc = whole ? grad_launch<lanes.value, quads.value, true, most.value>(threads, lds, &launch)
                           : grad_launch<lanes.value, quads.value, false, most.value>(threads, lds, &launch);
            };
            if constexpr (lanes.value) with(std::integral_constant<int, 768>{});
            else if (threads <= 768 && quads.value == 2) with(std::integral_constant<int, quads.value == 2 ? 768 : 1024>{});
            else with(std::integral_constant<int, 1024>{});
        });
        if (rc) return rc;
    }
    if (d->rows) {
        const size_t gates = std::max(d->gates, (size_t)1);
        if (whole) {
            const size_t most = std::max((size_t)1, kTeamRows / runs.per_gate);   // gates of a team
            runs.gates = (unsigned)(std::min(most, ceil_div(gates, launch.places * teams)) * teams);
            runs.count = (unsigned)ceil_div(gates, (size_t)runs.gates);
        } else {
            // One to three rounds of all places, whichever leaves the fewest turns of a team; a workgroup's beginning and end cost some two of them.  Down to one
            // row for a team: [1024 x 256] 11.2 us, with six rows 18, [256 x 1024] 14.2 and, with two, 16.8.  Long rows' columns eight at least: [500 x 20000]
            // 182, with one 251.
            const size_t least = ceil_div((size_t)runs.per_gate, kTeamRows * teams);
            const size_t most = ceil_div((size_t)runs.per_gate, held ? teams : (size_t)8);
            size_t best = 0;
            for (size_t rounds = 0; rounds <= 3; rounds++) {   // (none: a run for each gate)
                size_t splits = std::max(least, std::min(most, std::max((size_t)1, rounds * launch.places / gates)));
                const size_t of_team = ceil_div(ceil_div((size_t)runs.per_gate, splits), teams);
                splits = std::max(least, ceil_div((size_t)runs.per_gate, of_team * teams));   // no more of them than so many rows need
                const size_t turns = ceil_div(gates * splits, launch.places) * (of_team + 2) + (gates * splits > 1 ? 4 : 0);   // (the runs' sums are a launch)
                if (best && turns >= best) continue;
                best = turns;
                runs.splits = (unsigned)splits;
            }
            runs.count = (unsigned)std::min(gates * runs.splits, (size_t)1 << 31);
        }
    }
    const size_t blocks = runs.count;
    DOPT_REQUIRE(blocks < kMostRuns, "%s: dimensions too large", who);
    const bool gate_sums = dgate && !runs.gates && (runs.splits > 1 || d->rows == 0);
    const size_t to_add = blocks == 1 ? 0 : kinds;   // (one run's sums are the results)
    const size_t sums = (to_add + gate_sums) * blocks * row, means = held ? 0 : ceil_div(d->rows * sizeof(Means), (size_t)256) * 256;
    char *const scratch = sums + means ? (char *)workspace(sums + means) : nullptr;
    if (sums + means && !scratch) return DOPT_HIP_ERR_OOM;
    float *at = (float *)(scratch + means);
    for (int k = 0; k < kKinds; k++) {
        g.sums[k] = results[k];
        if (!results[k] || !to_add) continue;
        g.sums[k] = at;
        at += blocks * d->cols;
    }
    g.gate_sums = at;
    if (d->rows && held) {
        int of_team = waves;
        void *arguments[] = {&g, &runs, &of_team};
        DOPT_HIP_CHECK(hipLaunchKernel(launch.kernel, dim3((unsigned)blocks), dim3(launch.threads), arguments, launch.lds, stream()));
    } else if (d->rows) {
        hipLaunchKernelGGL(join_grad_long_k, dim3((unsigned)std::min(d->rows, (size_t)num_cus() * 8)), dim3(kLong), 0, stream(), g, (Means *)scratch);
        DOPT_REQUIRE(column_tiles * runs.count < kMostColumns, "%s: dimensions too large", who);
        if (kinds || dgate) hipLaunchKernelGGL(join_columns_k, dim3((unsigned)(column_tiles * runs.count)), dim3(kBlock), 0, stream(), g, runs, (const Means *)scratch);
        DOPT_LAUNCH_CHECK();
    }
    Fold fold{};
    fold.cols = (int)d->cols;
    fold.tiles = ceil_div(d->cols, (size_t)32);
    size_t fold_blocks = 0;
    auto add = [&](const float *from, float *to, size_t count, size_t rows) {
        const int at_once = rows > 1 && count <= 64 ? 4 : 1;
        const size_t of_it = ceil_div(rows, (size_t)at_once);
        fold.one[fold.n++] = Fold::One{from, to, count, rows, at_once, of_it};
        fold_blocks += of_it;
    };
    for (int k = 0; k < kKinds; k++)
        if (results[k] && to_add) add(g.sums[k], results[k], blocks, 1);
    if (gate_sums && d->gates) add(g.gate_sums, dgate, d->rows ? runs.splits : 0, d->gates);
    if (!fold_blocks) return DOPT_HIP_OK;
    DOPT_REQUIRE(fold_blocks * fold.tiles < (size_t)1 << 22, "%s: dimensions too large", who);
    hipLaunchKernelGGL(join_fold_k, dim3((unsigned)(fold_blocks * fold.tiles)), dim3(1024), 0, stream(), fold);
    DOPT_LAUNCH_CHECK();
    return DOPT_HIP_OK;
}

}  // extern "C"
