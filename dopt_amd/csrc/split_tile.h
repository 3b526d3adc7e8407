// A tile of a product of fp32 matrices whose operands become two fp16 parts on their way into LDS (half_parts.h): nothing is laid out in front.
//
// The reduction goes by chunks of 32 steps, which the workgroup's teams of four wavefronts take in turn.  Of the rows and columns that a wavefront brings a team
// knows what they are held times, 2^s, from the largest magnitude so far: s falls where a chunk has a value that 2^15 / 2^s does not cover, by one more
// than it must, so that the next one seldom falls again; then the team's sums follow, multiplied by powers of two.  Rows keep 22 bits of a value, or 2^-38
// of their largest one.  NaN goes through the parts; sums of a row with an infinity, whose low part would be NaN, are formed by fp32 instructions behind the
// others.  Sums of 4096 steps are added in one accumulator (dense_wide.h).
#pragma once

#include "dense_wide.h"

namespace dopt {

constexpr int kChunk = 32;                    // steps
constexpr int kUnset = 300;                   // of a row that has been zero so far
constexpr unsigned kPassChunks = (unsigned)kPass * 16 / kChunk;
constexpr int kSplitTile = 64, kSplitHalf = 2 * kSplitTile * kChunk * 4;   // rows and columns; bytes of a chunk of both operands
template <int kTeams>
constexpr int kSplitLds = kTeams * 2 * kSplitHalf;

// An operand: value (row, k) is at x[row * pitch + k], or, across the reduction, at x[k * pitch + row].
struct Matrix32 {
    const float *x;
    size_t pitch;
    unsigned rows;
};

// What a thread has of a chunk of 64 rows of an operand: eight steps of a row.  Along the reduction four lanes that lie 1 and 8 apart have a row, in such
// an order that eight lanes side by side write to all of LDS' banks; across it, four lanes that lie 16 apart, and sixteen lanes side by side have
// neighbouring rows.
template <bool kAcross>
struct Feed {
    const float *at;
    size_t pitch;
    float v[2][8];     // of the next two chunks
    float scale;       // 2^shift
    unsigned limit;    // the first magnitude that is too large for it
    int shift;
    bool odd;          // the row has an infinity
    int row, k8;

    __device__ __forceinline__ void begin(const Matrix32 &m, unsigned row0)
    {
        const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6 & 3;
        if (kAcross) {
            row = (lane & 15) + 16 * wave;
            k8 = lane >> 4;
        } else {
            row = (lane >> 1 & 1) | (lane >> 3 & 2) | (lane & 4) | (lane >> 2 & 8) | 16 * wave;
            k8 = (lane & 1) | (lane >> 2 & 2);
        }
        pitch = m.pitch;
        const unsigned r = min(row0 + row, m.rows - 1);
        at = kAcross ? m.x + r : m.x + r * pitch;
        shift = kUnset;
        scale = 0.0f;
        limit = 0;
        odd = false;
    }
    template <int P>
    __device__ __forceinline__ void load(unsigned k0, unsigned K)
    {
        const unsigned k = k0 + 8 * k8;
        if (k0 + kChunk <= K) {
            if (kAcross) {
                const float *const p = at + k * pitch;
#pragma unroll
                for (int e = 0; e < 8; e++) v[P][e] = p[e * pitch];
            } else {
                *(v4f_any *)v[P] = *(const v4f_any *)(at + k);
                *(v4f_any *)(v[P] + 4) = *(const v4f_any *)(at + k + 4);
            }
            return;
        }
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float t = at[min(k + e, K - 1) * (kAcross ? pitch : 1)];
            v[P][e] = k + e < K ? t : 0.0f;
        }
    }
    // Into LDS, [step][32 rows]; `fell`: by how much a row's shift changes.  True where it does.
    template <int P>
    __device__ __forceinline__ bool put(char *lds, int *fell)
    {
        const float *const f = v[P];
        float most;   // of the magnitudes; NaN may or may not count
        asm("v_max3_f32 %0, |%1|, |%2|, |%3|\n\tv_max3_f32 %0, |%4|, |%5|, %0\n\tv_max3_f32 %0, |%6|, |%7|, %0\n\tv_max_f32 %0, |%8|, %0"
            : "=&v"(most)
            : "v"(f[0]), "v"(f[1]), "v"(f[2]), "v"(f[3]), "v"(f[4]), "v"(f[5]), "v"(f[6]), "v"(f[7]));
        unsigned top = __builtin_bit_cast(unsigned, most);
        auto with = [&](int other) { top = max(top, (unsigned)other); };
        if (kAcross) {
            with(__shfl_xor((int)top, 16, 64));
            with(__shfl_xor((int)top, 32, 64));
        } else {
            with(__builtin_amdgcn_mov_dpp((int)top, 0xB1, 0xf, 0xf, true));    // the neighbour
            with(__builtin_amdgcn_mov_dpp((int)top, 0x128, 0xf, 0xf, true));   // eight lanes on
        }
        int by = 0;
        if (top >= limit) {
            if (top >= 0x7f800000u) {
                odd = true;
            } else if (top) {
                const int to = min(shift_of(top) - 1, 127);
                by = to - shift;
                shift = to;
                scale = __builtin_ldexpf(1.0f, to);
                limit = __builtin_bit_cast(unsigned, __builtin_ldexpf(1.0f, 15 - to));
            }
        }
        v8h h, l;
#pragma unroll
        for (int e = 0; e < 8; e++) h[e] = (_Float16)(f[e] * scale);
        asm("" : "+v"(h));   // (else each value is rounded once more, for l)
#pragma unroll
        for (int e = 0; e < 8; e++) l[e] = (_Float16)__builtin_fmaf(f[e], scale, -(float)h[e]);
        char *const block = lds + ((k8 >> 1) * 2 + (row >> 5)) * 2048;
        *(v8h *)(block + piece_at(row, 2 * (k8 & 1))) = h;
        *(v8h *)(block + piece_at(row, 2 * (k8 & 1) + 1)) = l;
        if (k8 == 0) fell[row] = by;
        return by != 0;
    }
};

// A tile of a result of ep.N columns; at least one step, row and column.  The workgroup's teams share its reduction, or (kShare false) have a tile each, of
// reductions that are as long: one that begins behind the last row or column is none.
template <int kTeams, bool kShare, bool kAcrossA, bool kAcrossB, bool kPasses>
__device__ __forceinline__ void split_tile(const Matrix32 &A, const Matrix32 &B, unsigned K, unsigned m0, unsigned n0, const DenseEpilogue &ep, float *y, char *lds)
{
    constexpr int T = kSplitTile, kOfA = kSplitHalf / 2;
    constexpr int kSharing = kShare ? kTeams : 1, kTiles = kTeams / kSharing;
    __shared__ int fell_of[kTeams][2][2 * T], shifts[kTeams][2 * T], moved_of[kTeams][2][4], odd_of[kTiles][2 * T], any_odd_of[kTiles];
    const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6 & 3, team = (int)threadIdx.x >> 8, wm = wave & 1, wn = wave >> 1;
    int(&fell)[2][2 * T] = fell_of[team], (&moved)[2][4] = moved_of[team];
    char *const of_team = lds + team * 2 * kSplitHalf;
    const int tile = kShare ? 0 : team, shared = kShare ? team : 0, thread = (int)threadIdx.x & (256 * kSharing - 1);   // of the tile
    int(&odd)[2 * T] = odd_of[tile], &any_odd = any_odd_of[tile];
    if (thread < 2 * T) odd[thread] = 0;
    if (thread == 0) any_odd = 0;
    Feed<kAcrossA> a;
    Feed<kAcrossB> b;
    a.begin(A, m0);
    b.begin(B, n0);
    v16f acc[1][1] = {}, all = {};
    const unsigned chunks = (K + kChunk - 1) / kChunk, turns = (chunks + kSharing - 1) / kSharing;
    auto load = [&](unsigned turn, auto parity) {
        const unsigned c = turn * kSharing + shared;
        if (c >= chunks) return;
        a.template load<parity.value>(c * kChunk, K);
        b.template load<parity.value>(c * kChunk, K);
    };
    auto chunk = [&](unsigned turn, auto parity) {
        constexpr int P = decltype(parity)::value;
        const bool live = kSharing == 1 || turn * kSharing + shared < chunks;
        char *const to = of_team + P * kSplitHalf;
        if (live) {
            bool any = a.template put<P>(to, fell[P]);
            any |= b.template put<P>(to + kOfA, fell[P] + T);
            any = __ballot(any) != 0;
            if (lane == 0) moved[P][wave] = any;
            load(turn + 2, parity);
        }
        meet();
        if (!live) return;
        const char *const rows = to + wm * 2048, *const cols = to + kOfA + wn * 2048;
        Side<1> ra, rb;
        ra.read(rows, lane);
        rb.read(cols, lane);
        if (turn && (moved[P][0] | moved[P][1] | moved[P][2] | moved[P][3])) {
            const int of_col = fell[P][T + wn * 32 + (lane & 31)];
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const int d = of_col + fell[P][wm * 32 + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3)];
                acc[0][0][e] = __builtin_ldexpf(acc[0][0][e], d);
                if (kPasses) all[e] = __builtin_ldexpf(all[e], d);
            }
        }
        multiply(ra, rb, acc);
        multiply(rows + 2 * 2048, cols + 2 * 2048, lane, acc);
        if (kPasses && (turn + 1) % kPassChunks == 0) {
            all += acc[0][0];
            acc[0][0] = v16f{};
        }
    };
    constexpr std::integral_constant<int, 0> first{};
    constexpr std::integral_constant<int, 1> second{};
    load(0, first);
    load(1, second);
    for (unsigned turn = 0; turn < turns; turn += 2) {
        chunk(turn, first);
        if (turn + 1 < turns) chunk(turn + 1, second);
    }
    if (kPasses) acc[0][0] += all;
    auto tell = [&](auto &feed, int from) {
        if (feed.k8 == 0) shifts[team][from + feed.row] = feed.shift;
        if (feed.odd) odd[from + feed.row] = any_odd = 1;
    };
    tell(a, 0);
    tell(b, T);
    meet();   // (whoever writes to LDS from here on has seen all of the last chunk)
    const int col = wn * 32 + (lane & 31);
    const unsigned n = n0 + col;
    auto row_of = [&](int e) { return wm * 32 + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3); };
#pragma unroll
    for (int e = 0; e < 16; e++) acc[0][0][e] = __builtin_ldexpf(acc[0][0][e], -(shifts[team][row_of(e)] + shifts[team][T + col]));
    // Teams add up their sums, a quarter or half of the rows each.
    float *const image = (float *)lds + ((int)threadIdx.x & 255);
    if constexpr (kSharing > 1) {
#pragma unroll
        for (int e = 0; e < 16; e++) image[(team * 16 + e) * 256] = acc[0][0][e];
        meet();
    }
    if (n < B.rows && !odd[T + col]) {
        const float bias = ep.bias_of(n);
        with_activation(ep.act, [&](auto kind) {
            // (a loop, whose sums move down: less code to fetch)
#pragma unroll 1
            for (int t = shared * (4 / kSharing); t < (shared + 1) * (4 / kSharing); t++) {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    float z = acc[0][0][e];
                    if constexpr (kSharing > 1) {
                        z = image[(4 * t + e) * 256];
#pragma unroll
                        for (int i = 1; i < kSharing; i++) z += image[(i * 16 + 4 * t + e) * 256];
                    }
                    const int r = row_of(4 * t + e);
                    const unsigned m = m0 + r;
                    if (m >= A.rows || odd[r]) continue;
                    const size_t at = m * ep.N + n;
                    z += bias;
                    if (ep.pre) ep.pre[at] = z;
                    y[at] = act_value<kind.value>(z);
                }
                if constexpr (kSharing == 1) {
#pragma unroll
                    for (int e = 0; e < 12; e++) acc[0][0][e] = acc[0][0][e + 4];
                }
            }
        });
    }
    if (!any_odd) return;
    for (int i = thread; i < T * T; i += 256 * kSharing) {
        const unsigned m = m0 + i / T, n = n0 + i % T;
        if (m >= A.rows || n >= B.rows || !(odd[i / T] | odd[T + i % T])) continue;
        float s = 0.0f;
        for (size_t k = 0; k < K; k++) s += A.x[kAcrossA ? k * A.pitch + m : m * A.pitch + k] * B.x[kAcrossB ? k * B.pitch + n : n * B.pitch + k];
        y[m * ep.N + n] = ep(s, m * ep.N + n);
    }
}

}  // namespace dopt
