// Groups of consecutive rows, given by where they begin: offsets[0 .. G] on the device, a group g from offsets[g] up to offsets[g + 1].
// Whatever the values are, a kernel sees boundaries that lie within the rows and do not fall: each is taken as the largest up to it, and
// as M beyond that.  Rows in front of the first group and behind the last one belong to none.
#pragma once

#include <initializer_list>

#include "common.h"

namespace dopt {

// Units of 2^shift rows: of the groups alone, or of the rows of no group as well (rest); at least one for each (all).  See search_segments.
struct Units {
    int shift;
    bool rest, all;
    __host__ __device__ constexpr int key() const { return shift | rest << 5 | all << 6; }
};
// What lies in front of a piece of 64 segments: units, and the row where the last segment ends.
struct Front {
    unsigned units, bound;
};
constexpr int kMostFronts = 5;   // kinds of units that one call's kernels search for
constexpr size_t kNoFronts = 256;   // groups that are searched from the first one on

struct Groups {
    const int *offsets;   // (null without groups)
    unsigned G, M;
    // Where a search may begin, [kind][piece], for many groups: every workgroup searches, and going through all pieces in front takes the square of their
    // number ([64 x 64] from 64 in 4096 groups 564 us and with fronts 26, [4096 x 128] from 128 in 512 and 256 groups 17.1 and 14.0 and with them 17.2 and 13.0).
    // Null for few.
    const Front *fronts;
    unsigned pieces;
    int keys[kMostFronts];
    __device__ __forceinline__ const Front *front_of(int key) const
    {
        if (__builtin_expect(!fronts, 1)) return nullptr;
        for (int i = 0; i < kMostFronts; i++)
            if (keys[i] == key) return fronts + (size_t)i * pieces;
        return nullptr;
    }
};

// Some rows of one group, or of none.
struct Segment {
    int group;             // G: rows of no group, -1: there is no such unit
    unsigned begin, end;   // rows
    unsigned first;        // units of the segments in front of it
    unsigned unit;         // which of its own it is
};

// The inclusive scan of a wavefront.
template <class F>
__device__ __forceinline__ unsigned wave_scan(unsigned v, F &&join)
{
    const int lane = (int)threadIdx.x & 63;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const unsigned up = (unsigned)__shfl_up((int)v, d, 64);
        if (lane >= d) v = join(v, up);
    }
    return v;
}

// Segments in the order of the rows: rows of no group, the groups, rows of no group (rest), or the groups alone.
__host__ __device__ inline unsigned segments_of(const Groups &q, bool rest) { return rest ? q.G + 2 : q.G; }
__device__ __forceinline__ unsigned row_at(const Groups &q, unsigned i) { return (unsigned)min(max(q.offsets[i], 0), (int)q.M); }
// Where the first segment begins, and where segment s ends unless one in front of it ends behind that.
__device__ __forceinline__ unsigned first_row(const Groups &q, bool rest) { return !rest && q.G ? row_at(q, 0) : 0; }
__device__ __forceinline__ unsigned end_of(const Groups &q, bool rest, unsigned s)
{
    const unsigned at = rest ? s : s + 1;
    return at <= q.G && s < segments_of(q, rest) && q.offsets ? row_at(q, at) : q.M;
}
__device__ __forceinline__ unsigned units_of(unsigned begin, unsigned end, int shift, bool all)
{
    const unsigned n = (unsigned)(((size_t)end - begin + ((size_t)1 << shift) - 1) >> shift);
    return all && n == 0 ? 1 : n;
}

// A segment of r rows is ceil(r / 2^shift) units, or one where it is empty and kAll.  `stop(units in front, units up to and with the segment, segment)` says in
// which of them the search ends; every wavefront does it for itself, 64 segments at a time, from the piece on that `choose(fronts, pieces)` names where there
// are fronts, else from the first one on.
template <bool kRest, bool kAll, class C, class F>
__device__ __forceinline__ Segment search_segments(const Groups &q, int shift, unsigned &total, C &&choose, F &&stop)
{
    const unsigned lane = threadIdx.x & 63, count = segments_of(q, kRest);
    unsigned units = 0, bound = first_row(q, kRest), base = 0;
    if (const Front *const fronts = q.front_of(Units{shift, kRest, kAll}.key())) {
        const unsigned piece = choose(fronts, (count + 63) / 64);
        units = fronts[piece].units;
        bound = fronts[piece].bound;
        base = 64 * piece;
    }
    for (; base < count; base += 64) {
        const unsigned s = base + lane;
        const unsigned end = max(bound, wave_scan(end_of(q, kRest, s), [](unsigned a, unsigned b) { return max(a, b); }));
        unsigned begin = (unsigned)__shfl_up((int)end, 1, 64);
        if (lane == 0) begin = bound;
        const unsigned n = s < count ? units_of(begin, end, shift, kAll) : 0;
        const unsigned upto = units + wave_scan(n, [](unsigned a, unsigned b) { return a + b; });
        const unsigned long long hit = __ballot(s < count && stop(upto - n, upto, s));
        if (hit) {
            const int l = __ffsll(hit) - 1;
            Segment r;
            const unsigned which = base + (unsigned)l;
            r.group = kRest ? (which == 0 || which == q.G + 1 ? (int)q.G : (int)which - 1) : (int)which;
            r.begin = (unsigned)__builtin_amdgcn_readlane((int)begin, l);
            r.end = (unsigned)__builtin_amdgcn_readlane((int)end, l);
            r.first = (unsigned)__builtin_amdgcn_readlane((int)(upto - n), l);
            r.unit = (unsigned)__builtin_amdgcn_readlane((int)n, l);   // (their number, for now)
            return r;
        }
        units = (unsigned)__builtin_amdgcn_readlane((int)upto, 63);
        bound = (unsigned)__builtin_amdgcn_readlane((int)end, 63);
    }
    total = units;
    return Segment{-1, 0, 0, units, 0};
}
// The segment of unit t.
template <bool kRest, bool kAll = false>
__device__ __forceinline__ Segment find_unit(const Groups &q, int shift, unsigned t)
{
    unsigned total;
    Segment r = search_segments<kRest, kAll>(
        q, shift, total,
        [&](const Front *fronts, unsigned pieces) {   // the last piece with no more than t units in front of it; the first one has none
            const unsigned lane = threadIdx.x & 63;
            unsigned piece = 0;
            while (pieces > 1) {   // 64 places of what is left at a time
                const unsigned step = (pieces + 63) / 64, at = lane * step;
                const unsigned last = (unsigned)__popcll(__ballot(at < pieces && fronts[piece + min(at, pieces - 1)].units <= t)) - 1;
                piece += last * step;
                pieces = min(step, pieces - last * step);
            }
            return piece;
        },
        [&](unsigned, unsigned upto, unsigned) { return t < upto; });
    r.unit = t - r.first;
    return r;
}
// Group g; `unit`: how many it has.
template <bool kAll = false>
__device__ __forceinline__ Segment find_group(const Groups &q, int shift, unsigned g)
{
    unsigned total;
    return search_segments<false, kAll>(
        q, shift, total, [&](const Front *, unsigned) { return g / 64; }, [&](unsigned, unsigned, unsigned s) { return s == g; });
}
template <bool kRest, bool kAll = false>
__device__ __forceinline__ unsigned count_units(const Groups &q, int shift)
{
    unsigned total = 0;
    search_segments<kRest, kAll>(
        q, shift, total, [](const Front *, unsigned pieces) { return pieces - 1; }, [](unsigned, unsigned, unsigned) { return false; });
    return total;
}
// No more units than this, whatever the offsets are.
inline size_t most_units(size_t M, size_t segments, int shift) { return (M >> shift) + segments; }

// Scratch memory of a call, whose kernels search for these units, and the fronts of them where there are many groups (dense_groups.hip).
int groups_scratch(Groups *q, std::initializer_list<Units> units, size_t bytes, char **scratch);

}  // namespace dopt
