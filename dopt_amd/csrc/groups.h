// Groups of consecutive rows, given by where they begin: offsets[0 .. G] on the device, a group g from offsets[g] up to offsets[g + 1].
// Whatever the values are, a kernel sees boundaries that lie within the rows and do not fall: each is taken as the largest up to it, and
// as M beyond that.  Rows in front of the first group and behind the last one belong to none.
#pragma once

#include "common.h"

namespace dopt {

struct Groups {
    const int *offsets;   // (null without groups)
    unsigned G, M;
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

// Segments in the order of the rows: rows of no group, the groups, rows of no group (kRest), or the groups alone.  A segment of r rows is
// ceil(r / 2^shift) units, or one where it is empty and kAll.  `stop(units in front, units up to and with the segment, segment)` says in which of
// them the search ends; every wavefront does it for itself, 64 segments at a time.
template <bool kRest, bool kAll, class F>
__device__ __forceinline__ Segment search_segments(const Groups &q, int shift, unsigned &total, F &&stop)
{
    const unsigned lane = threadIdx.x & 63, count = kRest ? q.G + 2 : q.G;
    unsigned units = 0, bound = 0;
    if (!kRest && count) bound = (unsigned)min(max(q.offsets[0], 0), (int)q.M);
    for (unsigned base = 0; base < count; base += 64) {
        const unsigned s = base + lane, at = kRest ? s : s + 1;   // the segment ends at offsets[at]
        unsigned end = q.M;
        if (at <= q.G && s < count && q.offsets) end = (unsigned)min(max(q.offsets[at], 0), (int)q.M);
        end = max(bound, wave_scan(end, [](unsigned a, unsigned b) { return max(a, b); }));
        unsigned begin = (unsigned)__shfl_up((int)end, 1, 64);
        if (lane == 0) begin = bound;
        unsigned n = s < count ? (unsigned)(((size_t)end - begin + ((size_t)1 << shift) - 1) >> shift) : 0;
        if (kAll && s < count && n == 0) n = 1;
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
    Segment r = search_segments<kRest, kAll>(q, shift, total, [&](unsigned, unsigned upto, unsigned) { return t < upto; });
    r.unit = t - r.first;
    return r;
}
// Group g; `unit`: how many it has.
template <bool kAll = false>
__device__ __forceinline__ Segment find_group(const Groups &q, int shift, unsigned g)
{
    unsigned total;
    return search_segments<false, kAll>(q, shift, total, [&](unsigned, unsigned, unsigned s) { return s == g; });
}
template <bool kRest, bool kAll = false>
__device__ __forceinline__ unsigned count_units(const Groups &q, int shift)
{
    unsigned total = 0;
    search_segments<kRest, kAll>(q, shift, total, [](unsigned, unsigned, unsigned) { return false; });
    return total;
}
// No more units than this, whatever the offsets are.
inline size_t most_units(size_t M, size_t segments, int shift) { return (M >> shift) + segments; }

}  // namespace dopt
