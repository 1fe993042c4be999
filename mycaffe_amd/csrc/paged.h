// Sequences in a paged cache: which rows of a launch are whose, and where a position's keys and values lie.
//
// All of it comes in tensors of the base type, fp32 or double, as every index of this ABI does (embedding ids, transposition counts): whole numbers,
// exact in fp32 up to 2^24, which the entry points hold every count to.  What the device reads is never trusted: every number is brought into
// its range here before anything is addressed with it, and a number that is not a number counts as the lowest of its range or as
// no page.  Host and device compile the same lines (the host's test feeds them everything that can go wrong).
#pragma once
#include <stdint.h>
#ifdef __HIPCC__
#include <hip/hip_runtime.h>
#endif

#include <algorithm>
#include <utility>

namespace mch {

#ifdef __HIPCC__
#define PAGED_FN __host__ __device__ inline
#else
#define PAGED_FN inline
#endif

constexpr int PAGED_EXACT = 1 << 24;   // whole numbers up to here are exact in fp32
// Lists of work are counted up to here and no further.  The host sees to it that sequences whose starts never decrease stay below; a list that does
// reach it (starts that decrease give the same tokens to many sequences) is none.
constexpr int PAGED_MOST = 0x3fffffff;
PAGED_FN int paged_sum(int a, int b) { return a + b < PAGED_MOST ? a + b : PAGED_MOST; }   // of two up to PAGED_MOST

// v as a whole number in lo .. hi
template <typename T> PAGED_FN int paged_int(T v, int lo, int hi) { return v >= (T)hi ? hi : v > (T)lo ? (int)v : lo; }
// an entry of a block table: a page, or -1
template <typename T> PAGED_FN int paged_page(T v, int pages) { return v >= (T)0 && v < (T)pages ? (int)v : -1; }

// New tokens of a sequence: rows first .. first + count - 1 of the launch, cached positions 0 .. len - 1 with the new ones last
struct PagedSpan { int first, count, len; };
template <typename T> PAGED_FN PagedSpan paged_span(T start, T next, T len, int tokens, int positions)
{
    PagedSpan s;
    s.first = paged_int(start, 0, tokens);
    s.count = paged_int(next, s.first, tokens) - s.first;
    s.len = paged_int(len, 0, positions);
    return s;
}

// A list of `total` units of work dealt to at most `most` workgroups, at least `least` units each: equal runs, the first ones longer by one
struct PagedRuns {
    int W, run, more;
    PAGED_FN PagedRuns(int total, int most, int least)
    {
        const int want = total / least;
        W = want < 1 ? (total > 0 ? 1 : 0) : want < most ? want : most;
        run = W ? total / W : 0;
        more = total - run * W;
    }
    PAGED_FN int begin(int i) const { return run * i + (i < more ? i : more); }
    PAGED_FN int of(int u) const { return u < (run + 1) * more ? u / (run + 1) : more + (u - (run + 1) * more) / run; }   // whose unit u is
};
// Workgroup -> place in the list, so that an XCD (workgroup i is on XCD i % 8) has neighbouring runs; -1: none of W
PAGED_FN int paged_place(int block, int W)
{
    const int x = block & 7, k = block >> 3, each = W >> 3, rest = W & 7;
    return k < each + (x < rest ? 1 : 0) ? x * each + (x < rest ? x : rest) + k : -1;
}
#ifdef __HIPCC__
// the sequence whose rows hold token `i`: the last one that starts at or before it.  All 64 lanes ask.
__device__ __forceinline__ int sequence_of(const float* starts, int batch, int tokens, int i)
{
    int n = 0;
    for (int b0 = 0; b0 < batch; b0 += 64) {
        const int b = b0 + (threadIdx.x & 63);
        const bool before = b < batch && paged_int(starts[b], 0, tokens) <= i;
        const uint64_t m = __ballot(before);
        if (!m) break;
        n = b0 + 64 - __builtin_clzll(m);
    }
    return n - 1;
}
#endif
// Units of the first t tiles of a chunk: tiles of perTile tokens, the first of them over `before` + perTile positions, every further one over perTile more;
// about 32 << shift positions a unit, and one for the tile
PAGED_FN int paged_units_before(int before, int perTile, int t, int shift)
{
    const unsigned long long n = t;
    return (int)((n * (unsigned)before + (unsigned)perTile * (n * (n + 1) / 2)) >> (5 + shift)) + t;
}
// the tile that unit u is in, of those that begin before `tiles`
PAGED_FN int paged_tile_of(int before, int perTile, int tiles, int shift, int u)
{
    int lo = 0, hi = tiles - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (paged_units_before(before, perTile, mid, shift) <= u) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// ---- what the entry points check, l as in the calls: {batch, tokens, heads, kvHeads, hs, pages, pageSize, maxPages, 7 handles, stridePage, strideHead, stridePos}
inline bool paged_sizes_ok(const long long* l)
{
    for (int i = 0; i < 8; i++)
        if (l[i] < 1 || l[i] > PAGED_EXACT) return false;
    return l[2] <= 65535 && l[2] % l[3] == 0 && l[4] <= 256 && l[4] % 2 == 0 && l[6] * l[7] <= PAGED_EXACT && l[15] >= 0 && l[16] >= 0 && l[17] >= 0;
}
// values from the first of a cache to behind its last; -1: more than `most`
inline long long paged_reach(const long long* l, long long most)
{
    const long long n[3] = {l[5], l[3], l[6]};
    long long reach = l[4];
    for (int i = 0; i < 3; i++) {
        if (n[i] == 1) continue;
        if (l[15 + i] > most) return -1;
        reach += (n[i] - 1) * l[15 + i];
    }
    return reach <= most ? reach : -1;
}
// Whether every value of two caches, `apart` values from each other, has a place of its own: each stride reaches past what the smaller ones span, and so
// does the distance where the two interleave (rows k | v, say)
inline bool paged_apart(const long long* l, long long apart, long long reach)
{
    std::pair<long long, long long> dims[4] = {{l[15], l[5]}, {l[16], l[3]}, {l[17], l[6]}, {apart, apart < reach ? 2 : 1}};
    std::sort(dims, dims + 4);
    long long span = l[4];
    for (const auto& d : dims) {
        if (d.second == 1) continue;
        if (d.first < span) return false;
        span += (d.second - 1) * d.first;
    }
    return true;
}

}  // namespace mch
