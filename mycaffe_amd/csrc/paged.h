// Sequences in a paged cache: which rows of a launch are whose, and where a position's keys and values lie.
//
// All of it comes in fp32 tensors, as every index of this ABI does (embedding ids, transposition counts): whole numbers, exact up
// to 2^24, which the entry points hold every count to.  What the device reads is never trusted: every number is brought into
// its range here before anything is addressed with it, and a number that is not a number counts as the lowest of its range or as
// no page.  Host and device compile the same lines (the host's test feeds them everything that can go wrong).
#pragma once
#include <stdint.h>

namespace mch {

#ifdef __HIPCC__
#define PAGED_FN __host__ __device__ inline
#else
#define PAGED_FN inline
#endif

constexpr int PAGED_EXACT = 1 << 24;   // whole numbers up to here are exact in fp32

// v as a whole number in lo .. hi
PAGED_FN int paged_int(float v, int lo, int hi) { return v >= (float)hi ? hi : v > (float)lo ? (int)v : lo; }
// an entry of a block table: a page, or -1
PAGED_FN int paged_page(float v, int pages) { return v >= 0.f && v < (float)pages ? (int)v : -1; }

// New tokens of a sequence: rows first .. first + count - 1 of the launch, cached positions 0 .. len - 1 with the new ones last
struct PagedSpan { int first, count, len; };
PAGED_FN PagedSpan paged_span(float start, float next, float len, int tokens, int positions)
{
    PagedSpan s;
    s.first = paged_int(start, 0, tokens);
    s.count = paged_int(next, s.first, tokens) - s.first;
    s.len = paged_int(len, 0, positions);
    return s;
}

}  // namespace mch
