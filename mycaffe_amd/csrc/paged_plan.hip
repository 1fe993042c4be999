// A step's plan over a paged cache: which sequences grow, which pages they get, where every new token lies.
//
// Sequence b wants n = new[b] tokens behind its len positions; n < 0: it ends.  In this order:
//   the pages of the sequences that end go on the stack of free pages, sequence after sequence;
//   a sequence without positions that begins behind the prompt of another one takes over that one's first whole pages, up to shared[b] positions;
//   sequence after sequence takes ceil((len + n) / pageSize) - ceil(len / pageSize) pages from the top of the stack.
// The first one for which pages or rows do not reach waits, and all behind it: sums over the batch decide, and no sequence overtakes another.
// Numbers are whole ones in the base type; what is read is brought into its range here, as everywhere in a paged cache.
#include <algorithm>

#include "kernels.h"
#include "paged.h"

namespace mch {

namespace {

constexpr int THREADS = 1024, WAVES = THREADS / 64;

// sums over the workgroup of numbers up to PAGED_MOST: of those before the thread's own, and of all (sums: WAVES numbers a call, read until the next barrier)
__device__ __forceinline__ int scan(int v, int* sums, int* all)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int x = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int y = __shfl_up(x, o);
        x = lane >= o ? paged_sum(x, y) : x;
    }
    const int mine = __shfl_up(x, 1);
    __syncthreads();
    if (lane == 63) sums[wave] = x;
    __syncthreads();
    int before = 0, sum = 0;
#pragma unroll
    for (int i = 0; i < WAVES; i++) {
        before = i < wave ? paged_sum(before, sums[i]) : before;
        sum = paged_sum(sum, sums[i]);
    }
    *all = sum;
    return lane ? paged_sum(before, mine) : before;
}

template <typename T> struct Plan {
    PagedPlanArgs a;
    __device__ const T* in(const void* p) const { return (const T*)p; }
    __device__ int positions() const { return a.maxPages * a.pageSize; }
    __device__ int pages_of(int len) const { return (len + a.pageSize - 1) / a.pageSize; }
    // -1: ends; else the tokens that it wants
    __device__ int wish(int b) const
    {
        const T v = in(a.wish)[b];
        return v <= (T)-1 ? -1 : paged_int(v, 0, PAGED_EXACT);
    }
    __device__ int len(int b) const { return paged_int(in(a.lens)[b], 0, positions()); }
    // whole pages that belong to others, as far as the sequence says so
    __device__ int borrowed(int b) const { return a.shared ? paged_int(in(a.shared)[b], 0, positions()) / a.pageSize : 0; }
    // pages that a sequence without positions begins behind, and whose they are
    __device__ int take(int b, int* lender) const
    {
        if (!a.from || !a.shared) return 0;
        const int f = paged_page(in(a.from)[b], a.batch);
        if (f < 0 || f == b || wish(f) < 0) return 0;
        *lender = f;
        return min(borrowed(b), len(f) / a.pageSize);
    }
};

// What one sequence asks for: positions it has to begin with, entries first .. first + need - 1 that it needs, rows (0: it cannot grow)
struct Ask { int begin, first, need, rows, take, lender; };
template <typename T> __device__ Ask ask_of(const Plan<T>& p, int b)
{
    Ask k = {0, 0, 0, 0, 0, -1};
    const int n = p.wish(b);
    k.begin = p.len(b);
    if (n <= 0) return k;
    if (k.begin == 0) {
        k.take = p.take(b, &k.lender);
        k.begin = k.take * p.a.pageSize;
    }
    k.first = p.pages_of(k.begin);
    if (n > p.positions() - k.begin) return k;
    k.rows = n;
    k.need = p.pages_of(k.begin + n) - k.first;
    return k;
}

// Workgroup 0 decides and writes everything that its decisions change; the others copy what they do not, where the block table or the list of free pages
// is not written in place (in place, they all are: a length that changes decides nothing then).
template <typename T> __global__ __launch_bounds__(THREADS) void paged_plan_kernel(Plan<T> p, int writeTokens)
{
    const PagedPlanArgs& a = p.a;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const T *table = (const T*)a.table, *free = (const T*)a.free;
    T *tableOut = (T*)a.tableOut, *freeOut = (T*)a.freeOut, *last = (T*)a.last;
    const bool copyTable = table != tableOut, copyFree = free != freeOut;
    const int have = paged_int(free[0], 0, a.pages);
    if (blockIdx.x) {
        const int others = gridDim.x - 1, me = blockIdx.x - 1;
        if (copyFree)
            for (long long i = (long long)me * THREADS + tid; i < have; i += (long long)others * THREADS) freeOut[1 + i] = free[1 + i];
        if (copyTable)
            for (int b = me * WAVES + wave; b < a.batch; b += others * WAVES) {
                const Ask k = ask_of(p, b);
                const bool ends = p.wish(b) < 0;
                const T *from = table + (size_t)b * a.maxPages;
                T* to = tableOut + (size_t)b * a.maxPages;
                for (int e = lane; e < a.maxPages; e += 64)
                    if (ends) to[e] = (T)-1;
                    else if (e >= k.take && (e < k.first || e >= k.first + k.need)) to[e] = from[e];
            }
        return;
    }
    __shared__ int sums[2][WAVES], sStart[THREADS + 1], sNeed[THREADS + 1], sFirst[THREADS], sBegin[THREADS];
    // ---- the sequences that end: how many pages each gives back, then the pages themselves ----
    int count = have;
    for (int b0 = 0; b0 < a.batch; b0 += THREADS) {
        const int mine = b0 + tid;
        const bool ends = mine < a.batch && p.wish(mine) < 0;
        if (!__syncthreads_or(ends)) continue;
        sNeed[tid] = 0;
        const uint64_t some = __ballot(ends);
        for (uint64_t m = some; m; m &= m - 1) {
            const int at = 64 * wave + __builtin_ctzll(m), b = b0 + at, to = p.pages_of(p.len(b));
            int n = 0;
            for (int e0 = p.borrowed(b); e0 < to; e0 += 64)
                n += __popcll(__ballot(e0 + lane < to && paged_page(table[(size_t)b * a.maxPages + e0 + lane], a.pages) >= 0));
            if (lane == 0) sNeed[at] = n;
        }
        __syncthreads();
        int all;
        const int before = scan(sNeed[tid], sums[0], &all);
        sStart[tid] = before;
        __syncthreads();
        for (uint64_t m = some; m; m &= m - 1) {
            const int at = 64 * wave + __builtin_ctzll(m), b = b0 + at, to = p.pages_of(p.len(b));
            int n = paged_sum(count, sStart[at]);
            for (int e0 = p.borrowed(b); e0 < to; e0 += 64) {
                const int page = e0 + lane < to ? paged_page(table[(size_t)b * a.maxPages + e0 + lane], a.pages) : -1;
                const uint64_t given = __ballot(page >= 0);
                const int place = paged_sum(n, __popcll(given & ((1ull << lane) - 1)));
                if (page >= 0 && place < a.pages) freeOut[1 + place] = (T)page;
                n = paged_sum(n, __popcll(given));
            }
        }
        count = min(paged_sum(count, all), a.pages);
    }
    // what a lender has is what it had before the call: where lengths change in place, all of them are looked up before any is changed
    if (a.from)
        for (int b = tid; b < a.batch; b += THREADS) last[b] = (T)ask_of(p, b).take;
    __syncthreads();
    // ---- sequence after sequence, 1024 of them at a time ----
    int taken = 0, rows = 0, askedPages = 0, askedRows = 0;
    for (int b0 = 0; b0 < a.batch; b0 += THREADS) {
        const int b = b0 + tid, n = b < a.batch ? p.wish(b) : 0;
        Ask k = {0, 0, 0, 0, 0, -1};
        T shared = (T)0;
        if (b < a.batch) {
            // as ask_of, but for the lender's length
            k.begin = p.len(b);
            shared = a.shared ? (T)paged_int(((const T*)a.shared)[b], 0, p.positions()) : (T)0;
            if (n > 0) {
                if (k.begin == 0 && a.from) {
                    k.take = (int)last[b];
                    k.lender = k.take ? (int)((const T*)a.from)[b] : -1;
                    k.begin = k.take * a.pageSize;
                }
                k.first = p.pages_of(k.begin);
                if (n <= p.positions() - k.begin) {
                    k.rows = n;
                    k.need = p.pages_of(k.begin + n) - k.first;
                }
            }
        }
        int allPages, allRows;
        const int pagesBefore = paged_sum(askedPages, scan(k.need, sums[0], &allPages)), rowsBefore = paged_sum(askedRows, scan(k.rows, sums[1], &allRows));
        const bool granted = k.rows && paged_sum(pagesBefore, k.need) <= count && paged_sum(rowsBefore, k.rows) <= a.tokens;
        askedPages = paged_sum(askedPages, allPages);
        askedRows = paged_sum(askedRows, allRows);
        // those that wait are behind all that are granted: sums over the granted ones are these, up to the first that waits
        const int grantedRows = granted ? k.rows : 0, grantedPages = granted ? k.need : 0;
        int chunkRows, chunkPages;
        const int rowAt = rows + scan(grantedRows, sums[0], &chunkRows), pageAt = taken + scan(grantedPages, sums[1], &chunkPages);
        sStart[tid] = rowAt;
        sNeed[tid] = pageAt;
        sFirst[tid] = k.first;
        sBegin[tid] = k.begin;
        if (tid == 0) {
            sStart[THREADS] = rows + chunkRows;
            sNeed[THREADS] = taken + chunkPages;
        }
        const bool wasEmpty = b < a.batch && p.len(b) == 0;
        __syncthreads();
        if (b < a.batch) {
            ((T*)a.lensOut)[b] = n < 0 ? (T)0 : granted ? (T)(k.begin + k.rows) : (T)p.len(b);
            ((T*)a.starts)[b] = (T)rowAt;
            last[b] = granted ? (T)(rowAt + k.rows - 1) : (T)-1;
            if (a.sharedOut) ((T*)a.sharedOut)[b] = n < 0 ? (T)0 : granted && wasEmpty ? (T)(k.take * a.pageSize) : shared;
        }
        // pages: one thread each, that finds its sequence
        auto whose = [&](const int* starts, int i) -> int {
            int lo = 0, hi = THREADS;
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (starts[mid] <= i) lo = mid;
                else hi = mid;
            }
            return lo;
        };
        for (int i = taken + tid; i < taken + chunkPages; i += THREADS) {
            const int s = whose(sNeed, i);
            const int at = count - 1 - i;
            const T page = at < have ? free[1 + at] : freeOut[1 + at];
            tableOut[(size_t)(b0 + s) * a.maxPages + sFirst[s] + i - sNeed[s]] = (T)paged_page(page, a.pages);
        }
        // borrowed pages, and of a row that is copied what the others have left for those that wait
        for (uint64_t m = __ballot(k.take > 0 || (copyTable && !granted && k.need > 0)); m; m &= m - 1) {
            const int s = __builtin_ctzll(m), to = __shfl(k.take, s), lender = __shfl(k.lender, s), first = __shfl(k.first, s), need = __shfl(k.need, s);
            const bool ok = __shfl((int)granted, s);
            const size_t row = (size_t)(b0 + 64 * wave + s) * a.maxPages;
            if (ok)
                for (int e = lane; e < to; e += 64) tableOut[row + e] = table[(size_t)lender * a.maxPages + e];
            else if (copyTable) {
                for (int e = lane; e < to; e += 64) tableOut[row + e] = table[row + e];
                for (int e = first + lane; e < first + need; e += 64) tableOut[row + e] = table[row + e];
            }
        }
        if (!copyTable)
            for (uint64_t m = __ballot(n < 0); m; m &= m - 1) {
                const size_t row = (size_t)(b0 + 64 * wave + __builtin_ctzll(m)) * a.maxPages;
                for (int e = lane; e < a.maxPages; e += 64) tableOut[row + e] = (T)-1;
            }
        __syncthreads();
        if (writeTokens)
            for (int i = rows + tid; i < rows + chunkRows; i += THREADS) {
                const int s = whose(sStart, i), pos = sBegin[s] + i - sStart[s], e = pos / a.pageSize;
                // entries in front of the new ones are as they were
                const T* from = e >= sFirst[s] ? (const T*)tableOut : table;
                const int page = paged_page(from[(size_t)(b0 + s) * a.maxPages + e], a.pages);
                if (a.positions) ((T*)a.positions)[i] = (T)pos;
                if (a.slots) ((T*)a.slots)[i] = page >= 0 ? (T)(page * a.pageSize + pos - e * a.pageSize) : (T)-1;
            }
        rows += chunkRows;
        taken += chunkPages;
        __syncthreads();
    }
    if (tid == 0) {
        ((T*)a.starts)[a.batch] = (T)rows;
        freeOut[0] = (T)(count - taken);
    }
}

// positions and slots of the rows of a large step, a workgroup a sequence
template <typename T> __global__ __launch_bounds__(256) void paged_plan_rows_kernel(Plan<T> p)
{
    const PagedPlanArgs& a = p.a;
    const T* starts = (const T*)a.starts;
    for (int b = blockIdx.x; b < a.batch; b += gridDim.x) {
        const int first = (int)starts[b], count = (int)starts[b + 1] - first, begin = (int)((const T*)a.lensOut)[b] - count;
        for (int i = threadIdx.x; i < count; i += 256) {
            const int pos = begin + i, e = pos / a.pageSize, page = paged_page(((const T*)a.tableOut)[(size_t)b * a.maxPages + e], a.pages);
            if (a.positions) ((T*)a.positions)[first + i] = (T)pos;
            if (a.slots) ((T*)a.slots)[first + i] = page >= 0 ? (T)(page * a.pageSize + pos - e * a.pageSize) : (T)-1;
        }
    }
}

constexpr int ROWS_OF_ONE = 8192;   // rows up to which the first workgroup writes their places too

template <typename T> hipError_t launch(hipStream_t s, const PagedPlanArgs& a)
{
    Plan<T> p = {a};
    const long long entries = (a.table != a.tableOut ? (long long)a.batch * a.maxPages : 0) + (a.free != a.freeOut ? a.pages : 0);
    const int others = (int)std::min<long long>(256, (entries + 4 * THREADS - 1) / (4 * THREADS));
    const bool rows = a.positions || a.slots, own = a.tokens <= ROWS_OF_ONE;
    hipLaunchKernelGGL((paged_plan_kernel<T>), 1 + others, THREADS, 0, s, p, rows && own ? 1 : 0);
    if (rows && !own) hipLaunchKernelGGL((paged_plan_rows_kernel<T>), std::min(a.batch, 65535), 256, 0, s, p);
    return hipGetLastError();
}

}  // namespace

hipError_t k_paged_plan(hipStream_t s, bool wide, const PagedPlanArgs& a) { return wide ? launch<double>(s, a) : launch<float>(s, a); }

}  // namespace mch
