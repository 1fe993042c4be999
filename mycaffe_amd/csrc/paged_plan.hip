// A step's plan over a paged cache: which sequences grow, which pages they get, where every new token lies.
//
// Sequence b wants n = new[b] tokens behind its len positions; n < 0: it ends.  In this order:
//   the pages of the sequences that end go on the stack of free pages, sequence after sequence;
//   a sequence without positions that begins behind the prompt of another one takes over that one's first whole pages, up to shared[b] positions;
//   sequence after sequence takes ceil((len + n) / pageSize) - ceil(len / pageSize) pages from the top of the stack.
// The first one for which pages or rows do not reach waits, and all behind it: sums over the batch decide, and no sequence overtakes another.
// Of the stack only what remains is written: a page that comes back and is taken again in the same call goes straight to the row that gets it.
// Numbers are whole ones in the base type; what is read is brought into its range here, as everywhere in a paged cache.
#include <algorithm>

#include "attn_paged.h"
#include "kernels.h"
#include "paged.h"

namespace mch {

namespace {

// sums over the workgroup of numbers up to PAGED_MOST: of those before the thread's own, and of all (sums: as many numbers as wavefronts, read until the next call)
template <int THREADS> __device__ __forceinline__ int scan(int v, int* sums, int* all)
{
    constexpr int WAVES = THREADS / 64;
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), x = wave_scan(v);
    __syncthreads();
    if (lane == 63) sums[wave] = x;
    __syncthreads();
    const int upTo = wave_scan(lane < WAVES ? sums[lane] : 0);
    *all = __builtin_amdgcn_readlane(upTo, WAVES - 1);
    const int before = wave ? __builtin_amdgcn_readlane(upTo, wave ? wave - 1 : 0) : 0, mine = __builtin_amdgcn_update_dpp(0, x, 0x138, 0xf, 0xf, false);   // wave_shr 1
    return paged_sum(before, mine);
}

template <typename T> struct Plan {
    PagedPlanArgs a;
    __device__ const T* in(const void* p) const { return (const T*)p; }
    __device__ int positions() const { return a.maxPages * a.pageSize; }
    __device__ int pages_of(int len) const { return (len + a.pageSize - 1) / a.pageSize; }
    // free pages that remain whatever the call decides: a sequence takes no more than its rows fill and one that they begin
    __host__ __device__ int remain(int have) const { return std::max(have - a.tokens / a.pageSize - std::min(a.batch, a.tokens), 0); }
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
template <typename T> __device__ __forceinline__ Ask ask_of(const Plan<T>& p, int b, int wish, int len, int take, int lender)
{
    Ask k = {len, 0, 0, 0, 0, -1};
    if (wish <= 0) return k;
    if (len == 0) {
        k.take = take;
        k.lender = lender;
        k.begin = take * p.a.pageSize;
    }
    k.first = p.pages_of(k.begin);
    if (wish > p.positions() - k.begin) return k;
    k.rows = wish;
    k.need = p.pages_of(k.begin + wish) - k.first;
    return k;
}
template <typename T> __device__ __forceinline__ Ask ask_of(const Plan<T>& p, int b)
{
    int lender = -1;
    const int wish = p.wish(b), len = p.len(b), take = wish > 0 && len == 0 ? p.take(b, &lender) : 0;
    return ask_of(p, b, wish, len, take, lender);
}

// Workgroup 0 decides and writes everything that its decisions change or may change; the others copy what they cannot, where the block table and the list of free pages
// are not written in place (in place, they all are: a length that changes decides nothing then).
// What bounds it is one read behind the other in workgroup 0, so whatever it goes through - sequences, pages that come back, pages that are taken, entries that are copied -
// is one list of items each, a thread an item, whose sequence it finds in the list's sums.  Measured, all memory of its own: 4 sequences of one token 4.7 us (an empty call takes 3.3 - 3.8), 512
// with tables of 512 entries, a tenth of which end or begin, 17 - 20 us (13.2 and 5.6 for the rows), 256 prompts 16 - 17; with loops over the sequences in place of the lists 8.4, 30 and 33.
// In place, a token for each of 4, 64 and 512 sequences, 4.6, 5.7 and 6.1 us (elsewhere 5.0, 6.0 and 6.6).
template <typename T, int THREADS> __global__ __launch_bounds__(THREADS) void paged_plan_kernel(Plan<T> p, int writeTokens)
{
    constexpr int WAVES = THREADS / 64;
    const PagedPlanArgs& a = p.a;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const T *table = (const T*)a.table, *free = (const T*)a.free;
    T *tableOut = (T*)a.tableOut, *freeOut = (T*)a.freeOut, *last = (T*)a.last;
    const bool copyTable = table != tableOut, copyFree = free != freeOut;
    const int have = paged_int(free[0], 0, a.pages);
    if (blockIdx.x) {
        const int others = gridDim.x - 1, me = blockIdx.x - 1;
        constexpr int EACH = 8;   // reads under way
        const int remain = p.remain(have);
        if (copyFree)
            for (long long i0 = (long long)me * EACH * THREADS + tid; i0 < remain; i0 += (long long)others * EACH * THREADS) {
                T v[EACH];
#pragma unroll
                for (int j = 0; j < EACH; j++) v[j] = free[1 + min(i0 + j * THREADS, (long long)remain - 1)];
#pragma unroll
                for (int j = 0; j < EACH; j++)
                    if (i0 + j * THREADS < remain) freeOut[1 + i0 + j * THREADS] = v[j];
            }
        if (copyTable)
            for (int b = me * WAVES + wave; b < a.batch; b += others * WAVES) {
                const T *from = table + (size_t)b * a.maxPages;
                T* to = tableOut + (size_t)b * a.maxPages;
                T v[EACH];
                auto read = [&](int e0) __attribute__((always_inline)) {
#pragma unroll
                    for (int j = 0; j < EACH; j++) v[j] = from[min(e0 + 64 * j + lane, a.maxPages - 1)];
                };
                read(0);
                const Ask k = ask_of(p, b);
                const bool ends = p.wish(b) < 0;
                for (int e0 = 0; e0 < a.maxPages; e0 += 64 * EACH) {
#pragma unroll
                    for (int j = 0; j < EACH; j++) {
                        const int e = e0 + 64 * j + lane;
                        if (e < a.maxPages && (ends || (e >= k.take && (e < k.first || e >= k.first + k.need)))) to[e] = ends ? (T)-1 : v[j];
                    }
                    if (e0 + 64 * EACH < a.maxPages) read(e0 + 64 * EACH);
                }
            }
        return;
    }
    __shared__ int sums[3][WAVES], sStart[THREADS + 1], sNeed[THREADS + 1], sCopy[THREADS + 1], sFirst[THREADS], sBegin[THREADS], sTake[THREADS], sRows, sPages;
    __shared__ int sBack[THREADS + 1], sBackFrom[THREADS], sBackEnd[THREADS];
    // the sequence of item i of a list, by the sums in front of each
    auto whose = [&](const int* starts, int i) __attribute__((always_inline)) -> int {
        int lo = 0;
#pragma unroll
        for (int o = THREADS / 2; o > 0; o >>= 1) lo = starts[lo + o] <= i ? lo + o : lo;
        return lo;
    };
    // What a lender has is what it had before the call: where lengths change in place and there are more sequences than threads, all of them are looked up before
    // any is changed.
    const bool ahead = a.from && a.batch > THREADS;
    struct Asks { int wish, len, shared; Ask k; };
    auto asks_of = [&](int b, bool looked) __attribute__((always_inline)) -> Asks {
        Asks q = {0, 0, 0, {0, 0, 0, 0, 0, -1}};
        if (b >= a.batch) return q;
        q.wish = p.wish(b);
        q.len = p.len(b);
        q.shared = a.shared ? paged_int(((const T*)a.shared)[b], 0, p.positions()) : 0;
        int lender = -1, take = 0;
        if (q.wish > 0 && q.len == 0 && a.from) {
            if (looked) {
                take = (int)last[b];
                lender = take ? (int)((const T*)a.from)[b] : -1;
            } else take = p.take(b, &lender);
        }
        q.k = ask_of(p, b, q.wish, q.len, take, lender);
        return q;
    };
    const Asks first = asks_of(tid, false);   // read once, ahead of everything
    // ---- the pages of the sequences that end, in the order of the sequences: places have, have + 1, ... of the stack ----
    constexpr int EACH = 8;   // entries of a thread, one behind the other, at most
    // the entries of those of sequences b0 .. b0 + THREADS - 1 as a list
    auto entries_back = [&](int b0) __attribute__((always_inline)) -> int {
        const int mine = b0 + tid, wish = b0 ? mine < a.batch ? p.wish(mine) : 0 : first.wish;
        const bool ends = wish < 0;
        if (!__syncthreads_or(ends)) return 0;
        const int from = !ends ? 0 : b0 ? p.borrowed(mine) : first.shared / a.pageSize, to = !ends ? 0 : p.pages_of(b0 ? p.len(mine) : first.len);
        int items;
        const int at = scan<THREADS>(max(to - from, 0), sums[0], &items);
        sBack[tid] = at;
        sBackFrom[tid] = from - at;
        sBackEnd[tid] = at + max(to - from, 0);
        __syncthreads();
        return items;
    };
    // the thread's entries of that list, of THREADS EACH from i0 on (-1: no page), and where the first page of them goes behind the `at` that lie in front
    auto pages_back = [&](int b0, int items, int i0, int (&page)[EACH], int* at) __attribute__((always_inline)) -> int {
        const int per = min((items - i0 + THREADS - 1) / THREADS, EACH);
        int valid = 0, all, end = -1, s = 0;
        T entry[EACH];
#pragma unroll
        for (int e = 0; e < EACH; e++) {
            const int i = i0 + per * tid + e;
            entry[e] = (T)-1;
            if (e >= per || i >= items) continue;
            if (i >= end) {
                s = whose(sBack, i);
                end = sBackEnd[s];
            }
            entry[e] = table[(size_t)(b0 + s) * a.maxPages + sBackFrom[s] + i];
        }
#pragma unroll
        for (int e = 0; e < EACH; e++) {
            page[e] = paged_page(entry[e], a.pages);
            valid += page[e] >= 0;
        }
        const int place = paged_sum(*at, scan<THREADS>(valid, sums[1], &all));
        *at = min(paged_sum(*at, all), a.pages);
        return place;
    };
    int count = have, look[EACH], lookAt = have;
    bool one = true;   // one look at them is all of them
#pragma unroll
    for (int e = 0; e < EACH; e++) look[e] = -1;
    for (int b0 = 0; b0 < a.batch; b0 += THREADS) {
        const int items = entries_back(b0);
        one = one && a.batch <= THREADS && items <= EACH * THREADS;
        for (int i0 = 0; i0 < items; i0 += EACH * THREADS) lookAt = pages_back(b0, items, i0, look, &count);
    }
    // f(place, page) for those at places lo .. hi - 1
    auto back = [&](int lo, int hi, auto f) __attribute__((always_inline)) {
        auto each = [&](const int (&page)[EACH], int place) __attribute__((always_inline)) {
#pragma unroll
            for (int e = 0; e < EACH; e++)
                if (page[e] >= 0) {
                    if (place >= lo && place < hi) f(place, page[e]);
                    place++;
                }
        };
        if (lo >= hi) return;
        if (one) {
            each(look, lookAt);
            return;
        }
        int at = have;
        for (int b0 = 0; b0 < a.batch && at < hi; b0 += THREADS) {
            const int items = entries_back(b0);
            for (int i0 = 0; i0 < items; i0 += EACH * THREADS) {
                int page[EACH];
                const int place = pages_back(b0, items, i0, page, &at);
                each(page, place);
            }
        }
    };
    if (ahead)
        for (int b = tid; b < a.batch; b += THREADS) last[b] = (T)ask_of(p, b).take;
    __syncthreads();
    // ---- sequence after sequence, as many at a time as there are threads ----
    int taken = 0, rows = 0, askedPages = 0, askedRows = 0;
    for (int b0 = 0; b0 < a.batch; b0 += THREADS) {
        const int b = b0 + tid;
        const Asks asks = b0 ? asks_of(b, ahead) : first;
        const int n = asks.wish, len = asks.len;
        const Ask k = asks.k;
        if (tid == 0) { sRows = rows; sPages = taken; }
        int allPages, allRows, copies;
        const int pagesBefore = paged_sum(askedPages, scan<THREADS>(k.need, sums[0], &allPages)), rowsBefore = paged_sum(askedRows, scan<THREADS>(k.rows, sums[1], &allRows));
        // Of those that are granted nobody waits in front: the sums of what is asked are what they get.
        const bool granted = k.rows && paged_sum(pagesBefore, k.need) <= count && paged_sum(rowsBefore, k.rows) <= a.tokens;
        const uint64_t some = __ballot(granted);
        if (granted && lane == 63 - __builtin_clzll(some)) {
            atomicMax(&sRows, rowsBefore + k.rows);
            atomicMax(&sPages, pagesBefore + k.need);
        }
        // borrowed entries, and of a row that is copied what the others have left for those that wait
        const int copy = granted ? k.take : copyTable ? k.take + k.need : 0;
        sCopy[tid] = scan<THREADS>(copy, sums[2], &copies);
        const int rowsUpTo = sRows, pagesUpTo = sPages;   // (written before the scan's barriers)
        const int rowAt = min(rowsBefore, rowsUpTo);   // a sequence that gets nothing stands where the next one that does begins
        sStart[tid] = rowAt;
        sNeed[tid] = min(pagesBefore, pagesUpTo);
        sFirst[tid] = k.first;
        sBegin[tid] = k.begin;
        sTake[tid] = granted ? k.lender : -1 - k.take;
        askedPages = paged_sum(askedPages, allPages);
        askedRows = paged_sum(askedRows, allRows);
        if (b < a.batch) {
            ((T*)a.starts)[b] = (T)rowAt;
            last[b] = granted ? (T)(rowAt + k.rows - 1) : (T)-1;
            if (n >= 0) {   // (what those have that end is read until the end)
                ((T*)a.lensOut)[b] = granted ? (T)(k.begin + k.rows) : (T)len;
                if (a.sharedOut) ((T*)a.sharedOut)[b] = granted && len == 0 ? (T)(k.take * a.pageSize) : (T)asks.shared;
            }
        }
        __syncthreads();
        // page `i` of those that are taken is the stack's at place count - 1 - i
        auto give = [&](int i, int page) __attribute__((always_inline)) {
            const int s = whose(sNeed, i);
            tableOut[(size_t)(b0 + s) * a.maxPages + sFirst[s] + i - sNeed[s]] = (T)page;
        };
        for (int i = max(taken, count - have) + tid; i < pagesUpTo; i += THREADS) give(i, paged_page(free[count - i], a.pages));
        // those that come back: to the rows, and what is left of them, behind the last sequences, to the stack
        const int left = count - pagesUpTo;
        back(b0 + THREADS < a.batch ? max(have, left) : have, count - taken, [&](int place, int page) __attribute__((always_inline)) {
            if (place < left) freeOut[1 + place] = (T)page;
            else give(count - 1 - place, page);
        });
        for (int i = tid; i < copies; i += THREADS) {
            const int s = whose(sCopy, i), j = i - sCopy[s], lender = sTake[s], row = b0 + s;
            // of a row that waits: its first entries, as many as it would have borrowed, then those that it would have got
            const int e = lender >= 0 || j < -1 - lender ? j : sFirst[s] + j - (-1 - lender);
            tableOut[(size_t)row * a.maxPages + e] = table[(size_t)(lender >= 0 ? lender : row) * a.maxPages + e];
        }
        __syncthreads();
        if (writeTokens)
            for (int i = rows + tid; i < rowsUpTo; i += THREADS) {
                const int s = whose(sStart, i), pos = sBegin[s] + i - sStart[s], e = pos / a.pageSize;
                // entries in front of the new ones are as they were
                const T* from = e >= sFirst[s] ? (const T*)tableOut : table;
                const int page = paged_page(from[(size_t)(b0 + s) * a.maxPages + e], a.pages);
                if (a.positions) ((T*)a.positions)[i] = (T)pos;
                if (a.slots) ((T*)a.slots)[i] = page >= 0 ? (T)(page * a.pageSize + pos - e * a.pageSize) : (T)-1;
            }
        rows = rowsUpTo;
        taken = pagesUpTo;
        __syncthreads();
    }
    for (int b0 = 0; b0 < a.batch; b0 += THREADS) {
        const int b = b0 + tid;
        const bool ends = b < a.batch && (b0 ? p.wish(b) : first.wish) < 0;
        if (ends) {
            ((T*)a.lensOut)[b] = (T)0;
            if (a.sharedOut) ((T*)a.sharedOut)[b] = (T)0;
        }
        if (!copyTable)
            for (uint64_t m = __ballot(ends); m; m &= m - 1) {
                const size_t row = (size_t)(b0 + 64 * wave + __builtin_ctzll(m)) * a.maxPages;
                for (int e = lane; e < a.maxPages; e += 64) tableOut[row + e] = (T)-1;
            }
    }
    if (copyFree)
        for (int i0 = p.remain(have) + tid, end = min(have, count - taken); i0 < end; i0 += EACH * THREADS) {
            T v[EACH];
#pragma unroll
            for (int j = 0; j < EACH; j++) v[j] = free[1 + min(i0 + j * THREADS, end - 1)];
#pragma unroll
            for (int j = 0; j < EACH; j++)
                if (i0 + j * THREADS < end) freeOut[1 + i0 + j * THREADS] = v[j];
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

// Rows up to which the first workgroup writes their places too.  us, it | a launch more: 32 prompts, 4096 rows 7.6 | 9.5, 16384 8.8 | 10.4, 256 prompts, 32768 rows 15.3 | 12.0, 65536
// 57 | 15
constexpr int ROWS_OF_ONE = 16384;
// Sequences and rows up to which four wavefronts do.  us, four | sixteen: 4 sequences of one token 4.8 | 5.3, 8 prompts, 1024 rows 5.6 | 6.5, 32 sequences of one token 7.0 | 5.5
constexpr int BATCH_OF_FEW = 16, ROWS_OF_FEW = 1024;

template <typename T> hipError_t launch(hipStream_t s, const PagedPlanArgs& a)
{
    Plan<T> p = {a};
    const long long entries = (a.table != a.tableOut ? (long long)a.batch * a.maxPages : 0) + (a.free != a.freeOut ? p.remain(a.pages) : 0);
    const bool rows = a.positions || a.slots, own = a.tokens <= ROWS_OF_ONE, few = a.tokens <= ROWS_OF_FEW && a.batch <= BATCH_OF_FEW;
    const int others = (int)std::min<long long>(few ? 1024 : 256, (entries + 4095) / 4096);
    if (few) hipLaunchKernelGGL((paged_plan_kernel<T, 256>), 1 + others, 256, 0, s, p, rows ? 1 : 0);
    else hipLaunchKernelGGL((paged_plan_kernel<T, 1024>), 1 + others, 1024, 0, s, p, rows && own ? 1 : 0);
    if (rows && !own) hipLaunchKernelGGL((paged_plan_rows_kernel<T>), std::min(a.batch, 65535), 256, 0, s, p);
    return hipGetLastError();
}

}  // namespace

hipError_t k_paged_plan(hipStream_t s, bool wide, const PagedPlanArgs& a) { return wide ? launch<double>(s, a) : launch<float>(s, a); }

}  // namespace mch
