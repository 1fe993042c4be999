// Attention over the pages of a cache for groups of sequences that share their first positions: the prefix is read, and its products made, once for all tokens of a group.
//
// For a token of a group whose prefix are the positions 0 .. P - 1, with softmax statistics m, l and sums o of weights times values over each of the two sets of positions,
//     (m0, l0, o0) over the prefix,  (m1, l1, o1) over its own positions P .. p:   y = (o0 2^(m0 - m) + o1 2^(m1 - m)) / (l0 2^(m0 - m) + l1 2^(m1 - m)),  m = max(m0, m1).
// The prefix sees the group's tokens, of all sequences, as rows of one product (chunk_run, split_run), none of them masked; what is behind it is attention over
// pages from position P on.  Both are entries of one list of work, and the sums of both, in fp32, meet in a launch behind.
//
// P: the whole pages of what is said to be shared, as far as they lie in front of every new token of the group.
//
// Many rows over a prefix are bound by the matrix cores, few rows behind it by reading the cache, so both kinds of work run side by side, in shares by what they cost.  What
// remains is the wait for memory at the begin and end of items, and three launches that depend on each other (the list, the work, the sums).  Measured: 64 tokens, 32 heads on 8 of 128 in
// 16 bits, behind 8192 shared and up to 512 positions of their own, 108 MB and 8.9 GFLOP, 59 us (6 + 45 + 7; 248 without sharing); 192 tokens, 12 heads of 64, behind three times 2048 and up to
// 700, 247 MB, 90 us; 24 sequences of 2 to 5 tokens, 12 heads on 4 of 64 in fp32 over 16 bits, behind 3000 and up to 300, 30.6 us.
#include <algorithm>

#include "attn_paged_run.h"

namespace mch {

namespace {

constexpr int PREFIX_ENTRIES = 4096, PREFIX_GROUPS = 1024;                          // entries of the list (groups and sequences), groups of a launch
constexpr int PREFIX_GRID = 512;                                                    // workgroups, two a CU: both kinds run side by side, as many of each as its list asks for

// tokens first .. first + count - 1, the first at position pos, over the positions from .. len - 1 of the block table's row (of a prefix: all of them, pos = len)
struct PrefixSpan { int first, count, len, from, pos, row, prefix, pad; };

struct PrefixWork {
    PrefixSpan* spans;            // groups, then sequences
    int2* at;                     // of every entry: units of split_run's and chunk_run's list in front of its own
    int2 *splitBegin, *chunkBegin;   // of every run: entry, unit in it
    int* groupOf;                 // of every sequence, -1: none
    int* totals;                  // units of split_run's and chunk_run's list, whether they could be counted, workgroups of chunk_run
    float *splitPart, *chunkPart, *sums;
    const float *groups, *shared;
    int nGroups, n;               // groups, entries
};

struct OfPrefixes {
    static constexpr bool SUMS = true;
    typedef PrefixSpan Span;
    PrefixWork w;
    struct Start { int b, local; };
    __device__ int count(const PagedCache&) const { return w.n; }
    __device__ Span span(const PagedCache&, int b) const { return w.spans[b]; }
    __device__ Span all_lanes(const PagedCache&, int b) const
    {
        const Span s = w.spans[b];
        return Span{uniform(s.first), uniform(s.count), uniform(s.len), uniform(s.from), uniform(s.pos), uniform(s.row), uniform(s.prefix), 0};
    }
    __device__ static int from_of(const Span& s) { return s.from; }
    __device__ static int pos_of(const Span& s) { return s.pos; }
    __device__ static int row_of(const Span& s, int) { return s.row; }
    __device__ static int grow_of(const Span& s, int perTile) { return s.prefix ? 0 : perTile; }
    // {maximum, sum of weights, -, -, sums} of a token's head, on its side
    __device__ float* sums_of(const PagedCache& c, const Span& s, int token, int head, int hsp) const
    {
        return w.sums + (((size_t)s.prefix * c.tokens + token) * c.H + head) * (hsp + 4);
    }
    __device__ int chunk_blocks() const { return uniform(w.totals[3]); }
    __device__ int split_total() const { return uniform(w.totals[0]); }
    __device__ int chunk_total() const { return uniform(w.totals[1]); }
    __device__ Start split_start(int run) const { return Start{uniform(w.splitBegin[run].x), uniform(w.splitBegin[run].y)}; }
    __device__ Start chunk_start(int run) const { return Start{uniform(w.chunkBegin[run].x), uniform(w.chunkBegin[run].y)}; }
};

// units of an entry, as the two runs count them
struct PrefixUnits {
    SplitArgs split;
    ChunkArgs chunk;
    int unit, kvH, G;
    int splitGrid;                // workgroups of split_run in a launch of its own; 0: those that chunk_run leaves
    float splitCost, chunkCost;   // of a unit
    __device__ int split_blocks(int chunks) const { return splitGrid ? splitGrid : PREFIX_GRID - chunks; }
    __device__ bool is_chunk(const PrefixSpan& s) const { return split.few && (long long)s.count * G > split.few; }
    __device__ int units(const PrefixSpan& s) const { const int n = s.len - s.from; return n <= max(split.one, unit) ? 1 : (n + unit - 1) / unit; }
    __device__ int split_work(const PrefixSpan& s) const { return is_chunk(s) ? 0 : (s.count + split.perTile - 1) / split.perTile * split.headTiles * kvH * units(s); }
    __device__ int before(const PrefixSpan& s) const { return max(min(s.pos, s.len) - s.from, 0); }
    __device__ int tiles_before(const PrefixSpan& s, int tiles) const { return paged_units_before(before(s), s.prefix ? 0 : chunk.perTile, tiles, chunk.unit); }
    __device__ int chunk_each(const PrefixSpan& s) const { return tiles_before(s, (s.count + chunk.perTile - 1) / chunk.perTile); }   // of a key head and head tile
    __device__ int chunk_work(const PrefixSpan& s) const { return is_chunk(s) ? chunk_each(s) * kvH * chunk.headTiles : 0; }
};

// The list: what is shared, whose tokens and positions every entry has, where every workgroup begins.  One workgroup, a thread an entry, few of them where
// there are few; what is read is read at once.
template <int THREADS, int ENTRIES, int GROUPS> __global__ __launch_bounds__(THREADS) void attn_prefix_plan_kernel(PagedCache c, PrefixWork w, PrefixUnits u)
{
    constexpr int WAVES = THREADS / 64;
    __shared__ int sBound[GROUPS + 1], sPrefix[GROUPS], sRow[GROUPS], sFirst[ENTRIES + 1], sSums[2][WAVES], sAt[2][ENTRIES];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, positions = c.maxPages * c.pageSize;
    const int said = tid < w.nGroups ? paged_int(w.shared[tid], 0, positions) : 0;
    // bounds of the groups, never decreasing: the largest so far
    int bound = tid < w.nGroups ? paged_int(w.groups[tid], 0, c.batch) : 0;
    const int end = tid == 0 ? paged_int(w.groups[w.nGroups], 0, c.batch) : 0;
    PagedSpan span = {0, 0, 0}, own = {0, 0, 0};   // of sequence tid, and of the thread's entry
    const int sequence = tid - w.nGroups;
    if (sequence >= 0 && sequence < c.batch) own = paged_span(c.starts[sequence], c.starts[sequence + 1], c.lens[sequence], c.tokens, positions);
    const int rows = tid == 0 ? paged_int(c.starts[c.batch], 0, c.tokens) : 0;
    if (tid < c.batch) span = paged_span(c.starts[tid], c.starts[tid + 1], c.lens[tid], c.tokens, positions);
    for (int o = 1; o < 64; o <<= 1) {
        const int y = __shfl_up(bound, o);
        bound = lane >= o ? max(bound, y) : bound;
    }
    if (lane == 63) sSums[0][wave] = bound;
    __syncthreads();
    for (int i = 0; i < wave; i++) bound = max(bound, sSums[0][i]);
    if (tid < w.nGroups) {
        sBound[tid] = bound;
        sPrefix[tid] = positions + 1;
        sRow[tid] = c.batch;
    }
    if (tid == w.nGroups - 1) sSums[1][0] = bound;
    __syncthreads();
    if (tid == 0) {
        sBound[w.nGroups] = max(sSums[1][0], end);
        sFirst[c.batch] = rows;
    }
    __syncthreads();
    // of sequence b its group, or -1; the least position of a group's new tokens, and the first sequence with any, whose pages are read (others need not have any more)
    auto group_of = [&](int b) -> int {
        if (b < sBound[0] || b >= sBound[w.nGroups]) return -1;
        int lo = 0, hi = w.nGroups;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (sBound[mid] <= b) lo = mid;
            else hi = mid;
        }
        return lo;
    };
    for (int b = tid; b < c.batch; b += THREADS) {
        const PagedSpan s = b == tid ? span : paged_span(c.starts[b], c.starts[b + 1], c.lens[b], c.tokens, positions);
        sFirst[b] = s.first;
        const int g = group_of(b);
        if (g >= 0 && s.count > 0) {
            atomicMin(&sPrefix[g], max(s.len - s.count, 0));
            atomicMin(&sRow[g], b);
        }
    }
    __syncthreads();
    if (tid < w.nGroups) sPrefix[tid] = sPrefix[tid] > positions ? 0 : min(sPrefix[tid], said) / c.pageSize * c.pageSize;
    __syncthreads();
    // ---- the entries, and the units in front of each ----
    int total[2] = {0, 0};
    for (int v0 = 0; v0 < w.n; v0 += THREADS) {
        const int v = v0 + tid;
        int work[2] = {0, 0}, at[2];
        if (v < w.n) {
            PrefixSpan s;
            if (v < w.nGroups) {
                const int first = sBound[v], prefix = sPrefix[v];
                s = PrefixSpan{sFirst[first], prefix > 0 ? max(sFirst[sBound[v + 1]] - sFirst[first], 0) : 0, prefix, 0, prefix, sRow[v], 1, 0};
            } else {
                const int b = v - w.nGroups, g = group_of(b), from = g >= 0 ? sPrefix[g] : 0;
                const PagedSpan x = v0 == 0 && w.nGroups <= THREADS && sequence >= 0 ? own : paged_span(c.starts[b], c.starts[b + 1], c.lens[b], c.tokens, positions);
                s = PrefixSpan{x.first, x.count, x.len, from, x.len - x.count, b, 0, 0};
                w.groupOf[b] = from > 0 ? g : -1;
            }
            w.spans[v] = s;
            work[0] = u.split_work(s);
            work[1] = u.chunk_work(s);
        }
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int x = wave_scan(work[i]);
            at[i] = __builtin_amdgcn_update_dpp(0, x, 0x138, 0xf, 0xf, false);   // wave_shr 1
            if (lane == 63) sSums[i][wave] = x;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 2; i++) {
            int before = total[i];
            for (int k = 0; k < WAVES; k++) {
                const int x = sSums[i][k];
                before = k < wave ? paged_sum(before, x) : before;
                total[i] = paged_sum(total[i], x);
            }
            at[i] = paged_sum(before, at[i]);
            if (v < w.n) sAt[i][v] = at[i];
        }
        if (v < w.n) w.at[v] = make_int2(at[0], at[1]);
        __syncthreads();
    }
    // workgroups of each kind, in eights
    const bool countable = total[0] < PAGED_MOST && total[1] < PAGED_MOST;
    const float cost[2] = {total[0] * u.splitCost, total[1] * u.chunkCost};
    // (more than half of them only for runs of 512 positions: every run leaves 128 rows of sums behind)
    const int most = max(PREFIX_GRID / 2, min(PREFIX_GRID - (total[0] ? 8 : 0), total[1] / 16));
    const int chunks = !total[1] ? 0 : u.splitGrid ? PREFIX_GRID : max(8, min((int)(PREFIX_GRID * cost[1] / (cost[0] + cost[1])), most) & ~7);
    if (tid == 0) {
        w.totals[0] = countable ? total[0] : 0;
        w.totals[1] = countable ? total[1] : 0;
        w.totals[2] = countable;
        w.totals[3] = chunks;
    }
    if (!countable) return;
    // ---- where every run begins ----
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const PagedRuns runs(total[i], i ? chunks : u.split_blocks(chunks), i ? CHUNK_LEAST : 1);
        for (int k = tid; k < runs.W; k += THREADS) {
            const int unit = runs.begin(k);
            int lo = 0, hi = w.n;
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (sAt[i][mid] <= unit) lo = mid;
                else hi = mid;
            }
            (i ? w.chunkBegin : w.splitBegin)[k] = make_int2(lo, unit - sAt[i][lo]);
        }
    }
}

// on every XCD (workgroup i is on XCD i % 8) the first workgroups have the tiles of many rows, which the matrix cores bound, the others the split of positions, which memory does
template <typename TQ, typename TC, int HSP> __global__ __launch_bounds__(256, 2) void attn_prefix_kernel(PagedAttnArgs a, ChunkArgs chunk, SplitArgs split, OfPrefixes list)
{
    __shared__ union { SplitShared<TQ, TC, HSP, OfPrefixes> split; ChunkShared<TQ, TC, HSP> chunk; } shared;
    const int chunks = list.chunk_blocks(), block = blockIdx.x;
    if (block < chunks) chunk_run<TQ, TC, HSP>(a, chunk, block, chunks, shared.chunk, list);
    else split_run<TQ, TC, HSP>(a, split, block - chunks, PREFIX_GRID - chunks, shared.split, list);
}
template <typename TQ, typename TC, int HSP> __global__ __launch_bounds__(256, HSP <= 64 ? 4 : HSP <= 128 ? 2 : 1) void attn_prefix_split_kernel(PagedAttnArgs a, SplitArgs split, OfPrefixes list)
{
    __shared__ SplitShared<TQ, TC, HSP, OfPrefixes> shared;
    split_run<TQ, TC, HSP>(a, split, blockIdx.x, gridDim.x, shared, list);
}
template <typename TQ, typename TC, int HSP> __global__ __launch_bounds__(256, 2) void attn_prefix_chunk_kernel(PagedAttnArgs a, ChunkArgs chunk, OfPrefixes list)
{
    __shared__ ChunkShared<TQ, TC, HSP> shared;
    const int chunks = list.chunk_blocks(), block = blockIdx.x;
    if (block < chunks) chunk_run<TQ, TC, HSP>(a, chunk, block, chunks, shared, list);
}

// The sums of both sides, and of the pieces of each, put together: a wavefront a head of a token, LANES lanes of it four values each, and as many pieces at a time as
// that leaves groups of lanes, DEEP times over.  A workgroup has four heads of the sequence's tokens, every gridDim.z-th one.  (What it takes is mostly one read
// behind the other: rows of the sequence, its entries, the pieces.)
template <typename TQ, int HSP> __global__ __launch_bounds__(256) void attn_prefix_join_kernel(PagedAttnArgs a, PrefixWork w, PrefixUnits u)
{
    constexpr int LANES = HSP / 4, WAYS = 64 / LANES, DEEP = WAYS == 4 ? 4 : 8;
    const PagedCache& c = a.c;
    const int b = blockIdx.x, h = blockIdx.y * 4 + (threadIdx.x >> 6), lane = threadIdx.x % LANES, way = (threadIdx.x & 63) / LANES;
    const int total0 = w.totals[0], total1 = w.totals[1], countable = w.totals[2], chunks = w.totals[3], g = w.groupOf[b];
    const PrefixSpan own = w.spans[w.nGroups + b];
    const int2 ownAt = w.at[w.nGroups + b];
    if (!countable || h >= c.H) return;
    const PrefixSpan front = w.spans[max(g, 0)];
    const int2 frontAt = w.at[max(g, 0)];
    const int kh = h / u.G, j = h - kh * u.G;
    for (int t0 = blockIdx.z; t0 < own.count; t0 += gridDim.z) {
        const int token = own.first + t0;
        // of each side the first piece and the number of pieces; where there is one, it is the row's own
        const float* base[2];
        int step[2], values[2], n[2] = {0, 0};
        auto side = [&](int i, const PrefixSpan& s, const int2& at) __attribute__((always_inline)) {
            const int t = token - s.first;
            if (t < 0 || t >= s.count) return;   // (starts that decrease)
            int from, to, row;
            if (u.is_chunk(s)) {
                const int tile = t / u.chunk.perTile, ht = j / u.chunk.tileHeads, before = at.y + (kh * u.chunk.headTiles + ht) * u.chunk_each(s);
                const PagedRuns runs(total1, chunks, CHUNK_LEAST);
                from = runs.of(before + u.tiles_before(s, tile));
                to = runs.of(before + u.tiles_before(s, tile + 1) - 1);
                row = (t - tile * u.chunk.perTile) * u.chunk.tileHeads + j - ht * u.chunk.tileHeads;
                step[i] = 2 * 128 * (HSP + 2);
                base[i] = w.chunkPart + (size_t)from * step[i] + 2 * row;
                values[i] = 256 - 2 * row + row * HSP;
            } else {
                const int ht = j / u.split.tileHeads, units = u.units(s), tile = t / u.split.perTile, first = at.x + ((tile * u.split.headTiles + ht) * u.kvH + kh) * units;
                const PagedRuns runs(total0, u.split_blocks(chunks), 1);
                from = runs.of(first);
                to = runs.of(first + units - 1);
                row = (t - tile * u.split.perTile) * u.split.tileHeads + j - ht * u.split.tileHeads;
                step[i] = 2 * 16 * (HSP + 2);
                base[i] = w.splitPart + (size_t)from * step[i] + 2 * row;
                values[i] = 32 - 2 * row + row * HSP;
            }
            n[i] = to - from + 1;
            if (n[i] == 1) {
                base[i] = w.sums + (((size_t)s.prefix * c.tokens + token) * c.H + h) * (HSP + 4);
                values[i] = 4;
            }
        };
        side(0, own, ownAt);
        if (g >= 0) side(1, front, frontAt);
        float M = -INFINITY, L = 0.f;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
        const int pieces = n[0] + n[1];
        for (int z0 = 0; z0 < pieces; z0 += DEEP * WAYS) {
            float2 ml[DEEP];
            float4 v[DEEP];
#pragma unroll
            for (int d = 0; d < DEEP; d++) {
                const int z = min(z0 + d * WAYS + way, pieces - 1), i = z >= n[0], k = i ? z - n[0] : z, stride = i ? step[1] : step[0];
                // of the workgroup that began the tile the second part, of the others the first
                const float* from = (i ? base[1] : base[0]) + (size_t)k * stride + (k == 0 && (i ? n[1] : n[0]) > 1 ? stride / 2 : 0);
                ml[d] = *(const float2*)from;
                v[d] = *(const float4*)(from + (i ? values[1] : values[0]) + 4 * lane);
            }
            float Mn = M;
#pragma unroll
            for (int d = 0; d < DEEP; d++) Mn = z0 + d * WAYS + way < pieces ? fmaxf(Mn, ml[d].x) : Mn;
            const float f0 = weight_of(M, Mn);
            L *= f0;
            x.x *= f0; x.y *= f0; x.z *= f0; x.w *= f0;
#pragma unroll
            for (int d = 0; d < DEEP; d++) {
                if (z0 + d * WAYS + way >= pieces) break;
                const float f = weight_of(ml[d].x, Mn);
                L += ml[d].y * f;
                x.x += v[d].x * f; x.y += v[d].y * f; x.z += v[d].z * f; x.w += v[d].w * f;
            }
            M = Mn;
        }
        // the groups of lanes meet
        float m = M;
#pragma unroll
        for (int o = LANES; o < 64; o <<= 1) m = fmaxf(m, __shfl_xor(m, o));
        const float f = weight_of(M, m);
        L *= f;
        x.x *= f; x.y *= f; x.z *= f; x.w *= f;
#pragma unroll
        for (int o = LANES; o < 64; o <<= 1) {
            L += __shfl_xor(L, o);
            x.x += __shfl_xor(x.x, o); x.y += __shfl_xor(x.y, o); x.z += __shfl_xor(x.z, o); x.w += __shfl_xor(x.w, o);
        }
        const int d = 4 * lane;
        if (way == 0 && d < c.hs) {
            const float inv = 1.f / L;
            if (m == -INFINITY) x = make_float4(0.f, 0.f, 0.f, 0.f);
            else { x.x *= inv; x.y *= inv; x.z *= inv; x.w *= inv; }
            FlashTraits<TQ>::store4((TQ*)a.y + ((size_t)token * c.H + h) * c.hs + d, x.x, x.y, x.z, x.w);
        }
    }
}

// what of the scratch memory is whose, in bytes
struct PrefixPlan {
    PrefixUnits u;
    size_t spans, at, splitBegin, chunkBegin, groupOf, totals, splitPart, chunkPart, sums, bytes;
    bool chunks;
    double splitUnits, chunkUnits;   // no more than these
};
int padded(const PagedCache& c) { return c.hs <= 64 ? 64 : c.hs <= 128 ? 128 : 256; }
PrefixPlan prefix_plan(const PagedCache& c, DType dt, int groups, int maxNew)
{
    PrefixPlan p = {};
    const int G = c.H / c.kvH, n = groups + c.batch;
    // Single tokens of heads that share no key heads leave little for the matrix cores, and at head sizes up to 64 four workgroups of split_run fit a CU where two of both kinds
    // do: a launch for each.  12 heads of 64, 16 bits, 192 tokens behind three times 2048 and up to 700 positions 80 us for 87, up to 2000 168 for 220, 96 behind 512 and up to 700 53
    // for 53 (the other way 45 for 40 with nothing behind the prefix); 24 heads on 3 the other way, 35 for 27, 12 heads and 8 tokens each 51 for 45.
    if (padded(c) == 64 && prefix_rows(c.tokens, c.batch, maxNew) * G <= (long long)c.batch * 5 / 4) p.u.splitGrid = 2 * PREFIX_GRID;
    p.chunks = c.hs <= 128;
    p.u.kvH = c.kvH;
    p.u.G = G;
    p.u.unit = 4 * 16 * (c.ct == F32 ? 1 : 2);
    p.u.split.shift = p.u.chunk.shift = (c.pageSize & (c.pageSize - 1)) == 0 ? __builtin_ctz(c.pageSize) : -1;
    p.u.split.few = p.u.chunk.few = p.chunks ? 16 : 0;
    p.u.split.headTiles = (G + 15) / 16;
    p.u.split.tileHeads = (G + p.u.split.headTiles - 1) / p.u.split.headTiles;
    p.u.split.perTile = 16 / p.u.split.tileHeads;
    p.u.split.one = (long long)n * c.kvH * p.u.split.headTiles < PREFIX_GRID / 2 ? 2 * p.u.unit : 0;
    p.u.chunk.headTiles = (G + 127) / 128;
    p.u.chunk.tileHeads = (G + p.u.chunk.headTiles - 1) / p.u.chunk.headTiles;
    p.u.chunk.perTile = 128 / p.u.chunk.tileHeads;
    p.u.chunk.pair = 1;
    // ns a workgroup of two a CU: 2 us and 10 bytes a ns for positions read; 32 positions of 128 rows, or 1 << unit as many, 1.2 us, or 2000 products and sums a ns, six of
    // them one in fp32 (three over a 16-bit cache), and of a weight's two parts two one in 16 bits
    const float parts = dt == BF16 ? 1.5f : c.ct == BF16 ? 3 : 6;
    p.u.splitCost = 2000.f + p.u.unit * (float)c.hs * 2 * (c.ct == F32 ? 4 : 2) / 10.f;
    // lists are counted in 32 bits; every token is in two entries
    const double positions = c.maxPages * (double)c.pageSize, tokens = c.tokens;
    p.splitUnits = (double)c.kvH * p.u.split.headTiles * (p.chunks ? n : 2 * tokens / p.u.split.perTile + n) * (positions / p.u.unit + 1);
    const double tiles = (2 * tokens / p.u.chunk.perTile + n) * c.kvH * p.u.chunk.headTiles;
    while (p.chunkUnits = tiles * ((std::max(tokens, positions) + 128) / (32 << p.u.chunk.unit) + 2), p.u.chunk.unit < 20 && p.chunkUnits > 1e9) p.u.chunk.unit++;
    p.u.chunkCost = (1 << p.u.chunk.unit) * std::max(1200.f, 32.f * 128 * padded(c) * 4 * parts / 2000.f);
    size_t bytes = 0;
    auto take = [&](size_t n) { const size_t at = bytes; bytes += (n + 255) & ~(size_t)255; return at; };
    p.spans = take(n * sizeof(PrefixSpan));
    p.at = take(n * sizeof(int2));
    const int splits = std::max(PREFIX_GRID, p.u.splitGrid);
    p.splitBegin = take(splits * sizeof(int2));
    p.chunkBegin = take(PREFIX_GRID * sizeof(int2));
    p.groupOf = take(c.batch * sizeof(int));
    p.totals = take(4 * sizeof(int));
    p.splitPart = take((size_t)splits * 2 * 16 * (padded(c) + 2) * sizeof(float));
    p.chunkPart = take(p.chunks ? (size_t)PREFIX_GRID * 2 * 128 * (padded(c) + 2) * sizeof(float) : 0);
    p.sums = take((size_t)2 * c.tokens * c.H * (padded(c) + 4) * sizeof(float));
    p.bytes = bytes;
    return p;
}
inline bool at16(const void* p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace

// When what is shared is worth it (prefix_pays): with many rows a sequence the
// kernels of attention over pages have whole tiles of one sequence.  us, over pages | shared, 16 bits, heads of 128, single tokens with up to 300 positions of their own:
//   32 heads on 8, 16 sequences behind 1024 (88 MB) 21.9 | 25.1, 64 (352 MB) 48.4 | 36.7; behind 4096, 8 (145 MB) 29.1 | 27.7, 64 132 | 44;
//   16 on one, 16 behind 1024 (11 MB) 18.6 | 27.0, behind 4096 (36 MB) 40.2 | 30.1; 64 on one, 64 behind 1024 (44 MB) 40.9 | 37.7, behind 4096 78 | 62, behind 12000 190 | 97;
// in fp32 over 16 bits, 12 heads on 4 of 64, behind 1024, 24 (33 MB) 20.3 | 24.7, 96 (132 MB) 41.5 | 31.5, behind 4096 8 (36 MB) 22.2 | 26.0.
// By rows a sequence, 16 sequences, 16 bits: 32 heads on 8 behind 2048 and behind 16384, 18 52 | 42 and 181 | 100, 39 43 | 60 and 167 | 136, 81 51 | 93 and 182 | 265, 164 67 | 126 and 295 | 481; 8 on
// 8 behind 4096, 41 61 | 61, 82 71 | 99; fp32 behind 2048, 29 40 | 33, 61 38 | 46.
// What the host cannot know is what the tables hold: 64 sequences of 32 heads on 8 with 256 shared positions and up to 300 others share too, 44 us for 27.
constexpr size_t PREFIX_SCRATCH = 1ull << 30;   // sums of every row on both sides: 4096 tokens of 32 heads of 128 take 138 MB

size_t attn_prefix_workspace_bytes(const PagedCache& c, DType dt, const void* q, const void* y, int groups, int maxNew)
{
    const int e = dt == BF16 || c.ct == BF16 ? 8 : 4;
    const bool pieces = c.hs % e == 0 && c.sP % e == 0 && c.sH % e == 0 && c.sT % e == 0 && at16(c.k) && at16(c.v) && at16(q) && at16(y);
    const double bytes = (double)c.batch * c.maxPages * c.pageSize * c.kvH * c.hs * 2 * (c.ct == F32 ? 4 : 2);
    if (!pieces || groups > PREFIX_GROUPS || groups + c.batch > PREFIX_ENTRIES ||
        !prefix_pays(prefix_rows(c.tokens, c.batch, maxNew), c.batch, c.H / c.kvH, (long long)c.maxPages * c.pageSize, bytes, dt == F32)) return 0;
    const PrefixPlan p = prefix_plan(c, dt, groups, maxNew);
    return p.splitUnits < 1e9 && p.chunkUnits <= 1e9 && p.bytes <= PREFIX_SCRATCH ? p.bytes : 0;
}

hipError_t k_attn_prefix(hipStream_t s, DType dt, const PagedCache& c, const void* q, void* y, float scale, int groups, const float* bounds, const float* shared, int maxNew, void* workspace)
{
    PrefixPlan p = prefix_plan(c, dt, groups, maxNew);
    char* ws = (char*)workspace;
    PrefixWork w = {(PrefixSpan*)(ws + p.spans), (int2*)(ws + p.at), (int2*)(ws + p.splitBegin), (int2*)(ws + p.chunkBegin), (int*)(ws + p.groupOf), (int*)(ws + p.totals),
                    (float*)(ws + p.splitPart), (float*)(ws + p.chunkPart), (float*)(ws + p.sums), bounds, shared, groups, groups + c.batch};
    PagedAttnArgs a = {};
    a.c = c; a.q = q; a.y = y; a.c2 = scale * 1.44269504088896340736f;
    p.u.split.part = w.splitPart;
    p.u.chunk.part = w.chunkPart;
    if (w.n <= 256) hipLaunchKernelGGL((attn_prefix_plan_kernel<256, 256, 256>), 1, 256, 0, s, c, w, p.u);
    else hipLaunchKernelGGL((attn_prefix_plan_kernel<1024, PREFIX_ENTRIES, PREFIX_GROUPS>), 1, 1024, 0, s, c, w, p.u);
    const dim3 join(c.batch, (c.H + 3) / 4, std::min(64, (int)((prefix_rows(c.tokens, c.batch, maxNew) + c.batch - 1) / c.batch)));
    auto go = [&](auto type, auto ctype) {
        typedef decltype(type) T_;
        typedef decltype(ctype) TC_;
        auto sized = [&](auto size) {
            constexpr int HSP = decltype(size)::value;
            if (HSP == 64 && p.u.splitGrid) {
                if constexpr (HSP == 64) {
                    hipLaunchKernelGGL((attn_prefix_split_kernel<T_, TC_, HSP>), p.u.splitGrid, 256, 0, s, a, p.u.split, OfPrefixes{w});
                    hipLaunchKernelGGL((attn_prefix_chunk_kernel<T_, TC_, HSP>), PREFIX_GRID, 256, 0, s, a, p.u.chunk, OfPrefixes{w});
                }
            } else if constexpr (HSP <= 128) hipLaunchKernelGGL((attn_prefix_kernel<T_, TC_, HSP>), PREFIX_GRID, 256, 0, s, a, p.u.chunk, p.u.split, OfPrefixes{w});
            else hipLaunchKernelGGL((attn_prefix_split_kernel<T_, TC_, HSP>), PREFIX_GRID, 256, 0, s, a, p.u.split, OfPrefixes{w});
            hipLaunchKernelGGL((attn_prefix_join_kernel<T_, HSP>), join, 256, 0, s, a, w, p.u);
        };
        if (c.hs <= 64) sized(std::integral_constant<int, 64>{});
        else if (c.hs <= 128) sized(std::integral_constant<int, 128>{});
        else sized(std::integral_constant<int, 256>{});
        return hipGetLastError();
    };
    if (dt == F32) return c.ct == F32 ? go(float(), float()) : go(float(), bf16_t());
    return go(bf16_t(), bf16_t());
}

}  // namespace mch
