// What the kernels of attention over a paged cache share (attn_paged.hip, attn_paged_pipe.hip).
#pragma once
#include "kernels.h"
#include "paged.h"

namespace mch {

struct PagedAttnArgs {
    PagedCache c;
    const void* q;
    void* y;
    float c2;   // scale * log2(e)
};

// place and last place of a tile's pieces (place -1: none), its first token and head, tokens, heads
struct ChunkJoin { int place, to, token, head, tokens, heads, pad[2]; };

struct ChunkArgs {
    float* part;      // partial results, [place in the list][2][128 {maximum, sum} | 128 rows of HSP]
    ChunkJoin* join;   // of every workgroup: the tile that it began and left to the next ones
    int few;          // sequences of at most this many rows a key head are another kernel's
    int shift, perTile, tileHeads, headTiles;
    int unit;         // shift of paged_units_before
    int pair;         // tiles of perTile tokens that a workgroup's tile stands for (the pipe kernel's are two of the chunk kernel's)
    const int* redo;  // chunk kernel: not null, workgroups 2 i and 2 i + 1 do what the pipe kernel's workgroup i left, if redo[i]
};

// what all lanes of a wavefront have alike, in scalar registers
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ PagedSpan uniform(const PagedSpan& s) { return PagedSpan{uniform(s.first), uniform(s.count), uniform(s.len)}; }
__device__ __forceinline__ PagedSpan span_at(const PagedCache& c, int b)
{
    return uniform(paged_span(c.starts[b], c.starts[b + 1], c.lens[b], c.tokens, c.maxPages * c.pageSize));
}

// over a wavefront, numbers up to PAGED_MOST: the sums up to and with the lane's own (a row of sixteen lanes, then the rows before it)
__device__ __forceinline__ int wave_scan(int x)
{
    x = paged_sum(x, __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false));   // row_shr 1, 2, 4, 8
    x = paged_sum(x, __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false));
    x = paged_sum(x, __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false));
    x = paged_sum(x, __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false));
    x = paged_sum(x, __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false));   // row_bcast 15 to rows 1 and 3
    return paged_sum(x, __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false));   // row_bcast 31 to rows 2 and 3
}
// over 256 threads, numbers up to PAGED_MOST: the sum of those before the thread's own (PAGED_MOST: that or more), and of all of them
__device__ __forceinline__ int block_scan(int v, int* sums, int* all)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int x = wave_scan(v), mine = __builtin_amdgcn_update_dpp(0, x, 0x138, 0xf, 0xf, false);   // wave_shr 1
    __syncthreads();
    if (lane == 63) sums[wave] = x;
    __syncthreads();
    int before = 0, sum = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        before = i < wave ? paged_sum(before, sums[i]) : before;
        sum = paged_sum(sum, sums[i]);
    }
    *all = sum;
    return paged_sum(before, mine);
}

// The chunk kernel's list: sequences, their key heads and head tiles, their tiles, in units of about 32 positions of a tile.  All 256 threads.
// Units a workgroup has at least: what a piece costs beside its blocks (its places, queries and partial results) is some of them.  us with 3 | 4 | 6 | 8: 8 new tokens
// over 727 positions, 32 heads on 4 of 128, 16 bits 19.4 | 21.1 | 22.2 | 23.5; 68 over 400 and 121 over 985, 28 heads on 4 of 96, fp32 over a 16-bit cache 41.6 | 37.8 | 40.7 | 42.6; 2 prompts
// of 958 over 978, 10 heads of 128, fp32 78.8 | 78.1 | 79.2 | 83.7.  With 16 and 32: 2 prompts of 1024, 12 heads of 64, fp32 63 and 99 for 50.
constexpr int CHUNK_LEAST = 4;
__device__ __forceinline__ int chunk_tiles(const PagedCache& c, const ChunkArgs& w, const PagedSpan& s)
{
    return (long long)s.count * (c.H / c.kvH) > w.few ? (s.count + w.perTile - 1) / w.perTile : 0;
}
__device__ __forceinline__ int chunk_work(const PagedCache& c, const ChunkArgs& w, const PagedSpan& s)   // of one key head and head tile
{
    return paged_units_before(max(s.len - s.count, 0), w.perTile, chunk_tiles(c, w, s), w.unit);
}
// the total, and where unit `begin(place)` of its runs is: sequence, its span, and the unit within it; place -1: nothing
struct ChunkStart { int total, place, b, local; PagedSpan sp; };
__device__ __forceinline__ ChunkStart chunk_start(const PagedCache& c, const ChunkArgs& w, int block, int most)
{
    __shared__ int sums[4], seq, first;
    __shared__ PagedSpan span;
    const int groups = c.kvH * w.headTiles, tid = threadIdx.x;
    auto span_of = [&](int b) {
        return b < c.batch ? paged_span(c.starts[b], c.starts[b + 1], c.lens[b], c.tokens, c.maxPages * c.pageSize) : PagedSpan{0, 0, 0};
    };
    ChunkStart r = {};
    PagedSpan mine = span_of(tid);
    int work = chunk_work(c, w, mine) * groups, at = block_scan(work, sums, &r.total), all = r.total;
    for (int b0 = 256; b0 < c.batch; b0 += 256) {
        int more;
        block_scan(chunk_work(c, w, span_of(b0 + tid)) * groups, sums, &more);
        r.total = paged_sum(r.total, more);
    }
    r.total = uniform(r.total);
    if (r.total >= PAGED_MOST) { r.place = -1; return r; }
    const PagedRuns runs(r.total, most, CHUNK_LEAST);
    r.place = paged_place(block, runs.W);
    if (r.place < 0) return r;
    const int lo = runs.begin(r.place);
    for (int b0 = 0, base = 0;;) {
        if (at <= lo && lo < at + work) { seq = b0 + tid; first = at; span = mine; }
        base += all;
        if (lo < base) break;
        if ((b0 += 256) >= c.batch) { r.place = -1; return r; }
        mine = span_of(b0 + tid);
        work = chunk_work(c, w, mine) * groups;
        at = base + block_scan(work, sums, &all);
    }
    __syncthreads();
    r.b = uniform(seq);
    r.local = uniform(lo - first);
    r.sp = uniform(span);
    return r;
}

// What workgroup `block` of the pipe kernel works on; b < 0: nothing
struct ChunkTile { int b, tile, kh, ht; };
__device__ __forceinline__ ChunkTile chunk_tile(const PagedCache& c, const ChunkArgs& w, unsigned block)
{
    __shared__ int sums[4], seq, tile;
    const int groups = c.kvH * w.headTiles, want = block / groups, group = block - want * groups, tid = threadIdx.x;
    if (tid == 0) { seq = -1; tile = 0; }
    for (int b0 = 0, base = 0; b0 < c.batch && base <= want; b0 += 256) {
        int tiles = 0, all;
        if (b0 + tid < c.batch) {
            const PagedSpan s = paged_span(c.starts[b0 + tid], c.starts[b0 + tid + 1], c.lens[b0 + tid], c.tokens, c.maxPages * c.pageSize);
            if ((long long)s.count * (c.H / c.kvH) > w.few) tiles = (s.count + w.perTile * w.pair - 1) / (w.perTile * w.pair);
        }
        const int at = base + block_scan(tiles, sums, &all);
        if (at <= want && want < at + tiles) { seq = b0 + tid; tile = tiles - 1 - (want - at); }   // those that see most come first
        base += all;
    }
    __syncthreads();
    return ChunkTile{uniform(seq), uniform(tile), group / w.headTiles, group % w.headTiles};
}

// Tiles take turns, one a CU at head size 128 and two at 64, and the last turn is seldom full: where the positions of a tile are done in pieces, each by a workgroup, more and
// shorter turns leave less of the chip idle, at the price of writing and reading a piece's sums (132 KB at 128).  Pieces: as many as make it shortest, counted in turns.  us, whole | in pieces, 32 heads on 8 of 128 behind 16384 positions: 144 tiles 408 | 333, 200
// (one piece: what finding that out costs) 411 | 424, 304 847 | 664, 384 851 | 770; behind 8000, 304 438 | 379, behind 4000 244 | 239; 368 tiles of heads of 64 511 | 467.
constexpr int PIECES = 4, PIECE_KEYS = 1024;   // at most, and keys from which on a piece of a tile is worth its sums
__host__ __device__ constexpr int turn_of(int hs) { return hs == 64 ? 512 : 256; }   // tiles of a turn
__host__ __device__ inline int pieces_of(int tiles, int hs)
{
    const int turn = turn_of(hs);
    if (tiles > (hs == 64 ? turn : 2 * turn)) return 1;   // (two workgroups a CU: those of a turn that is half full are faster)
    int best = 1;
    float least = (float)((tiles + turn - 1) / turn);
    for (int n = 2; n <= PIECES && tiles * n <= 4 * turn; n++) {
        const float cost = (float)((tiles * n + turn - 1) / turn) / n + 0.03f * n * tiles / turn;
        if (cost < least) { least = cost; best = n; }
    }
    return best;
}
// the tiles of a launch of the pipe kernel
__device__ __forceinline__ int chunk_tile_count(const PagedCache& c, const ChunkArgs& w)
{
    __shared__ int sums[4];
    const int tid = threadIdx.x;
    int total = 0;
    for (int b0 = 0; b0 < c.batch; b0 += 256) {
        int tiles = 0, all;
        if (b0 + tid < c.batch) {
            const PagedSpan s = paged_span(c.starts[b0 + tid], c.starts[b0 + tid + 1], c.lens[b0 + tid], c.tokens, c.maxPages * c.pageSize);
            if ((long long)s.count * (c.H / c.kvH) > w.few) tiles = (s.count + w.perTile * w.pair - 1) / (w.perTile * w.pair);
        }
        block_scan(tiles, sums, &all);
        total = paged_sum(total, all);
    }
    return uniform(min(total, PAGED_MOST / (c.kvH * w.headTiles)) * c.kvH * w.headTiles);
}

// Chunks in 16-bit storage, head size 64 or 128, in tiles of 256 rows (w.pair 2); redo[i]: tile i is left to the chunk kernel
hipError_t attn_paged_pipe_launch(hipStream_t s, const PagedAttnArgs& a, const ChunkArgs& w, int blocks, int* redo);
// The same with the positions of each tile in up to four pieces, where that fills the chip better; part: as many bytes as these say
size_t attn_paged_pieces_bytes(const PagedCache& c, int blocks);
hipError_t attn_paged_pieces_launch(hipStream_t s, const PagedAttnArgs& a, const ChunkArgs& w, int blocks, int* redo, void* part);

}  // namespace mch
