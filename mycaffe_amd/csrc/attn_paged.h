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

struct ChunkArgs {
    float* part;      // [split][tile][key head x head tile][128 {maximum, sum} | 128 rows of HSP]
    int few;          // sequences of at most this many rows a key head are another kernel's
    int shift, perTile, tileHeads, headTiles, splits;
    int pair;         // tiles of perTile tokens that a workgroup's tile stands for (the pipe kernel's are two of the chunk kernel's)
    const int* redo;  // chunk kernel: not null, workgroups 2 i and 2 i + 1 do what the pipe kernel's workgroup i left, if redo[i]
};

// over 256 threads: the sum of the numbers before the thread's own, and all of them
__device__ __forceinline__ int block_scan(int v, int* sums, int* all)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int x = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int y = __shfl_up(x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 63) sums[wave] = x;
    __syncthreads();
    int before = 0, sum = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        before += i < wave ? sums[i] : 0;
        sum += sums[i];
    }
    *all = sum;
    return before + x - v;
}

// What workgroup `block` of a launch works on; b < 0: nothing
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
    return ChunkTile{seq, tile, group / w.headTiles, group % w.headTiles};
}

// Chunks in 16-bit storage, head size 64 or 128, in tiles of 256 rows (w.pair 2); flags[i]: the tile of workgroup i is left to the chunk kernel
hipError_t attn_paged_pipe_launch(hipStream_t s, const PagedAttnArgs& a, const ChunkArgs& w, int blocks, int* flags);

}  // namespace mch
