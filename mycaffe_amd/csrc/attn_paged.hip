// Attention of the new tokens of many sequences, one token or a chunk each, over keys and values in the pages of a cache.
//
// Token j of the n new ones of a sequence of len cached positions (the new ones last) is at position p = len - n + j:
//     y = sum over the positions t <= p whose page is given of softmax(scale q . k_t) v_t,   0 where there is none.
// What lies in positions that a token does not see (behind its own, behind the sequence, in pages not given) has no say, whatever it is; scores
// that are all -inf have no weights (0 / 0).
// Softmax statistics and sums are held in fp32; y is rounded once.
#include <algorithm>
#include <type_traits>

#include "attn_paged_run.h"
#include "kernels.h"
#include "lane_ops.h"
#include "paged.h"

namespace mch {

namespace {


// Any head size up to 256, any strides and addresses, no workspace: a workgroup has one token's head, a group of LPH lanes of its WAVES wavefronts
// every (64 WAVES / LPH)-th position, V values a lane, value by value in runs of LPH; ANY_DEEP positions' reads are under way together.  What
// bounds it is waiting for them, and every head reads its keys for itself.  Sixteen wavefronts where there are few tokens' heads, four else (us: one token over
// 1000 positions, 6 heads of 198, fp32 56 | 134, sixteen of them 69 | 191; 64 tokens over up to 60, 12 heads of 46, 16.1 | 7.1; chunks of 167 over 240, 297 over 593 and 137 over 157 and one token over 375, 6 heads of 46, 97 | 56).
constexpr int ANY_DEEP = 4;
template <typename T, typename TC, int V, int LPH, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void attn_paged_any_kernel(PagedAttnArgs a)
{
    constexpr int GROUPS = 64 / LPH, STEP = WAVES * GROUPS;
    __shared__ float sM[WAVES], sL[WAVES], sAcc[WAVES][LPH * V];
    __shared__ int sSeen[WAVES];
    const PagedCache& c = a.c;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, d0 = lane % LPH;
    const int token = blockIdx.z * gridDim.x + blockIdx.x, h = blockIdx.y;
    if (token >= c.tokens) return;
    const int b = sequence_of(c.starts, c.batch, c.tokens, token);
    if (b < 0) return;
    const PagedSpan sp = paged_span(c.starts[b], c.starts[b + 1], c.lens[b], c.tokens, c.maxPages * c.pageSize);
    if (token >= sp.first + sp.count) return;   // a row behind the last sequence
    const int last = sp.len - sp.count + (token - sp.first), kh = h / (c.H / c.kvH);
    const T* q = (const T*)a.q + ((size_t)token * c.H + h) * c.hs;
    float qv[V], acc[V], m = -INFINITY, l = 0.f;
    int at_d[V];
    bool seen = false;
#pragma unroll
    for (int i = 0; i < V; i++) {
        at_d[i] = min(d0 + LPH * i, c.hs - 1);
        qv[i] = d0 + LPH * i < c.hs ? value_of<T>(q[d0 + LPH * i]) : 0.f;
        acc[i] = 0.f;
    }
    for (int t0 = wave * GROUPS + lane / LPH; t0 <= last; t0 += ANY_DEEP * STEP) {
        TC k[ANY_DEEP][V], v[ANY_DEEP][V];
        bool given[ANY_DEEP];
#pragma unroll
        for (int j = 0; j < ANY_DEEP; j++) {
            const int t = t0 + j * STEP, entry = min(t, last) / c.pageSize, page = paged_page(c.table[(size_t)b * c.maxPages + entry], c.pages);
            given[j] = page >= 0 && t <= last;
            // what is not there: the cache's first values, left out below
            const long long at = given[j] ? page * c.sP + kh * c.sH + (t - entry * c.pageSize) * c.sT : 0;
#pragma unroll
            for (int i = 0; i < V; i++) {
                k[j][i] = ((const TC*)c.k)[at + at_d[i]];
                v[j][i] = ((const TC*)c.v)[at + at_d[i]];
            }
        }
#pragma unroll
        for (int j = 0; j < ANY_DEEP; j++) {
            float dot = 0.f;
#pragma unroll
            for (int i = 0; i < V; i++) dot += d0 + LPH * i < c.hs ? qv[i] * value_of<TC>(k[j][i]) : 0.f;
            dot = group_sum<LPH>(dot) * a.c2;
            if (!given[j]) continue;
            seen = true;
            const float mn = fmaxf(m, dot), ref = mn > -INFINITY ? mn : 0.f, f = exp2f(m - ref), w = exp2f(dot - ref);
            m = mn;
            l = l * f + w;
#pragma unroll
            for (int i = 0; i < V; i++) acc[i] = acc[i] * f + (d0 + LPH * i < c.hs ? w * value_of<TC>(v[j][i]) : 0.f);
        }
    }
    // the groups' sums meet, then the wavefronts'; one without positions has weight 0
    float M = m;
#pragma unroll
    for (int o = LPH; o < 64; o <<= 1) M = fmaxf(M, __shfl_xor(M, o));
    const float f = exp2f(m - (M > -INFINITY ? M : 0.f));
    seen = __any(seen);
    l *= f;
#pragma unroll
    for (int o = LPH; o < 64; o <<= 1) l += __shfl_xor(l, o);
#pragma unroll
    for (int i = 0; i < V; i++) {
        float s = acc[i] * f;
#pragma unroll
        for (int o = LPH; o < 64; o <<= 1) s += __shfl_xor(s, o);
        if (lane < LPH) sAcc[wave][d0 + LPH * i] = s;
    }
    if (lane == 0) { sM[wave] = M; sL[wave] = l; sSeen[wave] = seen; }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < WAVES; i++) {
        M = fmaxf(M, sM[i]);
        seen = seen || sSeen[i];
    }
    T* y = (T*)a.y + ((size_t)token * c.H + h) * c.hs;
    for (int d = threadIdx.x; d < c.hs; d += 64 * WAVES) {
        float x = 0.f, n = 0.f;
#pragma unroll
        for (int i = 0; i < WAVES; i++) {
            const float g = exp2f(sM[i] - (M > -INFINITY ? M : 0.f));
            x += sSeen[i] ? sAcc[i][d] * g : 0.f;
            n += sSeen[i] ? sL[i] * g : 0.f;
        }
        y[d] = stored<T>(seen ? x / n : 0.f);
    }
}


// single tokens and other short ones: the split of positions by itself
template <typename TQ, typename TC, int HSP>
__global__ __launch_bounds__(256, HSP <= 128 ? 2 : 1) void attn_paged_split_kernel(PagedAttnArgs a, SplitArgs w)
{
    __shared__ SplitShared<TQ, TC, HSP> shared;
    split_run<TQ, TC, HSP>(a, w, blockIdx.x, gridDim.x, shared, OfSequences());
}
// chunks, and the short ones among them: the first `chunks` workgroups have the chunks' list, the others the split's (us, two launches | one, the split behind | in front: a step
// of chunks and single tokens in fp32 72.4 | 64.3 | 67.2, chunks alone 47.6 | 43.7 | 45.1)
template <typename TQ, typename TC, int HSP>
__global__ __launch_bounds__(256, 2) void attn_paged_chunk_kernel(PagedAttnArgs a, ChunkArgs w, SplitArgs few, int chunks)
{
    __shared__ union { SplitShared<TQ, TC, HSP> split; ChunkShared<TQ, TC, HSP> chunk; } shared;
    if ((int)blockIdx.x < chunks) chunk_run<TQ, TC, HSP>(a, w, blockIdx.x, chunks, shared.chunk, OfSequences());
    else split_run<TQ, TC, HSP>(a, few, blockIdx.x - chunks, gridDim.x - chunks, shared.split, OfSequences());
}

// Tiles that a run ended in put together, 16 rows a workgroup, 16 lanes a row, from what the workgroup that began one has written down.
// A launch of its own: a tile has up to 64 KB a piece, which one workgroup takes longer to collect (7 pieces of 128 rows of 128: 100 us) than
// all of them to start anew.
template <typename TQ, int HSP>
__global__ __launch_bounds__(256) void attn_paged_join_kernel(PagedAttnArgs a, ChunkArgs w)
{
    constexpr int PART = 128 * (HSP + 2), LANES = 16, N = HSP / (4 * LANES);
    const PagedCache& c = a.c;
    const ChunkJoin t = w.join[blockIdx.x];
    const int row = blockIdx.y * 16 + threadIdx.x / LANES, token = row / w.tileHeads, head = row - token * w.tileHeads;
    if (t.place < 0 || token >= t.tokens || head >= t.heads) return;
    // piece z of the tile; eight of them in flight, past the last one that again with no weight
    auto part_of = [&](int z) { return w.part + ((size_t)min(z, t.to) * 2 + (z == t.place ? 1 : 0)) * PART; };
    float M = -INFINITY, L = 0.f;
    float4 x[N];
#pragma unroll
    for (int i = 0; i < N; i++) x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    constexpr int DEEP = 8;
    for (int z0 = t.place; z0 <= t.to; z0 += DEEP) {
        float2 ml[DEEP];
        float4 v[DEEP][N];
#pragma unroll
        for (int j = 0; j < DEEP; j++) {
            const float* from = part_of(z0 + j);
            ml[j] = *(const float2*)(from + 2 * row);
#pragma unroll
            for (int i = 0; i < N; i++) v[j][i] = *(const float4*)(from + 256 + row * HSP + 4 * LANES * i + 4 * (threadIdx.x % LANES));
        }
        float Mn = M;
#pragma unroll
        for (int j = 0; j < DEEP; j++) Mn = z0 + j <= t.to ? fmaxf(Mn, ml[j].x) : Mn;
        const float f0 = weight_of(M, Mn);
        L *= f0;
#pragma unroll
        for (int i = 0; i < N; i++) { x[i].x *= f0; x[i].y *= f0; x[i].z *= f0; x[i].w *= f0; }
#pragma unroll
        for (int j = 0; j < DEEP; j++) {
            if (z0 + j > t.to) break;
            const float f = weight_of(ml[j].x, Mn);
            L += ml[j].y * f;
#pragma unroll
            for (int i = 0; i < N; i++) { x[i].x += v[j][i].x * f; x[i].y += v[j][i].y * f; x[i].z += v[j][i].z * f; x[i].w += v[j][i].w * f; }
        }
        M = Mn;
    }
    TQ* y = (TQ*)a.y + ((size_t)(t.token + token) * c.H + t.head + head) * c.hs;
    const float inv = 1.f / L;
#pragma unroll
    for (int i = 0; i < N; i++) {
        const int d = 4 * LANES * i + 4 * (threadIdx.x % LANES);
        if (d >= c.hs) continue;
        if (M == -INFINITY) x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        else { x[i].x *= inv; x[i].y *= inv; x[i].z *= inv; x[i].w *= inv; }
        FlashTraits<TQ>::store4(y + d, x[i].x, x[i].y, x[i].z, x[i].w);
    }
}

constexpr int SPLIT_GRID = 512;   // two workgroups a CU; of heads of more than 128, one (64 tokens over 4096 positions, 2 key heads of 256, 16 bits: 103 us, with 512 112)
constexpr int ANY_MANY = 512;     // tokens' heads from which on the plain kernel has four wavefronts for one

inline bool at16(const void* p) { return ((uintptr_t)p & 15) == 0; }
// rows and cache in pieces of 16 bytes
inline bool in_pieces(const PagedCache& c, DType dt, const void* q, const void* y)
{
    const int e = dt == BF16 || c.ct == BF16 ? 8 : 4;
    return c.hs % e == 0 && c.sP % e == 0 && c.sH % e == 0 && c.sT % e == 0 && at16(c.k) && at16(c.v) && at16(q) && at16(y);
}

}  // namespace

// Rows of a key head up to which a sequence's positions are what is split, beyond which its rows are: one 16-row tile.  Two of them read the cache
// twice (us, two kernels, 32 heads on 8 key heads of 128, 4096 positions, 16-bit storage: 4 sequences of 8 new tokens, 32 rows, 41 | 36; 8 of 16, 64 rows, 84 | 61).
constexpr int FEW_ROWS = 16;
// Whole tiles of 256 rows from which on the pipe kernel takes a launch (it does not split them): half as many as CUs at head size 128, a workgroup
// a CU, three quarters at 64, two a CU.  us, chunk kernel | pipe: heads of 128, 64 tiles 210 | 401, 128 225 | 217, 256 300 | 251; heads of 64, 128 160 | 163,
// 168 39 | 45, 192 108 | 93 and 194 | 166, 384 54 | 47.
constexpr int PIPE_TILES_128 = 128, PIPE_TILES_64 = 192;
constexpr int CHUNK_ROWS = 128, CHUNK_GRID = 512;   // two workgroups a CU

// how a launch of the chunk kernels looks: what it takes from the host are the numbers of tokens and sequences alone
struct ChunkPlan { int headTiles, tileHeads, perTile, grid, unit, pipe; double units; };   // pipe: workgroups of the pipe kernel, 0 without it; units: no more than these
static ChunkPlan chunk_plan(const PagedCache& c, DType dt)
{
    const int G = c.H / c.kvH;
    ChunkPlan p;
    p.headTiles = (G + CHUNK_ROWS - 1) / CHUNK_ROWS;
    p.tileHeads = (G + p.headTiles - 1) / p.headTiles;
    p.perTile = CHUNK_ROWS / p.tileHeads;
    // every sequence may end inside a tile; those that have tiles have more than FEW_ROWS rows
    const long long having = std::min<long long>(c.batch, (long long)c.tokens * G / (FEW_ROWS + 1)), groups = (long long)c.kvH * p.headTiles;
    const long long whole = (long long)c.tokens / (2 * p.perTile) * groups, pipe = whole + having * groups;
    p.pipe = 0;
    if (dt == BF16 && ((c.hs == 128 && whole >= PIPE_TILES_128) || (c.hs == 64 && whole >= PIPE_TILES_64)) && (long long)c.tokens * G >= 256ll * c.batch && pipe < 1 << 22 &&
        ((c.pages - 1) * c.sP + (c.pageSize - 1) * c.sT) >> 3 < 0xffffffffll)
        p.pipe = (int)pipe;
    // the list is counted in 32 bits
    const double tiles = (double)(c.tokens / p.perTile + having) * groups, positions = std::max((double)c.tokens, c.maxPages * (double)c.pageSize) + CHUNK_ROWS;
    p.unit = 0;
    while (p.units = tiles * (positions / (32 << p.unit) + 2), p.unit < 20 && p.units > 1e9) p.unit++;
    p.grid = (int)std::min<double>(CHUNK_GRID, std::max(1.0, p.units / CHUNK_LEAST));
    return p;
}
static int padded_size(const PagedCache& c) { return c.hs <= 64 ? 64 : c.hs <= 128 ? 128 : 256; }

// the split kernel's partial results, and behind them the chunk kernel's or the pipe kernel's flags
static size_t split_bytes(const PagedCache& c) { return (size_t)SPLIT_GRID * 2 * 16 * (padded_size(c) + 2) * sizeof(float); }

// Whether a launch of the pipe kernel may have its tiles in pieces: at about as many tiles as there are if the last one of every sequence is half full, and over long tables
static bool in_turns(const PagedCache& c, DType dt)
{
    const ChunkPlan p = chunk_plan(c, dt);
    const int about = (int)std::min<long long>(((long long)c.tokens / (2 * p.perTile) * c.kvH * p.headTiles + p.pipe) / 2, 1 << 16);
    bool some = false;
    for (int tiles = about - about / 10; tiles <= about + about / 10; tiles++) some = some || pieces_of(tiles, c.hs) > 1;
    return p.pipe && some && c.maxPages * c.pageSize >= 6144;
}

size_t attn_paged_workspace_bytes(const PagedCache& c, DType dt, bool pieces)
{
    const ChunkPlan p = chunk_plan(c, dt);
    const bool chunks = c.hs <= 128 && (long long)c.tokens * (c.H / c.kvH) > FEW_ROWS;
    if (pieces && (!chunks || !in_turns(c, dt))) return 0;
    const size_t chunk = !chunks ? 0 : p.pipe ? ((size_t)p.pipe * sizeof(int) + 255 & ~(size_t)255) + (pieces ? attn_paged_pieces_bytes(c, p.pipe) : 0) : (size_t)p.grid * (2 * CHUNK_ROWS * (padded_size(c) + 2) * sizeof(float) + sizeof(ChunkJoin));
    return split_bytes(c) + chunk;
}
size_t attn_paged_tickets() { return SPLIT_GRID; }

hipError_t k_attn_paged(hipStream_t s, DType dt, const PagedCache& c, const void* q, void* y, float scale, int maxNew, void* workspace, int* tickets, bool pieces)
{
    PagedAttnArgs a = {};
    a.c = c; a.q = q; a.y = y; a.c2 = scale * 1.44269504088896340736f;
    auto go = [&](auto type, auto ctype) {
        typedef decltype(type) T_;
        typedef decltype(ctype) TC_;
        const int G = c.H / c.kvH;
        SplitArgs w = {};
        w.part = (float*)workspace;
        w.tickets = tickets;
        w.shift = (c.pageSize & (c.pageSize - 1)) == 0 ? __builtin_ctz(c.pageSize) : -1;
        w.headTiles = (G + 15) / 16;
        w.tileHeads = (G + w.headTiles - 1) / w.headTiles;
        w.perTile = 16 / w.tileHeads;
        const int most = maxNew > 0 ? std::min(maxNew, c.tokens) : c.tokens;
        // Steps of single tokens with few others among them are the split's as a whole, up to a quarter more tokens than sequences: it reads the cache of a longer sequence once for
        // 16 rows, and the chunk kernel's launch is longer by its registers, its list and the launch behind.  us, chunk kernel | split, one chunk of 1 + x times the sequences' number among
        // single tokens, 32 heads on 8 of 128 in 16 bits: x 1/4 over 2000 positions, 16 sequences 38.7 | 32.4, 64 92 | 73, 256 126 | 107; over 8000, 64 312 | 256.  12 heads of 64 in fp32,
        // 256 over 500 69 | 58.  From there on lengths decide, which are not known here: x 1/2, 32 heads on 4, 16 over 2000 37.5 | 23.7, 256 over 4000 123 | 139; x 2, 32 on 8, 64 over 2000
        // 109 | 96, over 8000 306 | 344.
        const bool chunks = c.hs <= 128 && (long long)most * G > FEW_ROWS && c.tokens > c.batch + c.batch / 4;
        w.few = chunks ? FEW_ROWS : 0;
        // Up to two units in one where there are few sequences: going on for a tile takes less than putting two partial results together (us, 12 heads over 100
        // positions, fp32, 9.6 | 8.2).  With many of them a unit has to stand for its length (64 sequences of up to 4096, 8 key heads, 120 | 124).
        w.one = (long long)c.batch * c.kvH * w.headTiles < SPLIT_GRID / 2 ? 2 * 4 * 16 * (c.ct == F32 ? 1 : 2) : 0;
        // its list is counted in 32 bits
        const double units = (double)c.kvH * w.headTiles * (chunks ? c.batch : c.tokens / w.perTile + c.batch) * (c.maxPages * (double)c.pageSize / 64 + 1);
        const bool fits = !chunks || chunk_plan(c, dt).units <= 1e9;
        if (workspace && in_pieces(c, dt, q, y) && units < PAGED_MOST && fits) {
            if (chunks) {
                const ChunkPlan p = chunk_plan(c, dt);
                float* own = (float*)((char*)workspace + split_bytes(c));
                ChunkArgs g = {own, (ChunkJoin*)(own + (size_t)p.grid * 2 * CHUNK_ROWS * (padded_size(c) + 2)), FEW_ROWS, w.shift, p.perTile, p.tileHeads, p.headTiles, p.unit, p.pipe ? 2 : 1, p.pipe ? (const int*)own : nullptr};
                if (p.pipe) {
                    const hipError_t e = pieces ? attn_paged_pieces_launch(s, a, g, p.pipe, (int*)own, (char*)own + ((size_t)p.pipe * sizeof(int) + 255 & ~(size_t)255))
                                                : attn_paged_pipe_launch(s, a, g, p.pipe, (int*)own);
                    if (e != hipSuccess) return e;
                }
                const int grid = p.pipe ? 2 * p.pipe : p.grid;
                if (c.hs <= 64) hipLaunchKernelGGL((attn_paged_chunk_kernel<T_, TC_, 64>), grid + SPLIT_GRID, 256, 0, s, a, g, w, grid);
                else hipLaunchKernelGGL((attn_paged_chunk_kernel<T_, TC_, 128>), grid + SPLIT_GRID, 256, 0, s, a, g, w, grid);
                if (!p.pipe && grid > 1) {
                    if (c.hs <= 64) hipLaunchKernelGGL((attn_paged_join_kernel<T_, 64>), dim3(grid, 8), 256, 0, s, a, g);
                    else hipLaunchKernelGGL((attn_paged_join_kernel<T_, 128>), dim3(grid, 8), 256, 0, s, a, g);
                }
                return hipGetLastError();
            }
            if (c.hs <= 64) hipLaunchKernelGGL((attn_paged_split_kernel<T_, TC_, 64>), SPLIT_GRID, 256, 0, s, a, w);
            else if (c.hs <= 128) hipLaunchKernelGGL((attn_paged_split_kernel<T_, TC_, 128>), SPLIT_GRID, 256, 0, s, a, w);
            else hipLaunchKernelGGL((attn_paged_split_kernel<T_, TC_, 256>), SPLIT_GRID / 2, 256, 0, s, a, w);
            return hipGetLastError();
        }
        const int x = std::min(c.tokens, 1 << 21);   // an axis of a launch has less than 2^32 threads
        const dim3 grid(x, c.H, (c.tokens + x - 1) / x);
        auto any = [&](auto lanes) {
            constexpr int LPH = decltype(lanes)::value;
            if ((long long)c.tokens * c.H < ANY_MANY) hipLaunchKernelGGL((attn_paged_any_kernel<T_, TC_, 4, LPH, 16>), grid, 1024, 0, s, a);
            else hipLaunchKernelGGL((attn_paged_any_kernel<T_, TC_, 4, LPH, 4>), grid, 256, 0, s, a);
        };
        if (c.hs <= 64) any(std::integral_constant<int, 16>{});
        else if (c.hs <= 128) any(std::integral_constant<int, 32>{});
        else any(std::integral_constant<int, 64>{});
        return hipGetLastError();
    };
    if (dt == F32) return c.ct == F32 ? go(float(), float()) : go(float(), bf16_t());
    return go(bf16_t(), bf16_t());
}

}  // namespace mch
