// What a workgroup of attention over pages does with its run of a list of work: the split of positions (split_run) and tiles of many rows (chunk_run).  Whose work
// is on the list, and what becomes of the sums, a policy says: the sequences of a launch (attn_paged.hip), or prefixes and what is behind them (attn_prefix.hip).
#pragma once
#include <algorithm>
#include <type_traits>

#include "attn_paged.h"
#include "flash_traits.h"
#include "kernels.h"
#include "lane_ops.h"
#include "paged.h"

namespace mch {

namespace {

template <typename T> __device__ __forceinline__ float value_of(T v);
template <> __device__ __forceinline__ float value_of<float>(float v) { return v; }
template <> __device__ __forceinline__ float value_of<bf16_t>(bf16_t v) { return bf16_to_f32(v); }
template <typename T> __device__ __forceinline__ T stored(float v);
template <> __device__ __forceinline__ float stored<float>(float v) { return v; }
template <> __device__ __forceinline__ bf16_t stored<bf16_t>(float v) { return f32_to_bf16(v); }

// The sequences of a launch, as starts and lengths say them; sums become rows of y
struct OfSequences {
    static constexpr bool SUMS = false;
    typedef PagedSpan Span;
    __device__ static int count(const PagedCache& c) { return c.batch; }
    __device__ static Span span(const PagedCache& c, int b) { return paged_span(c.starts[b], c.starts[b + 1], c.lens[b], c.tokens, c.maxPages * c.pageSize); }
    __device__ static Span all_lanes(const PagedCache& c, int b) { return span_at(c, b); }
    __device__ static int from_of(const Span&) { return 0; }
    __device__ static int pos_of(const Span& s) { return s.len - s.count; }      // position of its first token
    __device__ static int row_of(const Span&, int b) { return b; }               // of the block table
    __device__ static int grow_of(const Span&, int perTile) { return perTile; }  // positions that every further tile has more
    __device__ static float* sums_of(const PagedCache&, const Span&, int, int, int) { return nullptr; }   // where sums stay (SUMS)
};

// ---- few rows a sequence: the positions are what is split --------------------------------------------------------------------------
// 16 rows - tokens times the heads that share a key head - make the columns of one 16 x 16 matrix product, so every key and value is read once
// for all of them: what bounds this kernel is reading the cache.  All positions of all sequences, in units of four tiles of KT positions, are
// one list that is dealt to the workgroups in equal runs, whatever the lengths: a run ends inside an item (a sequence's key head and row
// tile), which the last workgroup to finish puts together.  A wavefront has every fourth tile, with statistics of its own; tiles of the wavefronts
// meet in LDS at the end of an item.  Measured: 64 sequences of up to 4096 positions, 32 heads on 8 of 128, 16 bits, 559 MB 117 us (4.8 TB/s; single tokens over a
// contiguous cache of that size are read at 5.6); one of 131000, 537 MB 120 us; one of 100, 12 heads of 64 in fp32, 7.2 us.
//
// Scores are S^T = K Q^T, so that a lane has one row: register v of a tile holds key 4 (lane / 16) + v of row lane % 16, which is the operand
// layout that O^T = V^T P^T wants of P (which slot of the contraction is which key only has to agree between the two).  Keys go from memory to the
// operand registers as they are.  16-bit values take the way through LDS, where the transposing read makes columns of them; fp32 sums (rows in
// fp32) contract four keys at a time, one a lane group, and take values, of either type, as they come.
typedef float floatx4 __attribute__((ext_vector_type(4)));

struct SplitArgs {
    float* part;      // partial results, [workgroup][2][16 {maximum, sum} | 16 rows of HSP]
    int* tickets;     // one a workgroup; zero between launches
    int few;          // sequences of more rows a key head than this are another kernel's (0: all are this one's)
    int shift;        // log2 of the page size, or -1
    int perTile;      // tokens a row tile
    int tileHeads;    // heads a row tile, of G
    int headTiles;    // row tiles that the G heads of a key head take
    int one;          // sequences of at most this many positions are one unit
};

// of a maximum over scores that a row sees: what tells "all of them -inf" from "none"
constexpr float SCORE_FLOOR = -3.0e38f;

__device__ __forceinline__ void put2(float* p, float a, float b)
{
    union { float f[2]; uint64_t u; } x = {{a, b}};
    __hip_atomic_store((uint64_t*)p, x.u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 get2(const float* p)
{
    union { uint64_t u; float2 f; } x;
    x.u = __hip_atomic_load((const uint64_t*)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return x.f;
}
// weight of sums with maximum m beside others whose maximum is M (sums without a score are zero or not a number)
__device__ __forceinline__ float weight_of(float m, float M) { return m > -INFINITY ? __builtin_amdgcn_exp2f(m - M) : 1.f; }

template <typename T> __device__ __forceinline__ bool not_finite(u32x4 x)
{
    constexpr uint32_t E = sizeof(T) == 4 ? 0x7f800000u : 0x7f807f80u;
    bool r = false;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (sizeof(T) == 4) r = r || (x[i] & E) == E;
        else r = r || (x[i] & 0x7f80u) == 0x7f80u || (x[i] & 0x7f800000u) == 0x7f800000u;
    }
    return r;
}

template <typename TQ, typename TC, int HSP, typename L = OfSequences> struct SplitShared {
    static constexpr int KT = sizeof(TC) == 4 ? 16 : 32, STAGE = sizeof(TQ) == 2 ? KT * HSP * 2 : 0, LDO = HSP + 4;
    __attribute__((aligned(16))) unsigned char mem[4 * STAGE > 4 * 16 * LDO * 4 ? 4 * STAGE : 4 * 16 * LDO * 4];
    float m[4][16], l[4][16];
    typename L::Span span;
    int scan[4], seq, at, bad, ticket;
};
// what workgroup `block` of `blocks` has of the list
template <typename TQ, typename TC, int HSP, typename L>
__device__ __forceinline__ void split_run(const PagedAttnArgs& a, const SplitArgs& w, int block, int blocks, SplitShared<TQ, TC, HSP, L>& shared, const L& list)
{
    typedef SplitShared<TQ, TC, HSP, L> S;
    typedef typename L::Span Span;
    constexpr bool B16 = sizeof(TQ) == 2;
    constexpr int EPL = 16 / (int)sizeof(TC), NF = HSP / (4 * EPL);            // values a piece, pieces a lane and key
    constexpr int KG = sizeof(TC) == 4 ? 1 : 2, KT = 16 * KG, UNIT = 4 * KT;   // groups of 16 keys a tile
    constexpr int VE = sizeof(TC) == 4 ? 4 : HSP / 16 < 8 ? HSP / 16 : 8, NH = HSP / (16 * VE), NO = HSP / 16;
    constexpr int ROWB = HSP * 2, STAGE = S::STAGE, LDO = S::LDO, PART = 16 * (HSP + 2);
    static_assert(KT == S::KT && (HSP == 64 || HSP == 128 || HSP == 256), "tile");
    unsigned char* smem = shared.mem;
    auto &sM = shared.m, &sL = shared.l;
    auto& sSpan = shared.span;
    auto& sScan = shared.scan;
    int &sSeq = shared.seq, &sAt = shared.at, &sBad = shared.bad, &sTicket = shared.ticket;
    float* sO = (float*)smem;                                                   // [wavefront][row][LDO], once the stages are done with

    const PagedCache& c = a.c;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r16 = lane & 15, g = lane >> 4;
    const int G = c.H / c.kvH;

    // units of a sequence; a row tile without positions is one all the same (its rows are zeros)
    auto span_of = [&](int b) { return list.span(c, b); };
    auto units_of = [&](const Span& s) { const int n = s.len - list.from_of(s); return n <= max(w.one, UNIT) ? 1 : (n + UNIT - 1) / UNIT; };
    auto tiles_of = [&](const Span& s) -> int { return w.few && (long long)s.count * G > w.few ? 0 : (s.count + w.perTile - 1) / w.perTile * w.headTiles; };
    auto work_of = [&](const Span& s) -> int { return tiles_of(s) * c.kvH * units_of(s); };
    PagedRuns runs(0, 1, 1);
    Span sp;
    int b = 0, local, lo, hi;
    if constexpr (L::SUMS) {   // it is written down
        runs = PagedRuns(list.split_total(), blocks, 1);
        if (block >= runs.W) return;
        lo = runs.begin(block);
        hi = runs.begin(block + 1);
        const auto at = list.split_start(block);
        b = at.b;
        local = at.local;
        sp = list.all_lanes(c, b);
    } else if (c.batch == 1) {   // no sums, no sequence to be found
        sp = span_at(c, 0);
        runs = PagedRuns(work_of(sp), blocks, 1);
        if (block >= runs.W) return;
        local = lo = runs.begin(block);
        hi = runs.begin(block + 1);
    } else if (c.batch <= 64) {   // every wavefront for itself
        const PagedSpan mine = lane < c.batch ? span_of(lane) : PagedSpan{0, 0, 0};
        const int work = lane < c.batch ? work_of(mine) : 0, upTo = wave_scan(work), total = __builtin_amdgcn_readlane(upTo, 63);
        if (total >= PAGED_MOST) return;
        runs = PagedRuns(total, blocks, 1);
        if (block >= runs.W) return;
        lo = runs.begin(block);
        hi = runs.begin(block + 1);
        b = __builtin_ctzll(__ballot(lo < upTo));   // the sequence that has unit `lo`
        local = lo - (__builtin_amdgcn_readlane(upTo, b) - __builtin_amdgcn_readlane(work, b));
        sp = PagedSpan{__builtin_amdgcn_readlane(mine.first, b), __builtin_amdgcn_readlane(mine.count, b), __builtin_amdgcn_readlane(mine.len, b)};
    } else {
        const PagedSpan none = {0, 0, 0};
        PagedSpan mine = tid < c.batch ? span_of(tid) : none;
        int total, work = work_of(mine), at = block_scan(work, sScan, &total), all = total;
        for (int b0 = 256; b0 < c.batch; b0 += 256) {
            int more;
            block_scan(b0 + tid < c.batch ? work_of(span_of(b0 + tid)) : 0, sScan, &more);
            total = paged_sum(total, more);
        }
        if (uniform(total) >= PAGED_MOST) return;
        runs = PagedRuns(uniform(total), blocks, 1);
        if (block >= runs.W) return;
        lo = runs.begin(block);
        hi = runs.begin(block + 1);
        // the sequence that has unit `lo`
        for (int b0 = 0, base = 0;;) {
            if (at <= lo && lo < at + work) { sSeq = b0 + tid; sAt = at; sSpan = mine; }
            base += all;
            if (lo < base) break;
            if ((b0 += 256) >= c.batch) return;
            mine = b0 + tid < c.batch ? span_of(b0 + tid) : none;
            work = work_of(mine);
            at = base + block_scan(work, sScan, &all);
        }
        __syncthreads();
        b = uniform(sSeq);
        local = uniform(lo - sAt);
        sp = uniform(sSpan);
    }

    const TC *kp = (const TC*)c.k, *vp = (const TC*)c.v;
    for (int u = lo; u < hi;) {
        // ---- the item and the piece of it that is this workgroup's ----
        const int units = units_of(sp);
        const int item = local / units, unit0 = local - item * units, count = min(units - unit0, hi - u);
        const int tile = item / c.kvH, kh = item - tile * c.kvH, ht = tile % w.headTiles, j0 = tile / w.headTiles * w.perTile;
        const int h0 = kh * G + ht * w.tileHeads, nh = min(w.tileHeads, G - ht * w.tileHeads), nt = min(w.perTile, sp.count - j0);
        const int base = list.pos_of(sp) + j0, from = list.from_of(sp);          // position of the tile's first token
        const int p0 = from + unit0 * UNIT, p1 = min(unit0 + count == units ? sp.len : from + (unit0 + count) * UNIT, base + nt);
        const int token = r16 / w.tileHeads, head = r16 - token * w.tileHeads;   // of the lane's row
        const bool rowLive = token < nt && head < nh;
        const int last = base + token;
        auto row_at = [&](int t, int h) { return ((size_t)(sp.first + j0 + t) * c.H + h0 + h) * c.hs; };

        // ---- the row's queries, in the operand layout ----
        u32x4 qb[B16 ? NF : 1];
        float qf[B16 ? 1 : NF * EPL];
        {
            const TQ* q = (const TQ*)a.q + (rowLive ? row_at(token, head) : 0);
#pragma unroll
            for (int f = 0; f < NF; f++) {
                const int d = (4 * f + g) * EPL;
                if constexpr (B16) qb[f] = rowLive && d < c.hs ? *(const u32x4*)(q + d) : u32x4{0u, 0u, 0u, 0u};
                else
#pragma unroll
                    for (int e = 0; e < EPL; e += 4) {
                        const float4 x = rowLive && d < c.hs ? *(const float4*)(q + d + e) : make_float4(0.f, 0.f, 0.f, 0.f);
                        qf[f * EPL + e] = x.x; qf[f * EPL + e + 1] = x.y; qf[f * EPL + e + 2] = x.z; qf[f * EPL + e + 3] = x.w;
                    }
            }
        }
        // ---- where keys lie: the lane's keys r16 and 16 + r16 of a tile ----
        const float* table = c.table + (size_t)list.row_of(sp, b) * c.maxPages;
        auto entry_of = [&](int t, float (&e)[KG]) {
#pragma unroll
            for (int k = 0; k < KG; k++) {
                const int p = t + 16 * k + r16;
                e[k] = p < p1 ? table[w.shift >= 0 ? p >> w.shift : p / c.pageSize] : -1.f;
            }
        };
        auto places = [&](int t, const float (&e)[KG], long long (&off)[KG]) {
#pragma unroll
            for (int k = 0; k < KG; k++) {
                const int p = t + 16 * k + r16, page = p < p1 ? paged_page(e[k], c.pages) : -1;
                const int slot = w.shift >= 0 ? p & (c.pageSize - 1) : p % c.pageSize;
                off[k] = page >= 0 ? page * c.sP + slot * c.sT + kh * c.sH : -1;
            }
        };
        const u32x4 zero4 = {0u, 0u, 0u, 0u};
        auto piece_of = [&](const TC* p, long long off, int d) -> u32x4 { return off >= 0 && d < c.hs ? *(const u32x4*)(p + off + d) : zero4; };
        u32x4 kf[KG][NF], vf[B16 ? KG : 1][B16 ? NF : 1], vd[B16 ? 1 : KG][4][NH];
        auto load_k = [&](const long long (&off)[KG]) {
#pragma unroll
            for (int k = 0; k < KG; k++)
#pragma unroll
                for (int f = 0; f < NF; f++) kf[k][f] = piece_of(kp, off[k], (4 * f + g) * EPL);
        };
        auto load_v = [&](const long long (&off)[KG]) {
            if constexpr (B16) {
#pragma unroll
                for (int k = 0; k < KG; k++)
#pragma unroll
                    for (int f = 0; f < NF; f++) vf[k][f] = piece_of(vp, off[k], (4 * f + g) * EPL);
            } else {
#pragma unroll
                for (int k = 0; k < KG; k++)
#pragma unroll
                    for (int v = 0; v < 4; v++) {
                        const long long o = __shfl(off[k], 4 * g + v);
#pragma unroll
                        for (int h = 0; h < NH; h++) {
                            const int d = 16 * VE * h + VE * r16;
                            if constexpr (sizeof(TC) * VE == 16) vd[k][v][h] = piece_of(vp, o, d);
                            else {
                                const uint2 x = o >= 0 && d < c.hs ? *(const uint2*)(vp + o + d) : make_uint2(0u, 0u);
                                vd[k][v][h] = u32x4{x.x, x.y, 0u, 0u};
                            }
                        }
                    }
            }
        };
        // ---- the wavefront's tiles ----
        floatx4 o[NO];
        float m = -INFINITY, l = 0.f;
        bool bad = false;
#pragma unroll
        for (int i = 0; i < NO; i++) o[i] = floatx4{0.f, 0.f, 0.f, 0.f};
        unsigned char* stage = smem + wave * STAGE;
        long long off[KG], next[KG];
        float entry[KG];
        int t = p0 + wave * KT;
        if (tid == 0) sBad = 0;
        if (t < p1) {
            entry_of(t, entry);
            places(t, entry, off);
            load_k(off);
            load_v(off);
            entry_of(t + UNIT, entry);
        }
        for (; t < p1; t += UNIT) {
            floatx4 s[KG];
#pragma unroll
            for (int k = 0; k < KG; k++) {
                s[k] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int f = 0; f < NF; f++) {
                    if constexpr (B16) s[k] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(*(bf16x8*)&kf[k][f], *(bf16x8*)&qb[f], s[k], 0, 0, 0);
                    else
#pragma unroll
                        for (int e = 0; e < EPL; e++) {
                            float x;
                            if constexpr (EPL == 4) x = __uint_as_float(kf[k][f][e]);
                            else x = __uint_as_float(e & 1 ? kf[k][f][e >> 1] & 0xffff0000u : kf[k][f][e >> 1] << 16);
                            s[k] = __builtin_amdgcn_mfma_f32_16x16x4f32(x, qf[f * EPL + e], s[k], 0, 0, 0);
                        }
                }
            }
            uint32_t given = 0;                                                  // keys of the tile that lie in a page
#pragma unroll
            for (int k = 0; k < KG; k++) given |= (uint32_t)(__ballot(off[k] >= 0) & 0xffffu) << (16 * k);
            // the next tile's keys, and the entries of the one behind it
            places(t + UNIT, entry, next);
            load_k(next);
            entry_of(t + 2 * UNIT, entry);

            const bool open = t + KT <= base + 1;                                // every row sees all of it
            float mx = -INFINITY;
#pragma unroll
            for (int k = 0; k < KG; k++)
#pragma unroll
                for (int v = 0; v < 4; v++) s[k][v] *= a.c2;
            if (open && given == (KG == 2 ? 0xffffffffu : 0xffffu)) {
#pragma unroll
                for (int k = 0; k < KG; k++)
#pragma unroll
                    for (int v = 0; v < 4; v++) mx = fmaxf(mx, s[k][v]);
                mx = fmaxf(mx, SCORE_FLOOR);
            } else {
#pragma unroll
                for (int k = 0; k < KG; k++)
#pragma unroll
                    for (int v = 0; v < 4; v++) {
                        const int key = 16 * k + 4 * g + v;
                        const bool sees = (given >> key & 1) && t + key <= last;
                        mx = fmaxf(mx, sees ? fmaxf(s[k][v], SCORE_FLOOR) : -INFINITY);
                        s[k][v] = sees ? s[k][v] : -INFINITY;
                    }
            }
            mx = max_lane_xor<16>(mx);
            mx = fmaxf(max_lane_xor<32>(mx), m);
            const float ref = mx > -INFINITY ? mx : 0.f, alpha = __builtin_amdgcn_exp2f(m - ref);
            const bool moved = __any(mx != m);
            m = mx;
            float sum = 0.f;
#pragma unroll
            for (int k = 0; k < KG; k++)
#pragma unroll
                for (int v = 0; v < 4; v++) {
                    s[k][v] = __builtin_amdgcn_exp2f(s[k][v] - ref);
                    sum += s[k][v];
                }
            l = l * alpha + sum;
            if (moved)
#pragma unroll
                for (int i = 0; i < NO; i++) o[i] *= alpha;
            if constexpr (B16) {
#pragma unroll
                for (int k = 0; k < KG; k++)
#pragma unroll
                    for (int f = 0; f < NF; f++) {
                        const int row = 16 * k + r16, sw = HSP == 64 ? (row >> 1) & 7 : row & 15;
                        *(u32x4*)(stage + row * ROWB + (((4 * f + g) ^ sw) << 4)) = vf[k][f];
                        if (!open) bad = bad || not_finite<TC>(vf[k][f]);
                    }
                load_v(next);
                wave_lds_fence();
                // weights as two bf16 numbers, sixteen bits of them: the second product is free beside the reading
                u32x4 p, rest;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float x = s[e >> 1 ? KG - 1 : 0][2 * (e & 1)], y = s[e >> 1 ? KG - 1 : 0][2 * (e & 1) + 1];
                    p[e] = pack_bf16x2(x, y);
                    rest[e] = pack_bf16x2(x - __uint_as_float(p[e] << 16), y - __uint_as_float(p[e] & 0xffff0000u));
                }
#pragma unroll
                for (int i = 0; i < NO; i++) {
                    uint2 half[2];
#pragma unroll
                    for (int k = 0; k < 2; k++) {
                        const int row = 16 * k + 4 * g + (r16 >> 2), sw = HSP == 64 ? (row >> 1) & 7 : row & 15, piece = 2 * i + ((r16 & 3) >> 1);
                        half[k] = lds_read_tr16((const bf16_t*)(stage + row * ROWB + ((piece ^ sw) << 4) + (r16 & 1) * 8));
                    }
                    u32x4 vt = {half[0].x, half[0].y, half[1].x, half[1].y};
                    o[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(*(bf16x8*)&vt, *(bf16x8*)&p, o[i], 0, 0, 0);
                    o[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(*(bf16x8*)&vt, *(bf16x8*)&rest, o[i], 0, 0, 0);
                }
                wave_lds_fence();
            } else {
#pragma unroll
                for (int k = 0; k < KG; k++)
#pragma unroll
                    for (int v = 0; v < 4; v++)
#pragma unroll
                        for (int h = 0; h < NH; h++) {
                            if (!open) bad = bad || not_finite<TC>(vd[k][v][h]);
#pragma unroll
                            for (int e = 0; e < VE; e++) {
                                float x;
                                if constexpr (sizeof(TC) == 4) x = __uint_as_float(vd[k][v][h][e]);
                                else x = __uint_as_float(e & 1 ? vd[k][v][h][e >> 1] & 0xffff0000u : vd[k][v][h][e >> 1] << 16);
                                o[h * VE + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(x, s[k][v], o[h * VE + e], 0, 0, 0);
                            }
                        }
                load_v(next);
            }
#pragma unroll
            for (int k = 0; k < KG; k++) off[k] = next[k];
        }
        // ---- the wavefronts meet ----
        l = add_lane_xor<32>(add_lane_xor<16>(l));
        __syncthreads();                                                         // the stages are done with
        if (g == 0) { sM[wave][r16] = m; sL[wave][r16] = l; }
#pragma unroll
        for (int i = 0; i < NO; i++)
#pragma unroll
            for (int v = 0; v < 4; v++) {
                const int d = B16 ? 16 * i + 4 * g + v : 16 * VE * (i / VE) + VE * (4 * g + v) + i % VE;
                sO[(wave * 16 + r16) * LDO + d] = o[i][v];
            }
        if (__any(bad) && lane == 0) sBad = 1;
        __syncthreads();
        if (sBad) {
            // A value that is not finite lies where only some of the rows look: weights of zero would not keep it from the others.  Row by row, then.
            __syncthreads();
            for (int r = wave; r < nt * w.tileHeads; r += 4) {
                const int tk = r / w.tileHeads, hd = r - tk * w.tileHeads;
                if (hd >= nh) continue;
                const TQ* q = (const TQ*)a.q + row_at(tk, hd);
                constexpr int VPL = HSP <= 128 ? 2 : HSP / 64;
                float qv[VPL], acc[VPL], mr = -INFINITY, lr = 0.f;
#pragma unroll
                for (int i = 0; i < VPL; i++) acc[i] = 0.f;
#pragma unroll
                for (int i = 0; i < VPL; i++) qv[i] = lane + 64 * i < c.hs ? value_of<TQ>(q[lane + 64 * i]) : 0.f;
                for (int p = p0; p < p1 && p <= base + tk; p++) {
                    const int e = p / c.pageSize, page = paged_page(table[e], c.pages);
                    if (page < 0) continue;
                    const long long at = page * c.sP + (p - e * c.pageSize) * c.sT + kh * c.sH;
                    float x = 0.f, val[VPL];
#pragma unroll
                    for (int i = 0; i < VPL; i++) {
                        const int d = lane + 64 * i;
                        x += d < c.hs ? qv[i] * value_of<TC>(kp[at + d]) : 0.f;
                        val[i] = d < c.hs ? value_of<TC>(vp[at + d]) : 0.f;
                    }
                    x = group_sum<64>(x) * a.c2;
                    const float mn = fmaxf(mr, fmaxf(x, SCORE_FLOOR)), f = __builtin_amdgcn_exp2f(mr - mn), wt = __builtin_amdgcn_exp2f(x - mn);
                    mr = mn;
                    lr = lr * f + wt;
#pragma unroll
                    for (int i = 0; i < VPL; i++) acc[i] = acc[i] * f + wt * val[i];
                }
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    if (lane == 0) { sM[i][r] = i ? -INFINITY : mr; sL[i][r] = i ? 0.f : lr; }
#pragma unroll
                    for (int j = 0; j < VPL; j++)
                        if (lane + 64 * j < HSP) sO[(i * 16 + r) * LDO + lane + 64 * j] = i ? 0.f : acc[j];
                }
            }
            __syncthreads();
        }
        const bool whole = count == units;
        const int rows = nt * w.tileHeads, pairs = c.hs >> 1;
        float* part = w.part + ((size_t)block * 2 + (unit0 == 0 ? 1 : 0)) * PART;
        for (int e = tid; e < rows * pairs; e += 256) {
            const int r = e / pairs, d = 2 * (e - r * pairs), tk = r / w.tileHeads, hd = r - tk * w.tileHeads;
            if (hd >= nh) continue;
            float M = -INFINITY, L_ = 0.f, x = 0.f, y = 0.f;
#pragma unroll
            for (int i = 0; i < 4; i++) M = fmaxf(M, sM[i][r]);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float f = weight_of(sM[i][r], M);
                const float2 v = *(const float2*)(sO + (i * 16 + r) * LDO + d);
                L_ += sL[i][r] * f;
                x += v.x * f;
                y += v.y * f;
            }
            if (L::SUMS && whole) {
                float* to = list.sums_of(c, sp, sp.first + j0 + tk, h0 + hd, HSP);
                *(float2*)(to + 4 + d) = make_float2(x, y);
                if (d == 0) *(float2*)to = make_float2(M, L_);
            } else if (whole) {
                TQ* out = (TQ*)a.y + row_at(tk, hd) + d;
                const float xs = M > -INFINITY ? x / L_ : 0.f, ys = M > -INFINITY ? y / L_ : 0.f;
                if constexpr (B16) *(uint32_t*)out = pack_bf16x2(xs, ys);
                else *(float2*)out = make_float2(xs, ys);
            } else {
                put2(part + 32 + r * HSP + d, x, y);
                if (d == 0) put2(part + 2 * r, M, L_);
            }
        }
        if (!L::SUMS && !whole) {
            // Who comes last puts the item together; its workgroups follow from the list alone.  Partial results go to the level that all XCDs
            // share, and are there before the ticket is taken.
            const int wf = runs.of(u - unit0), we = runs.of(u - unit0 + units - 1);
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
            if (tid == 0) sTicket = __hip_atomic_fetch_add(w.tickets + wf, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __syncthreads();
            if (sTicket == we - wf) {
                // DEEP partial results in flight (past the last one that again, with no weight)
                auto join = [&](auto deep) __attribute__((always_inline)) {
                    constexpr int DEEP = decltype(deep)::value;
                    for (int e = tid; e < rows * pairs; e += 256) {
                        const int r = e / pairs, d = 2 * (e - r * pairs), tk = r / w.tileHeads, hd = r - tk * w.tileHeads;
                        if (hd >= nh) continue;
                        float M = -INFINITY, L_ = 0.f, x = 0.f, y = 0.f;
                        for (int i = wf; i <= we; i += DEEP) {
                            float2 ml[DEEP], v[DEEP];
    #pragma unroll
                            for (int j = 0; j < DEEP; j++) {
                                const float* from = w.part + ((size_t)min(i + j, we) * 2 + (i + j == wf ? 1 : 0)) * PART;
                                ml[j] = get2(from + 2 * r);
                                v[j] = get2(from + 32 + r * HSP + d);
                            }
                            float Mn = M;
    #pragma unroll
                            for (int j = 0; j < DEEP; j++) Mn = i + j <= we ? fmaxf(Mn, ml[j].x) : Mn;
                            const float f0 = weight_of(M, Mn);
                            L_ *= f0; x *= f0; y *= f0;
    #pragma unroll
                            for (int j = 0; j < DEEP; j++) {
                                const float f = weight_of(ml[j].x, Mn);
                                L_ += i + j <= we ? ml[j].y * f : 0.f;
                                x += i + j <= we ? v[j].x * f : 0.f;
                                y += i + j <= we ? v[j].y * f : 0.f;
                            }
                            M = Mn;
                        }
                        TQ* out = (TQ*)a.y + row_at(tk, hd) + d;
                        const float xs = M > -INFINITY ? x / L_ : 0.f, ys = M > -INFINITY ? y / L_ : 0.f;
                        if constexpr (B16) *(uint32_t*)out = pack_bf16x2(xs, ys);
                        else *(float2*)out = make_float2(xs, ys);
                    }
                };
                if (we - wf < 4) join(std::integral_constant<int, 4>{});
                else join(std::integral_constant<int, 16>{});
                if (tid == 0) __hip_atomic_store(w.tickets + wf, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);   // for the next launch
            }
        }
        // ---- the next item ----
        u += count;
        local += count;
        if (u < hi) {
            if (local == tiles_of(sp) * c.kvH * units) {
                local = 0;
                do {
                    if (++b >= list.count(c)) return;
                    sp = list.all_lanes(c, b);
                } while (tiles_of(sp) == 0);
            }
            __syncthreads();                                                     // LDS is read no more
        }
    }
}

// ---- chunks: rows by the hundred ----------------------------------------------------------------------------------------------------
// A workgroup has 128 rows of one key head (tokens times the heads that share it), 32 a wavefront, and stages blocks of KB keys and values in LDS for
// all of them: every value read from the cache meets 128 rows, and the matrix cores bound it.  Tiles of one key head go to one XCD (workgroups
// follow each other by key head), whose L2 then holds that head's keys and values.  The
// blocks of all tiles are one list that is dealt to the workgroups in equal runs; tiles that a run ends in are put together by a launch behind this one.
// Measured: 8 prompts of 2048, 12 heads of 64, fp32, 350 us (0.15 PFLOP/s of useful products, 0.9 of bf16 ones, which a large library product has 1.2 of);
// a step of 12 chunks and single tokens, ragged, 64 us with the launch behind: half of it starts, ends and tiles that are not full.
// Eight values as PARTS fragments of bf16: themselves, or of fp32 the three parts that hold its 24 bits, cut off (never rounded up to an infinity)
template <int PARTS> struct Parts { u32x4 p[PARTS]; };
__device__ __forceinline__ uint32_t upper_halves(float lo, float hi) { return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u); }
__device__ __forceinline__ float upper_half(float x) { return __uint_as_float(__float_as_uint(x) & 0xffff0000u); }
template <int PARTS> __device__ __forceinline__ void two_parts(float x, float y, uint32_t (&out)[PARTS])
{
#pragma unroll
    for (int i = 0; i < PARTS; i++) {
        out[i] = upper_halves(x, y);
        if (i + 1 < PARTS) {
            x -= upper_half(x);
            y -= upper_half(y);
        }
    }
}

// l + both values of a pair of bf16
__device__ __forceinline__ float pair_sum(uint32_t pair, float l)
{
    const bf16x2 ones = {(__bf16)1.0f, (__bf16)1.0f};
    return __builtin_amdgcn_fdot2_f32_bf16(*reinterpret_cast<bf16x2*>(&pair), ones, l, false);
}

// Products in fp32 are sums of products of bf16 parts: of the nine of two values of three parts the six that reach fp32's last bits, exact each and
// added in fp32; over a 16-bit cache the three that there are.  (32 x 32 x 16 of them take 32 cycles a part, in fp32 512: 2.7 and 5.3 times as long.)
// Three parts hold every bit from 2^-133 up, all 24 of values from 2^-110 up.  What is cut off of smaller queries and keys changes no score if the other factor is below
// 2^65 (2^-133 2^65 2^8 a score, times a scale of up to SCALE: 2^-29), and of values no sum that is not small itself.  Rows where a factor is larger, or a sum of weights times
// values is below SMALL of the sum of weights, are made one by one (below).  A weight below 2^-110 of its row's largest loses bits and is left as it is.
// (us, 2 prompts of 1024, 12 heads of 64, as before 43; a column of values all zero, looked through for smaller ones, 59 for 47 in the same loop; rows one by one 4800.)
constexpr float SCALE = 0x1p31f, SMALL = 0x1p-100f;
// 2^65, from which on an exponent's two upper bits are set: of a piece, what has them so in `large_bits` (infinities and NaN among them)
template <typename T> __device__ __forceinline__ void take_large(u32x4 x, uint32_t& bits)
{
#pragma unroll
    for (int i = 0; i < 4; i++) bits |= x[i] & (x[i] << 1);
}
template <typename T> constexpr uint32_t large_bits() { return sizeof(T) == 4 ? 0x40000000u : 0x40004000u; }
template <typename TQ, typename TC, int HSP> struct ChunkShared {
    static constexpr int NQ = sizeof(TQ) == 4 ? 3 : 1, NK = sizeof(TC) == 4 ? 3 : 1;              // parts of a query and a weight, of a key and a value
    static constexpr int KB = NK == 1 && (NQ == 1 || HSP == 64) ? 64 : 32, LD = HSP + 8;          // keys a block, values a row
    __attribute__((aligned(16))) bf16_t k[NK][KB * LD], v[NK][KB * LD];
    long long place[2][KB];
    uint64_t given[2];
    int bad, front, zero;
};
template <typename TQ, typename TC, int HSP, typename L>
__device__ __forceinline__ void chunk_run(const PagedAttnArgs& a, const ChunkArgs& w, int block, int blocks, ChunkShared<TQ, TC, HSP>& shared, const L& list)
{
    typedef typename L::Span Span;
    typedef FlashTraits<bf16_t> TR;
    typedef ChunkShared<TQ, TC, HSP> S;
    constexpr int NQ = S::NQ, NK = S::NK, KB = S::KB, LD = S::LD;
    constexpr int NW = NQ == 1 && L::SUMS ? 2 : NQ;                                               // parts of a weight
    constexpr int KJ = KB / 32, KF = HSP / 16, DT = HSP / 32, EPL = 16 / (int)sizeof(TC);
    constexpr int CPR = HSP / EPL, NP = KB * CPR / 256, RPP = 256 / CPR;                          // pieces a row; pieces a thread; rows a round
    constexpr int AHEAD = NK == 3 && HSP == 128 ? 1 : 2;                                          // value fragments under way (1: registers are full)
    constexpr int PART = 128 * (HSP + 2);
    auto &sK = shared.k, &sV = shared.v;
    auto& sPlace = shared.place;
    auto& sGiven = shared.given;
    int &sBad = shared.bad, &sFront = shared.front, &sZero = shared.zero;

    const PagedCache& c = a.c;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l32 = lane & 31, half = lane >> 5;
    const int G = c.H / c.kvH;
    const int groups = c.kvH * w.headTiles;
    struct { int total, place, b, local; Span sp; } at = {};
    ChunkTile left = {};
    int u = 0, hi = 1;
    if constexpr (L::SUMS) {
        at.total = list.chunk_total();
        const PagedRuns runs(at.total, blocks, CHUNK_LEAST);
        at.place = paged_place(block, runs.W);
        if (at.place < 0) return;
        const auto start = list.chunk_start(at.place);
        at.b = start.b;
        at.local = start.local;
        at.sp = list.all_lanes(c, at.b);
        u = runs.begin(at.place);
        hi = runs.begin(at.place + 1);
    } else if (w.redo) {
        if (!w.redo[block / w.pair]) return;
        left = chunk_tile(c, w, block / w.pair);
        if (left.b < 0) return;
        at.b = left.b;
        at.sp = span_at(c, at.b);
    } else {
        const ChunkStart start = chunk_start(c, w, block, blocks);
        at = {start.total, start.place, start.b, start.local, start.sp};
        if (tid == 0) w.join[block].place = -1;
        if (at.place < 0) return;
        const PagedRuns runs(at.total, blocks, CHUNK_LEAST);
        u = runs.begin(at.place);
        hi = runs.begin(at.place + 1);
    }
    while (u < hi) {
    // ---- the tile and the piece of it that is this workgroup's: units u0 .. u1 - 1 of `units` ----
    const Span sp = at.sp;
    const int b = at.b, from = list.from_of(sp), before = L::SUMS ? max(min(list.pos_of(sp), sp.len) - from, 0) : max(sp.len - sp.count, 0);
    const int grow = L::SUMS ? list.grow_of(sp, w.perTile) : w.perTile;                           // positions that every further tile has more
    int group, tile, u0 = 0, u1 = 1, units = 1;
    if (!L::SUMS && w.redo) {
        group = left.kh * w.headTiles + left.ht;
        tile = left.tile * w.pair + (block % w.pair);
    } else {
        const int tiles = L::SUMS ? (sp.count + w.perTile - 1) / w.perTile : chunk_tiles(c, w, PagedSpan{sp.first, sp.count, sp.len});
        const int each = paged_units_before(before, grow, tiles, w.unit), r = at.local - at.local / each * each;
        group = at.local / each;
        tile = paged_tile_of(before, grow, tiles, w.unit, r);
        const int start = paged_units_before(before, grow, tile, w.unit);
        units = paged_units_before(before, grow, tile + 1, w.unit) - start;
        u0 = r - start;
        u1 = min(units, u0 + hi - u);
    }
    const bool whole = u0 == 0 && u1 == units;
    const int kh = group / w.headTiles, ht = group - kh * w.headTiles;
    const int j0 = tile * w.perTile, nt = min(w.perTile, sp.count - j0), base = list.pos_of(sp) + j0;
    if (nt <= 0) return;   // (redo: the second half of a tile that has none)
    if (tid == 0) sBad = sZero = 0;
    const int h0 = kh * G + ht * w.tileHeads, nh = min(w.tileHeads, G - ht * w.tileHeads);
    const int end = min(sp.len, base + nt);                                                       // positions that some row sees
    const float* table = c.table + (size_t)list.row_of(sp, b) * c.maxPages;
    const TC *kp = (const TC*)c.k + kh * c.sH, *vp = (const TC*)c.v + kh * c.sH;
    auto page_at = [&](int p) -> float { return table[w.shift >= 0 ? p >> w.shift : p / c.pageSize]; };
    auto place_of = [&](int p, float e) -> long long {
        const int page = p < end && p >= from ? paged_page(e, c.pages) : -1;
        return page >= 0 ? page * c.sP + (w.shift >= 0 ? p & (c.pageSize - 1) : p % c.pageSize) * c.sT : -1;
    };
    const float c2 = fabsf(a.c2);

    // ---- the lane's row ----
    const int row = 32 * wave + l32, token = row / w.tileHeads, head = row - token * w.tileHeads;
    const bool live = token < nt && head < nh;
    const int last = live ? base + token : -1;
    const int waveEnd = 32 * wave / w.tileHeads < nt ? min(end, base + min((32 * wave + 31) / w.tileHeads, nt - 1) + 1) : 0, waveOpen = base + 32 * wave / w.tileHeads + 1;   // past what any, and what every row sees
    auto row_at = [&](int t, int h) { return ((size_t)(sp.first + j0 + t) * c.H + h0 + h) * c.hs; };
    const u32x4 zero4 = {0u, 0u, 0u, 0u};
    bool bad = NQ > 1 && !(c2 < SCALE);
    uint32_t largeQ = 0;
    Parts<NQ> qf[KF];
    {
        const TQ* q = (const TQ*)a.q + (live ? row_at(token, head) : 0);
#pragma unroll
        for (int f = 0; f < KF; f++) {
            const int d = 16 * f + 8 * half;
            if constexpr (NQ == 1) {
                qf[f].p[0] = live && d < c.hs ? *(const u32x4*)(q + d) : zero4;
                if (a.c2 < 0.f) qf[f].p[0] ^= u32x4{0x80008000u, 0x80008000u, 0x80008000u, 0x80008000u};
            } else {
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; e += 4) {
                    const float4 y = live && d + e < c.hs ? *(const float4*)(q + d + e) : make_float4(0.f, 0.f, 0.f, 0.f);
                    x[e] = y.x; x[e + 1] = y.y; x[e + 2] = y.z; x[e + 3] = y.w;
                }
#pragma unroll
                for (int e = 0; e < 8; e++) x[e] = a.c2 < 0.f ? -x[e] : x[e];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    uint32_t out[NQ];
                    two_parts<NQ>(x[2 * e], x[2 * e + 1], out);
#pragma unroll
                    for (int i = 0; i < NQ; i++) qf[f].p[i][e] = out[i];
                }
#pragma unroll
                for (int e = 0; e < 8; e++) largeQ |= __float_as_uint(x[e]) & (__float_as_uint(x[e]) << 1);
            }
        }
    }
    if (NQ > 1) bad = bad || (largeQ & large_bits<float>());
    // pages given up at the front are passed over
    if (wave == 0) {
        int front = L::SUMS ? from / c.pageSize : 0;
        const int entries = end > 0 ? (end - 1) / c.pageSize + 1 : 0;
        for (; front < entries; front += 64) {
            const uint64_t some = __ballot(front + lane < entries && paged_page(table[min(front + lane, entries - 1)], c.pages) >= 0);
            if (some) { front += __ffsll((unsigned long long)some) - 1; break; }
        }
        if (lane == 0) sFront = min(front, entries) * c.pageSize;
    }
    __syncthreads();
    const int kb0 = min(uniform(sFront), max(end, 0)) / KB, nkb = (max(end, 0) + KB - 1) / KB;
    const int first = kb0 + (int)((long long)(nkb - kb0) * u0 / units), stop = kb0 + (int)((long long)(nkb - kb0) * u1 / units);

    floatx16 o[DT];
#pragma unroll
    for (int i = 0; i < DT; i++)
#pragma unroll
        for (int v = 0; v < 16; v++) o[i][v] = 0.f;
    float m = -INFINITY, l = 0.f;

    // ---- staging: places two blocks ahead, values one ----
    u32x4 rk[NP], rv[NP];
    auto load = [&](int slot) {
#pragma unroll
        for (int i = 0; i < NP; i++) {
            const int r = tid / CPR + RPP * i, d = (tid % CPR) * EPL;
            const long long at = sPlace[slot][r];
            const bool there = at >= 0 && d < c.hs;
            rk[i] = there ? *(const u32x4*)(kp + at + d) : zero4;
            rv[i] = there ? *(const u32x4*)(vp + at + d) : zero4;
        }
    };
    auto publish = [&](int kb, float e) {   // wavefront 0
        const int p = kb * KB + lane;
        const long long at = lane < KB ? place_of(p, e) : -1;
        if (lane < KB) sPlace[kb & 1][lane] = at;
        const uint64_t given = __ballot(at >= 0);
        if (lane == 0) sGiven[kb & 1] = given;
    };
    auto entry = [&](int kb) -> float { const int p = kb * KB + lane; return lane < KB && p < end ? page_at(p) : -1.f; };
    float ahead = -1.f;
    if (wave == 0 && first < stop) {
        publish(first, entry(first));
        publish(first + 1, entry(first + 1));
        ahead = entry(first + 2);
    }
    __syncthreads();
    if (first < stop) load(first & 1);
    for (int kb = first; kb < stop; kb++) {
        const uint64_t given = sGiven[kb & 1];
        __syncthreads();                                                         // everybody has left the previous block
        uint32_t large = 0;
#pragma unroll
        for (int i = 0; i < NP; i++) {
            const int r = tid / CPR + RPP * i, d = (tid % CPR) * EPL;
            if constexpr (NK == 1) {
                *(u32x4*)(sK[0] + r * LD + d) = rk[i];
                *(u32x4*)(sV[0] + r * LD + d) = rv[i];
            } else {
                uint32_t k[2][NK], v[2][NK];
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    two_parts<NK>(__uint_as_float(rk[i][2 * e]), __uint_as_float(rk[i][2 * e + 1]), k[e]);
                    two_parts<NK>(__uint_as_float(rv[i][2 * e]), __uint_as_float(rv[i][2 * e + 1]), v[e]);
                }
#pragma unroll
                for (int e = 0; e < NK; e++) {
                    *(uint2*)(sK[e] + r * LD + d) = make_uint2(k[0][e], k[1][e]);
                    *(uint2*)(sV[e] + r * LD + d) = make_uint2(v[0][e], v[1][e]);
                }
            }
            // what only some rows see, and where parts are multiplied anything, has to be finite (parts of a value that is not do not add up to it)
            if (NK > 1 || NQ > 1 || kb * KB + KB > base + 1) bad = bad || not_finite<TC>(rv[i]);
            if (NK > 1 || NQ > 1) {
                take_large<TC>(rk[i], large);
                asm volatile("" : "+v"(large));   // here and now: else pieces are kept for it until the end, and registers spilt (8 chunks of 1500 over 3000, fp32, 940 us for 840)
            }
        }
        if (NK > 1 || NQ > 1) bad = bad || (large & large_bits<TC>());
        if (wave == 0 && kb + 2 < stop) publish(kb + 2, ahead);
        __syncthreads();
        if (kb + 1 < stop) load((kb + 1) & 1);
        if (wave == 0) ahead = entry(kb + 3);
        const int t = kb * KB;
        if (t >= waveEnd || !given) continue;
        floatx16 s[KJ];
#pragma unroll
        for (int j = 0; j < KJ; j++) {
#pragma unroll
            for (int v = 0; v < 16; v++) s[j][v] = 0.f;
            const int krow = (32 * j + l32) * LD + 8 * half;
#pragma unroll
            for (int f = 0; f < KF; f++)
#pragma unroll
                for (int x = NK - 1; x >= 0; x--) {
                    const u32x4 k = *(const u32x4*)(sK[x] + krow + 16 * f);
#pragma unroll
                    for (int y = NQ - 1; y >= 0; y--)
                        if (x + y < 3) s[j] = TR::mma(k, qf[f].p[y], s[j]);
                }
        }
        // values travel while the weights are made, AHEAD fragments in front of the product that they are for (us with none | 1 | 2 | 4: a step of chunks and
        // single tokens in fp32 73.9 | 73.2 | 72.0 | 73.3, 4 sequences of 8 new tokens over 4096 in 16 bits 37.3 | 37.2 | 36.7 | 38.8; fp32 heads
        // of 128, 8 chunks of 1500 over 3000, 826 with 1, 873 with 2)
        u32x4 vf[AHEAD][NK];
        auto value = [&](int n) {
            const int j = n / (2 * DT), x = n / DT % 2, i = n % DT;
#pragma unroll
            for (int z = 0; z < NK; z++) vf[n % AHEAD][z] = TR::load_vt_rowmajor(sV[z] + 32 * j * LD + 32 * i, LD, x, lane);
        };
#pragma unroll
        for (int n = 0; n < AHEAD; n++) value(n);
        // Maxima are taken of the products themselves (the queries carry the scale's sign), and the running one moves only when a row's grows by 2^8:
        // weights stay below that, and the sums are seldom scaled again.
        float mx = -INFINITY;
        bool any = true;
        if (t + KB <= waveOpen && given == (KB == 64 ? ~0ull : 0xffffffffull)) {
#pragma unroll
            for (int j = 0; j < KJ; j++)
#pragma unroll
                for (int v = 0; v < 16; v++) mx = fmaxf(mx, s[j][v]);
        } else {
            any = false;
#pragma unroll
            for (int j = 0; j < KJ; j++) {
                const uint32_t there = (uint32_t)(given >> (32 * j));
#pragma unroll
                for (int v = 0; v < 16; v++) {
                    const int key = 8 * (v >> 2) + 4 * half + (v & 3);
                    const bool sees = (there >> key & 1) && t + 32 * j + key <= last;
                    any = any || sees;
                    s[j][v] = sees ? s[j][v] : -INFINITY;
                    mx = fmaxf(mx, s[j][v]);
                }
            }
        }
        mx = any ? fmaxf(mx * c2, SCORE_FLOOR) : -INFINITY;
        mx = max_lane_xor<32>(mx);
        if (__any(mx > m + 8.f)) {
            mx = fmaxf(mx, m);
            const float alpha = __builtin_amdgcn_exp2f(m - (mx > -INFINITY ? mx : 0.f));
            m = mx;
            l *= alpha;
#pragma unroll
            for (int i = 0; i < DT; i++)
#pragma unroll
                for (int v = 0; v < 16; v++) o[i][v] *= alpha;
        }
        const float ref = m > -INFINITY ? -m : 0.f;
#pragma unroll
        for (int j = 0; j < KJ; j++)
#pragma unroll
            for (int v = 0; v < 16; v++) {
                s[j][v] = __builtin_amdgcn_exp2f(fmaf(s[j][v], c2, ref));
                if (NW > 1) l += s[j][v];
            }
        // weights in the operand layout: of 16-bit rows rounded to one bf16 number (eight bits, as the pipe kernel's) and added up as rounded, or, behind and in shared
        // prefixes, to two (sixteen bits: most rows of a group are single tokens, which split_run gives as many); of fp32 rows in three parts
        Parts<NW> p[KJ][2];
#pragma unroll
        for (int j = 0; j < KJ; j++)
#pragma unroll
            for (int x = 0; x < 2; x++) {
                if constexpr (NQ == 1) {
                    p[j][x].p[0] = TR::pack_p(s[j], x);
                    if constexpr (NW == 2) p[j][x].p[1] = TR::pack_rest(s[j], x, p[j][x].p[0]);
                    else
#pragma unroll
                        for (int e = 0; e < 4; e++) l = pair_sum(p[j][x].p[0][e], l);
                } else
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        uint32_t out[NW];
                        two_parts<NW>(s[j][8 * x + 2 * e], s[j][8 * x + 2 * e + 1], out);
#pragma unroll
                        for (int i = 0; i < NW; i++) p[j][x].p[i][e] = out[i];
                    }
            }
#pragma unroll
        for (int n = 0; n < KJ * 2 * DT; n++) {
            const int j = n / (2 * DT), x = n / DT % 2, i = n % DT;
#pragma unroll
            for (int z = NK - 1; z >= 0; z--)
#pragma unroll
                for (int y = NW - 1; y >= 0; y--)
                    if (z + y < 3) o[i] = TR::mma(vf[n % AHEAD][z], p[j][x].p[y], o[i]);
            if (n + AHEAD < KJ * 2 * DT) value(n + AHEAD);
        }
    }
    l = add_lane_xor<32>(l);
    if constexpr (NQ > 1) {
        // sums that are small or zero
        float least = INFINITY;
#pragma unroll
        for (int i = 0; i < DT; i++)
#pragma unroll
            for (int v = 0; v < 16; v += 4) {
                const float x = fminf(fminf(fabsf(o[i][v]), fabsf(o[i][v + 1])), fminf(fabsf(o[i][v + 2]), fabsf(o[i][v + 3])));
                least = fminf(least, 32 * i + 2 * v + 4 * half < c.hs ? x : INFINITY);
            }
        if (__any(live && least < l * SMALL)) {
            bool zero = false;
            if (live)
#pragma unroll
                for (int i = 0; i < DT; i++)
#pragma unroll
                    for (int v = 0; v < 16; v++)
                        if (32 * i + 8 * (v >> 2) + 4 * half < c.hs) {
                            zero = zero || o[i][v] == 0.f;
                            bad = bad || (fabsf(o[i][v]) < l * SMALL && o[i][v] != 0.f);
                        }
            if (__any(zero) && lane == 0) sZero = 1;
        }
    }
    if (__any(bad) && lane == 0) sBad = 1;
    __syncthreads();
    if (NK > 1 && sZero && !sBad) {
        // of values that are zero, or of such as lie below the last part?  (Reads of DEEP positions under way.)
        constexpr int DEEP = 4;
        const int d = min((tid % CPR) * EPL, c.hs - EPL), until = min(stop * KB, end);
        bool found = false;
        for (int p0 = first * KB + tid / CPR; p0 < until; p0 += DEEP * RPP) {
            float e[DEEP];
            u32x4 x[DEEP];
#pragma unroll
            for (int i = 0; i < DEEP; i++) e[i] = page_at(min(p0 + i * RPP, until - 1));
#pragma unroll
            for (int i = 0; i < DEEP; i++) {
                const long long at = place_of(min(p0 + i * RPP, until - 1), e[i]);
                x[i] = at >= 0 ? *(const u32x4*)(vp + at + d) : zero4;
            }
#pragma unroll
            for (int i = 0; i < 4 * DEEP; i++) found = found || (x[i / 4][i % 4] & 0x7fffffffu) - 1 < __float_as_uint(0x1p-110f) - 1;
        }
        __syncthreads();
        if (__any(found) && lane == 0) sBad = 1;
        __syncthreads();
    }

    float* part = w.part + ((size_t)at.place * 2 + (u0 == 0 ? 1 : 0)) * PART;
    if (!sBad) {
        if (live) {
            TQ* y = (TQ*)a.y + row_at(token, head);
            const float inv = 1.f / l;
            float* sums = L::SUMS && whole ? list.sums_of(c, sp, sp.first + j0 + token, h0 + head, HSP) : nullptr;
            if (!whole && half == 0) *(float2*)(part + 2 * row) = make_float2(m, l);
            if (L::SUMS && whole && half == 0) *(float2*)sums = make_float2(m, l);
#pragma unroll
            for (int i = 0; i < DT; i++)
#pragma unroll
                for (int v = 0; v < 4; v++) {
                    const int d = 32 * i + 8 * v + 4 * half;
                    if (d >= c.hs) continue;
                    float x[4] = {o[i][4 * v], o[i][4 * v + 1], o[i][4 * v + 2], o[i][4 * v + 3]};
                    if (!whole) *(float4*)(part + 256 + row * HSP + d) = make_float4(x[0], x[1], x[2], x[3]);
                    else if (L::SUMS) {
                        *(float4*)(sums + 4 + d) = make_float4(x[0], x[1], x[2], x[3]);
                    }
                    else {
#pragma unroll
                        for (int e = 0; e < 4; e++) x[e] = m > -INFINITY ? x[e] * inv : 0.f;
                        FlashTraits<TQ>::store4(y + d, x[0], x[1], x[2], x[3]);
                    }
                }
        }
    } else {
        // A value that is not finite lies where only some of the rows look, and weights of zero would not keep it from the others, or it has been cut in
        // parts, or parts do not hold what matters.  Row by row, then.
        for (int r = wave; r < nt * w.tileHeads; r += 4) {
            const int tk = r / w.tileHeads, hd = r - tk * w.tileHeads;
            if (hd >= nh) continue;
            const TQ* q = (const TQ*)a.q + row_at(tk, hd);
            float qv[2], acc[2] = {0.f, 0.f}, mr = -INFINITY, lr = 0.f;
#pragma unroll
            for (int i = 0; i < 2; i++) qv[i] = 2 * lane + i < c.hs ? value_of<TQ>(q[2 * lane + i]) : 0.f;
            for (int p = first * KB; p < stop * KB && p <= base + tk; p++) {
                const long long at = place_of(p, p < end ? page_at(p) : -1.f);
                if (at < 0) continue;
                float x = 0.f, val[2];
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const int d = 2 * lane + i;
                    x += d < c.hs ? qv[i] * value_of<TC>(kp[at + d]) : 0.f;
                    val[i] = d < c.hs ? value_of<TC>(vp[at + d]) : 0.f;
                }
                x = group_sum<64>(x) * a.c2;
                const float mn = fmaxf(mr, fmaxf(x, SCORE_FLOOR)), f = __builtin_amdgcn_exp2f(mr - mn), wt = __builtin_amdgcn_exp2f(x - mn);
                mr = mn;
                lr = lr * f + wt;
#pragma unroll
                for (int i = 0; i < 2; i++) acc[i] = acc[i] * f + wt * val[i];
            }
            if (2 * lane < c.hs) {
                if (!whole) *(float2*)(part + 256 + r * HSP + 2 * lane) = make_float2(acc[0], acc[1]);
                else if (L::SUMS) *(float2*)(list.sums_of(c, sp, sp.first + j0 + tk, h0 + hd, HSP) + 4 + 2 * lane) = make_float2(acc[0], acc[1]);
                else {
                    TQ* y = (TQ*)a.y + row_at(tk, hd) + 2 * lane;
                    y[0] = stored<TQ>(mr > -INFINITY ? acc[0] / lr : 0.f);
                    y[1] = stored<TQ>(mr > -INFINITY ? acc[1] / lr : 0.f);
                }
            }
            if (!whole && lane == 0) *(float2*)(part + 2 * r) = make_float2(mr, lr);
            if (L::SUMS && whole && lane == 0) *(float2*)list.sums_of(c, sp, sp.first + j0 + tk, h0 + hd, HSP) = make_float2(mr, lr);
        }
    }
    if (!L::SUMS && u0 == 0 && !whole && tid == 0) {
        const PagedRuns runs(at.total, blocks, CHUNK_LEAST);
        w.join[block] = ChunkJoin{at.place, runs.of(u + units - 1), sp.first + j0, h0, nt, nh, {0, 0}};
    }
    // ---- the next piece ----
    const int done = u1 - u0;
    u += done;
    at.local += done;
    if (u < hi) {
        const int all = L::SUMS ? paged_units_before(before, grow, (sp.count + w.perTile - 1) / w.perTile, w.unit) : chunk_work(c, w, PagedSpan{sp.first, sp.count, sp.len});
        if (at.local == all * groups) {
            at.local = 0;
            do {
                if (++at.b >= list.count(c)) return;
                at.sp = list.all_lanes(c, at.b);
            } while (chunk_tiles(c, w, PagedSpan{at.sp.first, at.sp.count, at.sp.len}) == 0);
        }
        __syncthreads();   // LDS is read no more
    }
    }
}

}  // namespace

}  // namespace mch
