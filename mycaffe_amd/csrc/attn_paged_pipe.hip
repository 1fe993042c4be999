// Attention of long chunks over a paged cache, 16-bit storage, head sizes 64 and 128: tiles of 256 rows, where there are enough of them for the chip.
//
// The wavefront is organised as in attn_flash2.hip, which says what bounds such a kernel (instruction issue and power beside the matrix cores) and how the
// three-stage pipeline inside a wavefront meets that: two tiles of 32 rows, the softmax of one next to the matrix products of the other, four stages of
// 64 keys in LDS, the masked blocks behind the loop.  What differs here:
//
//  * Rows are tokens times the heads that share a key head, so that a chunk of 64 tokens of four heads is a whole tile and its masked part 64 keys.
//  * Keys are counted from the first page that is given.  Where a key lies comes from the block table: four blocks ahead each wavefront looks sixteen keys
//    up and leaves their places in a ring of eight blocks in LDS (a place is 32 bits, in pieces of 16 bytes), from where the staging reads them.
//  * Weights are exp2(scale log2(e) s - m) with a fixed m a row: the largest score of its first 32 keys.  The scale stays in fp32 (one fused
//    multiply-add a score), and a row leaves the range only if a later score is higher by 44 than all of those.
//  * Weights are cut off to 16 bits and added up as they are then, so that a row's weights still sum to one: eight
//    bits each, y is off by 2.4e-3 of its norm, where its own rounding is 1.7e-3.  (A second product of what is cut off is half as many matrix instructions again.)
//  * What does not suit the pipeline is left to the chunk kernel, which runs behind this one for such tiles alone: tiles with a hole in their pages, rows
//    before the first page given, row sums outside [2^-60, 2^64], values that are not finite where not all rows look.
//
// Measured: 4 chunks of 1024 tokens over 8192 positions, 32 heads on 8 of 128, 515 GFLOP in 477 us (1080 TFLOP/s; a large library product has 1197).
#include <algorithm>
#include <type_traits>

#include "attn_paged.h"
#include "flash_pipe.h"
#include "kernels.h"

namespace mch {

namespace {

constexpr float PIPE_HI = 1.8446744e19f, PIPE_LO = 8.6736174e-19f;   // 2^64, 2^-60
constexpr int RING = 8;                                              // blocks whose places are kept

template <int HS>
__global__ __launch_bounds__(256, HS == 64 ? 2 : 1) void attn_paged_pipe_kernel(PagedAttnArgs a, ChunkArgs w, int* flags)
{
    typedef FlashTraits<bf16_t> TR;
    constexpr int NST = 4;                        // LDS stages of 64 keys
    constexpr int ROWB = HS * 2;                  // bytes of a key or value
    constexpr int BLKB = 64 * ROWB, VBASE = NST * BLKB, STEPB = 32 * ROWB;
    constexpr int KF = HS / 16, DT = HS / 32, NPV = 2 * DT, NSLOT = KF + NPV, EPS = 16 / NSLOT;
    constexpr int CPRW = ROWB / 16;               // 16-byte pieces of a key
    constexpr int CPW = 64 * CPRW / 256;          // pieces of a block and operand per lane
    static_assert((HS == 64 || HS == 128) && KF == NPV && 2 * CPW <= NSLOT, "tile / wavefront mismatch");
    extern __shared__ __attribute__((aligned(1024))) unsigned char pp_smem[];   // K stages, V stages, places
    uint32_t* ring = reinterpret_cast<uint32_t*>(pp_smem + 2 * VBASE);
    __shared__ int sFirst, sMissing, sBad;

    const PagedCache& c = a.c;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l32 = lane & 31, half = lane >> 5, i16 = lane & 15, g16 = (lane >> 4) & 1;

    // ---- the tile, and whether it is one for this kernel ----
    if (tid == 0) { sFirst = 0x7fffffff; sMissing = -1; sBad = 0; }
    const ChunkTile at = chunk_tile(c, w, blockIdx.x);
    if (at.b < 0) return;
    const PagedSpan sp = span_at(c, at.b);
    const int G = c.H / c.kvH, perTile = w.perTile * w.pair, j0 = at.tile * perTile, nt = min(perTile, sp.count - j0), base = sp.len - sp.count + j0;
    const int h0 = at.kh * G + at.ht * w.tileHeads, nh = min(w.tileHeads, G - at.ht * w.tileHeads);
    const int end = min(sp.len, base + nt), entries = end > 0 ? (end - 1) / c.pageSize + 1 : 0;
    const float* table = c.table + (size_t)at.b * c.maxPages;
    {
        int first = 0x7fffffff, missing = -1;
        for (int e = tid; e < entries; e += 256) {
            if (paged_page(table[e], c.pages) >= 0) first = min(first, e);
            else missing = e;
        }
        if (first < 0x7fffffff) atomicMin(&sFirst, first);
        if (missing >= 0) atomicMax(&sMissing, missing);
    }
    __syncthreads();
    const int given = uniform(sFirst), front = given < entries ? given * c.pageSize : 0;
    if (given >= entries || uniform(sMissing) > given || base < front) {
        if (tid == 0) flags[blockIdx.x] = 1;
        return;
    }
    const int Tk = end - front, lim0 = base - front;   // keys, and the last one that the tile's first token sees
    const unsigned char *kp = (const unsigned char*)((const bf16_t*)c.k + at.kh * c.sH), *vp = (const unsigned char*)((const bf16_t*)c.v + at.kh * c.sH);
    auto page_at = [&](int key) -> float { const int p = front + min(key, Tk - 1); return table[w.shift >= 0 ? p >> w.shift : p / c.pageSize]; };
    auto place_at = [&](int key, float entry) -> uint32_t {
        const int p = front + min(key, Tk - 1), slot = w.shift >= 0 ? p & (c.pageSize - 1) : p % c.pageSize;
        return (uint32_t)((max(paged_page(entry, c.pages), 0) * c.sP + slot * c.sT) >> 3);
    };

    // ---- the wavefront's two tiles (rows row0 .. + 31 and the 32 behind them) and their numbers of 32-key steps ----
    const int row0 = 64 * wave;
    int lim[2], firstLim[2], jobs[2];
#pragma unroll
    for (int x = 0; x < 2; x++) {
        const int r = row0 + 32 * x;
        lim[x] = lim0 + min((r + l32) / w.tileHeads, nt - 1);
        firstLim[x] = lim0 + min(r / w.tileHeads, nt - 1);
        jobs[x] = ((lim0 + min((r + 31) / w.tileHeads, nt - 1)) >> 5) + 1;
    }
    const int nplain = (firstLim[0] + 1) >> 5;         // steps that all rows see whole
    const int nkb = (Tk + 63) >> 6;

    // ---- staging: piece e = tid + 256 i of a block is 16-byte piece e % CPRW of key e / CPRW; in LDS it sits at piece position
    // (e % CPRW) ^ swizzle(key) of its key ----
    unsigned dstK[CPW], dstV[CPW];
    const int srow = tid / CPRW, scp = (tid % CPRW) << 4;
#pragma unroll
    for (int i = 0; i < CPW; i++) {
        const int row = srow + 256 / CPRW * i, cp = tid % CPRW;
        const int swK = HS == 64 ? (row >> 1) & 7 : row & 15;
        const int swV = HS == 64 ? 4 * ((row >> 1) & 1) : 4 * (row & 3);
        dstK[i] = row * ROWB + ((cp ^ swK) << 4);
        dstV[i] = VBASE + row * ROWB + ((cp ^ swV) << 4);
    }
    u32x4 st[2 * CPW];     // piece i of the K block (i < CPW) or the V block (i >= CPW) on its way from memory to LDS
    uint32_t place[CPW];   // where the pieces of the block that is requested next lie
    auto places_of = [&](int kb) {
#pragma unroll
        for (int i = 0; i < CPW; i++) place[i] = ring[(kb & (RING - 1)) * 64 + srow + 256 / CPRW * i];
    };
    auto gload = [&](u32x4& dst, int i) { dst = *(const u32x4*)((i < CPW ? kp : vp) + ((size_t)place[i % CPW] << 4) + scp); };
    auto sstore_piece = [&](const u32x4& src, int stageOff, int i) { *(u32x4*)(pp_smem + stageOff + (i < CPW ? dstK[i] : dstV[i - CPW])) = src; };
    auto stage_of = [&](int kb) { return (kb & (NST - 1)) * BLKB; };
    // The block that travels to stage_of(j) as "block j".  Past the last block it is the block that lives in that stage already (the same bytes once
    // more), so that after the last block the stages still hold the last NST blocks.
    auto staged_block = [&](int j) { return j < nkb ? j : max(j - NST, 0); };

    // ---- Q fragments (they carry the scale's sign) ----
    u32x4 qf[2][KF];
    const float c2 = fabsf(a.c2);
#pragma unroll
    for (int x = 0; x < 2; x++) {
        const int row = row0 + 32 * x + l32, token = row / w.tileHeads, head = row - token * w.tileHeads;
        const bool live = token < nt && head < nh;
        const bf16_t* q = (const bf16_t*)a.q + (live ? ((size_t)(sp.first + j0 + token) * c.H + h0 + head) * HS : 0);
#pragma unroll
        for (int f = 0; f < KF; f++) {
            qf[x][f] = live ? *(const u32x4*)(q + f * 16 + half * 8) : u32x4{0u, 0u, 0u, 0u};
            if (a.c2 < 0.f) qf[x][f] ^= u32x4{0x80008000u, 0x80008000u, 0x80008000u, 0x80008000u};
        }
    }

    // ---- fragment addresses in LDS ----
    // K fragment f of a step: key 32 (step & 1) + l32 of the step's block, piece 2 f + half
    int klane[KF];
#pragma unroll
    for (int f = 0; f < KF; f++) klane[f] = l32 * ROWB + (((2 * f + half) ^ (HS == 64 ? (l32 >> 1) & 7 : l32 & 15)) << 4);
    // V^T fragment (tt, dt): two transposing reads of four keys each; this lane supplies key 16 tt + 4 half + i16 / 4 (+ 8 for the second read),
    // bytes 64 dt + 32 g16 + 8 (i16 % 4) .. + 7 of it
    int vlane[DT];
#pragma unroll
    for (int dt = 0; dt < DT; dt++)
        vlane[dt] = VBASE + (4 * half + (i16 >> 2)) * ROWB + ((dt ^ (HS == 64 ? (i16 >> 3) & 1 : (i16 >> 2) & 3)) << 6) + g16 * 32 + (i16 & 3) * 8;
    // off: byte offset of the step inside the stages (stage of its block, plus half a block for an odd step)
    auto ldK = [&](int f, int off) -> u32x4 { return *(const u32x4*)(pp_smem + klane[f] + off); };
    auto ldV = [&](int idx, int off) -> u32x4 {   // idx = tt * DT + dt
        const bf16_t* p = (const bf16_t*)(pp_smem + vlane[idx % DT] + off + (idx / DT) * 16 * ROWB);
        const uint2 lo = lds_read_tr16(p), hi = lds_read_tr16(p + 8 * HS);
        return u32x4{lo.x, lo.y, hi.x, hi.y};
    };

    // ---- state ----
    // o[X]: output tiles, sb[X]: scores of tile X's next job, pkb[X]: packed weights of tile X's latest job, fr: the K fragments (0 .. KF) and V^T
    // fragments (KF ..) the coming MFMAs multiply with, ls[X]: the row sums so far (two partial sums each), nref[X]: minus the row's m
    floatx16 o[2][DT], sb[2];
    u32x4 pkb[2][2], fr[NSLOT];
    float ls[2][2] = {{0.f, 0.f}, {0.f, 0.f}}, nref[2];
    float exc0 = 0.f, exc1 = 0.f;   // the last two exponentials of the latest pinned phase, not yet packed
    const floatx16 zero16 = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};

    // ---- places of the first blocks; blocks 0 and 1 into their stages, block 2 requested ----
    ring[tid] = place_at(tid, page_at(tid));
    const int aheadKey = 16 * wave + i16;              // of a block: the key this lane looks up (four lanes alike)
    float entry = page_at(4 * 64 + aheadKey);
    __syncthreads();
    // the places of block kb + 4 into the ring, the table's entries for the one behind it requested
    auto look_ahead = [&](int kb) {
        if (kb + 4 < nkb) {
            if (lane < 16) ring[((kb + 4) & (RING - 1)) * 64 + aheadKey] = place_at((kb + 4) * 64 + aheadKey, entry);
            entry = page_at((kb + 5) * 64 + aheadKey);
        }
    };
    {
        places_of(0);
#pragma unroll
        for (int i = 0; i < 2 * CPW; i++) gload(st[i], i);
        places_of(staged_block(1));
#pragma unroll
        for (int i = 0; i < 2 * CPW; i++) gload(fr[i], i);
#pragma unroll
        for (int i = 0; i < 2 * CPW; i++) sstore_piece(st[i], stage_of(0), i);
        places_of(staged_block(2));
#pragma unroll
        for (int i = 0; i < 2 * CPW; i++) gload(st[i], i);
#pragma unroll
        for (int i = 0; i < 2 * CPW; i++) sstore_piece(fr[i], stage_of(1), i);
        __syncthreads();
    }
    // one block of the plain loops: block kb + 2 from the staging registers to its stage, block kb + 3 requested
    auto stage_step = [&](int kb) {
#pragma unroll
        for (int i = 0; i < 2 * CPW; i++) sstore_piece(st[i], stage_of(kb + 2), i);
        places_of(staged_block(kb + 3));
#pragma unroll
        for (int i = 0; i < 2 * CPW; i++) gload(st[i], i);
        look_ahead(kb);
    };
#pragma unroll
    for (int x = 0; x < 2; x++) {
        sb[x] = zero16;
        asm volatile("" : "+v"(sb[x]));
#pragma unroll
        for (int dt = 0; dt < DT; dt++) {
            o[x][dt] = zero16;
            asm volatile("" : "+a"(o[x][dt]));
        }
        pkb[x][0] = pkb[x][1] = u32x4{0u, 0u, 0u, 0u};
#pragma unroll
        for (int f = 0; f < KF; f++) asm volatile("" : "+a"(qf[x][f]));
    }
#pragma unroll
    for (int j = 0; j < NSLOT; j++) fr[j] = u32x4{0u, 0u, 0u, 0u};

    // softmax of one job, one instruction after the other: weights into pk, their sum into the row sums
    auto soft_seq = [&](auto x_, int step, bool plain, floatx16& sc, u32x4 (&pk)[2]) __attribute__((always_inline)) {
        constexpr int X = decltype(x_)::value;
        if (!plain) {
#pragma unroll
            for (int v = 0; v < 16; v++)
                if (step * 32 + 8 * (v >> 2) + 4 * half + (v & 3) > lim[X]) sc[v] = -INFINITY;
        }
        uint32_t wt[8];
#pragma unroll
        for (int q = 0; q < 8; q++) {
            wt[q] = f2_pack_trunc(__builtin_amdgcn_exp2f(fmaf(sc[2 * q], c2, nref[X])), __builtin_amdgcn_exp2f(fmaf(sc[2 * q + 1], c2, nref[X])));
            ls[X][q & 1] = f2_dot2_ones(wt[q], ls[X][q & 1]);
        }
        pk[0] = u32x4{wt[0], wt[1], wt[2], wt[3]};
        pk[1] = u32x4{wt[4], wt[5], wt[6], wt[7]};
    };
    auto pv_regs = [&](auto x_) {   // O^T += V^T P^T of tile X's latest job, V^T fragments from fr[KF ..)
        constexpr int X = decltype(x_)::value;
#pragma unroll
        for (int idx = 0; idx < NPV; idx++) f2_mma_o_acc(o[X][idx % DT], fr[KF + idx], pkb[X][idx / DT]);
    };
    // one whole job, nothing overlapped: used where a step needs a mask.  off: the step's byte offset in the stages
    auto cold_job = [&](auto x_, int step, int off) __attribute__((always_inline)) {
        constexpr int X = decltype(x_)::value;
        floatx16 t = zero16;
#pragma unroll
        for (int f = 0; f < KF; f++) t = TR::mma(ldK(f, off), qf[X][f], t);
        asm volatile("" : "+v"(t));   // the score tiles live in vector registers throughout
        sb[X] = t;
        soft_seq(x_, step, step * 32 + 31 <= firstLim[X], sb[X], pkb[X]);
#pragma unroll
        for (int idx = 0; idx < NPV; idx++) f2_mma_o_acc(o[X][idx % DT], ldV(idx, off), pkb[X][idx / DT]);
    };

    // One pinned phase of NSLOT slots, an MFMA each: the softmax of tile TS's job (scores sb[TS] -> weights pkb[TS]) next to the other tile's MFMAs - S^T of its
    // next job (into sb[1 - TS]) and O^T += V^T P^T of its latest one (weights pkb[1 - TS]) - all on the fragments in fr.  The softmax is spread
    // evenly: EPS exponentials a slot, a pair packed one slot after its second exponential and added to the row sum a slot after that; what
    // would fall behind the last slot is done in the first slots of the next phase.
    // RELOAD: behind every MFMA the fragment it used is replaced by the one at byte offset koff / voff.
    // PH (0 .. 3): the phase's share of the staging - pieces PH * PPP .. of the block two ahead go from their registers to the stage at sOff, and
    // the same pieces of the block three ahead (at `place`) are requested.
    constexpr int PPP = 2 * CPW / 4;
    static_assert(2 * CPW % 4 == 0 && PPP <= NSLOT / 2, "staging pieces per phase");
    auto hot_phase = [&](auto ts_, auto reload_, auto ph_, int koff, int voff, int sOff) __attribute__((always_inline)) {
        constexpr int TS = decltype(ts_)::value, TO = 1 - TS, PH = decltype(ph_)::value;
        constexpr bool RELOAD = decltype(reload_)::value;
        floatx16& sc = sb[TS];
        float ex[16];
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < NSLOT; j++) {
            // even slots: S^T, odd slots: O^T
            if (!(j & 1)) {
                const int f = j >> 1;
                if (f == 0) f2_mma_s_first(sb[TO], fr[f], qf[TO][f]);
                else f2_mma_s_acc(sb[TO], fr[f], qf[TO][f]);
                if (RELOAD) fr[f] = ldK(f, koff);
            } else {
                const int idx = j >> 1;
                f2_mma_o_acc(o[TO][idx % DT], fr[KF + idx], pkb[TO][idx / DT]);
                if (RELOAD) fr[KF + idx] = ldV(idx, voff);
            }
            if ((j & 1) && (j >> 1) < PPP) {
                const int i = PH * PPP + (j >> 1);
                sstore_piece(st[i], sOff, i);
                gload(st[i], i);
            }
#pragma unroll
            for (int e = j * EPS; e < (j + 1) * EPS; e++) {
                ex[e] = __builtin_amdgcn_exp2f(fmaf(sc[e], c2, nref[TS]));
                asm volatile("" : "+v"(ex[e]));   // keeps the instructions in this slot
            }
#pragma unroll
            for (int q = 0; q < 8; q++) {
                const int cs = (2 * q + 1) / EPS + 1;   // the slot that packs pair q, the next one adds it up
                if (cs == j) {
                    uint32_t x = f2_pack_trunc(ex[2 * q], ex[2 * q + 1]);
                    asm volatile("" : "+v"(x));
                    pkb[TS][q >> 2][q & 3] = x;
                }
                if (cs == j + NSLOT) {                  // q == 7 of the previous phase's job
                    uint32_t x = f2_pack_trunc(exc0, exc1);
                    asm volatile("" : "+v"(x));
                    pkb[TO][q >> 2][q & 3] = x;
                }
                if (cs + 1 == j) {
                    ls[TS][q & 1] = f2_dot2_ones(pkb[TS][q >> 2][q & 3], ls[TS][q & 1]);
                    asm volatile("" : "+v"(ls[TS][q & 1]));
                }
                if (cs + 1 == j + NSLOT) {
                    ls[TO][q & 1] = f2_dot2_ones(pkb[TO][q >> 2][q & 3], ls[TO][q & 1]);
                    asm volatile("" : "+v"(ls[TO][q & 1]));
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        exc0 = ex[14];
        exc1 = ex[15];
    };
    // what the last pinned phase (softmax of tile X) left for the first slots of a next one
    auto hot_tail = [&](auto x_) {
        constexpr int X = decltype(x_)::value;
        pkb[X][1][3] = f2_pack_trunc(exc0, exc1);
#pragma unroll
        for (int q = 0; q < 8; q++)
            if ((2 * q + 1) / EPS + 2 >= NSLOT) ls[X][q & 1] = f2_dot2_ones(pkb[X][q >> 2][q & 3], ls[X][q & 1]);
        exc0 = exc1 = 0.f;
    };
    typedef std::integral_constant<int, 0> I0;
    typedef std::integral_constant<int, 1> I1;
    typedef std::integral_constant<int, 2> I2;
    typedef std::integral_constant<int, 3> I3;
    typedef std::integral_constant<bool, false> BF;
    typedef std::integral_constant<bool, true> BT;

    // the K fragments of step 0, the rows' m from them, and S^T of tile 0's first job
#pragma unroll
    for (int f = 0; f < KF; f++) fr[f] = ldK(f, 0);
#pragma unroll
    for (int x = 1; x >= 0; x--) {
        floatx16 t = zero16;
#pragma unroll
        for (int f = 0; f < KF; f++) t = TR::mma(fr[f], qf[x][f], t);
        asm volatile("" : "+v"(t));
        float mx = -INFINITY;
#pragma unroll
        for (int v = 0; v < 16; v++) mx = fmaxf(mx, 8 * (v >> 2) + 4 * half + (v & 3) <= lim[x] ? t[v] : -INFINITY);
        nref[x] = -(f2_pair_max(mx) * c2);
        if (x == 0) sb[0] = t;
    }

    // Blocks whose two steps need no mask in either tile: four pinned phases each.  Going in, sb[0] holds tile 0's scores of the block's first step; tile 1's
    // latest weights (pkb[1], their V^T fragments in fr) are multiplied in the first phase - zeros before the first block.
    // Staging.  Going into block kb, blocks kb and kb + 1 are in their stages and the staging registers hold block kb + 2.  During the block they are written to
    // the stage that block kb - 2 had - every wavefront left it before the barrier of block kb - 1 - and are read from the second half of block kb + 1
    // on, behind that block's barrier.  Places written before the barrier of block kb are read from block kb + 1 on; the slot had been read for the
    // last time before the barrier of block kb - 3.
    int kb = 0;
    const int nhot = min(nkb, nplain >> 1);
    for (; kb < nhot; kb++) {
        const int cur = stage_of(kb), nxt = stage_of(kb + 1), wst = stage_of(kb + 2);
        places_of(staged_block(kb + 3));
        look_ahead(kb);
        hot_phase(I0{}, BT{}, I0{}, cur + STEPB, cur, wst);
        hot_phase(I1{}, BF{}, I1{}, 0, 0, wst);
        __syncthreads();
        hot_phase(I0{}, BT{}, I2{}, nxt, cur + STEPB, wst);
        hot_phase(I1{}, BF{}, I3{}, 0, 0, wst);
    }
    hot_tail(I1{});
    pv_regs(I1{});
    // the remaining blocks, one job after the other; the last NST, which stay in their stages, behind the loop, all wavefronts at once
    auto cold_block = [&](int kb) __attribute__((always_inline)) {
        const int t0 = 2 * kb, cur = stage_of(kb);
        if (t0 < jobs[0]) cold_job(I0{}, t0, cur);
        if (t0 < jobs[1]) cold_job(I1{}, t0, cur);
        if (t0 + 1 < jobs[0]) cold_job(I0{}, t0 + 1, cur + STEPB);
        if (t0 + 1 < jobs[1]) cold_job(I1{}, t0 + 1, cur + STEPB);
    };
    const int kbLate = max(kb, nkb - NST);
    for (; kb < nkb; kb++) {
        stage_step(kb);
        if (kb < kbLate) cold_block(kb);
        __syncthreads();
    }
    for (kb = kbLate; kb < nkb; kb++) cold_block(kb);

    // ---- what the tile's rows cannot be trusted with: sums out of range, values of later tokens that are not finite ----
    float lsum[2];
    bool bad = false;
#pragma unroll
    for (int x = 0; x < 2; x++) {
        lsum[x] = f2_pair_sum(ls[x][0] + ls[x][1]);
        bad = bad || !(lsum[x] >= PIPE_LO && lsum[x] <= PIPE_HI);
    }
    for (int e = tid; e < (nt - 1) * CPRW; e += 256) {
        const int key = lim0 + 1 + e / CPRW;
        const u32x4 v = *(const u32x4*)(vp + ((size_t)place_at(key, page_at(key)) << 4) + ((e % CPRW) << 4));
#pragma unroll
        for (int i = 0; i < 4; i++) bad = bad || (v[i] & 0x7f80u) == 0x7f80u || (v[i] & 0x7f800000u) == 0x7f800000u;
    }
    __syncthreads();   // everybody is done with the stages

    // ---- y = O^T / l; register v of tile dt is value 32 dt + 8 (v / 4) + 4 half + v % 4.  A lane owns a row, so its values are scattered over it; they go
    // through the wavefront's own 64 rows of LDS and leave as whole rows, 16 bytes a lane.  The pieces of a row are permuted by its number so that
    // neither side piles up on a few banks. ----
    static_assert(4 * BLKB <= 2 * VBASE, "one block of LDS per wavefront");
    unsigned char* ybuf = pp_smem + wave * BLKB;
#pragma unroll
    for (int x = 0; x < 2; x++) {
        const int r = 32 * x + l32;
        const float inv = 1.0f / lsum[x];
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
#pragma unroll
            for (int g = 0; g < 4; g++) {
                float y[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float v = o[x][dt][4 * g + i];
                    bad = bad || (__float_as_uint(v) & 0x7f800000u) == 0x7f800000u;
                    y[i] = v * inv;
                }
                *(uint2*)(ybuf + r * ROWB + (((4 * dt + g) ^ (r & (CPRW - 1))) << 4) + 8 * half) = make_uint2(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]));
            }
    }
    wave_lds_fence();
#pragma unroll
    for (int i = 0; i < CPRW; i++) {
        const int e = lane + 64 * i, r = e / CPRW, piece = e % CPRW, row = row0 + r, token = row / w.tileHeads, head = row - token * w.tileHeads;
        const u32x4 v = *(const u32x4*)(ybuf + r * ROWB + ((piece ^ (r & (CPRW - 1))) << 4));
        if (token < nt && head < nh) *(u32x4*)((bf16_t*)a.y + ((size_t)(sp.first + j0 + token) * c.H + h0 + head) * HS + piece * 8) = v;
    }
    if (__any(bad) && lane == 0) sBad = 1;
    __syncthreads();
    if (tid == 0) flags[blockIdx.x] = sBad;
}

template <int HS> hipError_t pipe_launch(hipStream_t s, const PagedAttnArgs& a, const ChunkArgs& w, int blocks, int* flags)
{
    constexpr int LDSB = 2 * 4 * 64 * HS * 2 + RING * 64 * 4;   // four K and four V stages, the places
    static bool attr = false;
    if (!attr) {
        const hipError_t e = hipFuncSetAttribute((const void*)attn_paged_pipe_kernel<HS>, hipFuncAttributeMaxDynamicSharedMemorySize, LDSB);
        if (e != hipSuccess) return e;
        attr = true;
    }
    hipLaunchKernelGGL((attn_paged_pipe_kernel<HS>), blocks, 256, LDSB, s, a, w, flags);
    return hipGetLastError();
}

}  // namespace

hipError_t attn_paged_pipe_launch(hipStream_t s, const PagedAttnArgs& a, const ChunkArgs& w, int blocks, int* flags)
{
    return a.c.hs == 64 ? pipe_launch<64>(s, a, w, blocks, flags) : pipe_launch<128>(s, a, w, blocks, flags);
}

}  // namespace mch
