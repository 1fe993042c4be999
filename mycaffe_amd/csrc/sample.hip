// The next token of every row of logits, drawn with a given random number.
//
// Weights w_i = exp((x_i - max x) / T).  Of the tokens in falling order of x, equal ones by their index: top-k keeps the first k, top-p of these the shortest run
// whose weights add up to at least p of theirs, min-p those with w >= m.  Drawn is the first token, in the order of the vocabulary, at which the sum of the weights of
// those that are left exceeds u times all of it.
//
// A draw compares u with sums over the whole vocabulary: a sum that is off by e moves every border by e, so with 100000 tokens fp32 sums draw another token every
// few hundred rows.  Weights are made in 64 bits, to 2^-48.5 of themselves, and held as whole numbers of 2^-FB of the largest, FB = 50 and less above 2^13 tokens (sample_bits: 46 at
// 131072), which add up to the same in any order; their sums are exact.
//
// A logit takes some 20 instructions of 64 bits where its weight counts, and none where only its place does (top-k): long rows are bound by these, and by their bins, short ones by one
// pass and one barrier behind the other.  A row is one workgroup's, its logits read two or three times (they stay in the caches); or slices of it are (below).  Measured, with
// rows that no cache of an XCD holds: top-p of a row of 32000 in fp32 24 - 25 us; 64 rows of 50261 in fp32, top-50, 27 us; 256 rows of 131072 in 16 bits with settings of their own 86 us
// (67 MB; largest logits 13, weights 35, borders 8, candidates 17, the rest 17); 48 rows of 200003 in 16 bits by temperature alone 23 us.
#include <algorithm>
#include <type_traits>

#include "kernels.h"
#include "lane_ops.h"

namespace mch {

namespace {

constexpr int THREADS = 1024, WAVES = THREADS / 64, BINS = 2048, FEW = 256;
static_assert(FEW <= THREADS / 4 && 2 * FEW <= BINS, "Rank, draw_of_few()");
typedef unsigned long long u64;
constexpr u64 RAW = 0x4330000000000000ull;   // the upper bits of a whole number in a double

// a b + c in a register of its own (the compiler copies c first and adds to the copy)
__device__ __forceinline__ double fma3(double a, double b, double c)
{
    double d;
    asm("v_fma_f64 %0, %1, %2, %3" : "=v"(d) : "v"(a), "v"(b), "v"(c));
    return d;
}

template <typename L> struct Logit {   // fp32, bf16 as fp32: keys of 32 bits; double: of 64
    typedef float V;
    typedef uint32_t K;
};
template <> struct Logit<double> {
    typedef double V;
    typedef u64 K;
};
__device__ __forceinline__ float read(float x) { return x; }
__device__ __forceinline__ float read(bf16_t x) { return bf16_to_f32(x); }
__device__ __forceinline__ double read(double x) { return x; }
// whole numbers in the order of the logits
__device__ __forceinline__ uint32_t key_of(float x)
{
    const uint32_t u = __float_as_uint(x);
    return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float(k ^ ((uint32_t)~((int32_t)k >> 31) | 0x80000000u)); }
__device__ __forceinline__ double of_key(u64 k) { return __longlong_as_double((long long)(k ^ ((u64)~((long long)k >> 63) | 0x8000000000000000ull))); }
__device__ __forceinline__ u64 key_of(double x)
{
    const u64 u = (u64)__double_as_longlong(x);
    return u ^ ((u64)((long long)u >> 63) | 0x8000000000000000ull);
}

template <int CTRL, int ROWS> __device__ __forceinline__ u64 dpp64(u64 v)   // 0 where there is no such lane
{
    const uint32_t lo = __builtin_amdgcn_update_dpp(0u, (uint32_t)v, CTRL, ROWS, 0xf, false), hi = __builtin_amdgcn_update_dpp(0u, (uint32_t)(v >> 32), CTRL, ROWS, 0xf, false);
    return (u64)hi << 32 | lo;
}
__device__ __forceinline__ u64 wave_scan(u64 v)   // up to and with the lane's own: within rows of sixteen lanes, then the rows before
{
    v += dpp64<0x111, 0xf>(v);   // row_shr 1, 2, 4, 8
    v += dpp64<0x112, 0xf>(v);
    v += dpp64<0x114, 0xf>(v);
    v += dpp64<0x118, 0xf>(v);
    v += dpp64<0x142, 0xa>(v);   // row_bcast 15 to rows 1 and 3
    return v + dpp64<0x143, 0xc>(v);   // row_bcast 31 to rows 2 and 3
}
__device__ __forceinline__ u64 lane_of(u64 v, int lane)
{
    return (u64)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)v, lane);
}
__device__ __forceinline__ u64 wave_sum(u64 v)
{
    v = wave_scan(v);
    return lane_of(v, 63);
}
__device__ __forceinline__ u64 shfl_xor64(u64 v, int o)
{
    const uint32_t lo = __shfl_xor((uint32_t)v, o), hi = __shfl_xor((uint32_t)(v >> 32), o);
    return (u64)hi << 32 | lo;
}
// over the workgroup: the sum before the thread's own, and of all (sums: WAVES numbers, read until the next barrier)
template <int WAVES = THREADS / 64> __device__ __forceinline__ u64 block_scan(u64 v, u64* sums, u64* all)
{
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const u64 x = wave_scan(v);
    __syncthreads();
    if (lane == 63) sums[wave] = x;
    __syncthreads();
    u64 each = sums[lane & (WAVES - 1)];   // sums of the wavefronts up to the lane's
    each += dpp64<0x111, 0xf>(each);
    each += dpp64<0x112, 0xf>(each);
    if (WAVES > 4) each += dpp64<0x114, 0xf>(each);
    if (WAVES > 8) each += dpp64<0x118, 0xf>(each);
    *all = lane_of(each, WAVES - 1);
    return (wave ? lane_of(each, wave ? wave - 1 : 0) : 0) + x - v;
}

// 2^(j / 32), rounded to nearest
__device__ const double ROOTS[32] = {1.0, 1.0218971486541166, 1.0442737824274138, 1.0671404006768237, 1.0905077326652577, 1.1143867425958924,
                                     1.1387886347566916, 1.1637248587775775, 1.189207115002721, 1.215247359980469, 1.241857812073484, 1.2690509571917332,
                                     1.2968395546510096, 1.3252366431597413, 1.3542555469368927, 1.383909881963832, 1.4142135623730951, 1.4451808069770467,
                                     1.4768261459394993, 1.5091644275934228, 1.5422108254079407, 1.5759808451078865, 1.6104903319492543, 1.645755478153965,
                                     1.681792830507429, 1.718619298122478, 1.7562521603732995, 1.7947090750031072, 1.8340080864093424, 1.8741676341103,
                                     1.9152065613971474, 1.9571441241754002};

// The row's logits and their weights.  Powers are counted in 32nds: weight = 2^(power / 32).
template <typename L> struct Row {
    typedef L L_;
    typedef typename Logit<L>::V V;
    typedef typename Logit<L>::K K;
    static constexpr int VEC = 16 / (int)sizeof(L), CHUNK = 64 * VEC, SIDE = VEC < 4 ? VEC : 4;   // logits of a lane's piece, of a wavefront's, of those that are worked on side by side
    const L* x;
    int vocab, perWave;   // chunks of a wavefront, which has one run of them
    V top;
    double rate;          // 32 log2(e) / T
    double least;         // powers from here down are weights of 0
    int bits;             // FB
    bool infinite;        // the largest logit is
    const double* roots;

    __device__ __forceinline__ void fetch(int i0, L (&raw)[VEC]) const   // those behind the row's end: -inf
    {
        if (i0 + VEC <= vocab) __builtin_memcpy(raw, x + i0, sizeof(raw));
        else
#pragma unroll
            for (int e = 0; e < VEC; e++) {
                if constexpr (sizeof(L) == 2) raw[e] = i0 + e < vocab ? x[i0 + e] : (L)0xff80;
                else raw[e] = i0 + e < vocab ? x[i0 + e] : -(L)INFINITY;
            }
    }
    // VEC logits (those that are not a number fail every comparison below, and weigh nothing); beside infinite ones nothing else is drawn, and they are all 0
    __device__ __forceinline__ void logits(const L (&raw)[VEC], V (&v)[VEC]) const
    {
#pragma unroll
        for (int e = 0; e < VEC; e++) v[e] = read(raw[e]);
        if (infinite)
#pragma unroll
            for (int e = 0; e < VEC; e++) v[e] = v[e] == (V)INFINITY ? (V)0 : -(V)INFINITY;
    }
    // the pieces of the wavefront in the order of the vocabulary, the next ones under way: f(chunk, first index, VEC logits)
    template <typename F> __device__ __forceinline__ void each(F f) const
    {
        constexpr int DEEP = 3;
        const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const int from = wave * perWave, to = min(from + perWave, (vocab + CHUNK - 1) / CHUNK);
        L next[DEEP][VEC];
#pragma unroll
        for (int d = 0; d < DEEP; d++) fetch((from + d) * CHUNK + lane * VEC, next[d]);
#pragma unroll 1
        for (int chunk = from; chunk < to; chunk++) {
            V v[VEC];
            logits(next[0], v);
#pragma unroll
            for (int d = 0; d + 1 < DEEP; d++)
#pragma unroll
                for (int e = 0; e < VEC; e++) next[d][e] = next[d + 1][e];
            fetch((chunk + DEEP) * CHUNK + lane * VEC, next[DEEP - 1]);
            f(chunk, chunk * CHUNK + lane * VEC, v);
        }
    }
    // 32 log2 of the weight, `least` where there is none
    __device__ __forceinline__ double power(V v) const { return fmax(((double)v - (double)top) * rate, least); }
    // 2^(y / 32) for y of -32000 .. 0 as a fraction p of 1/2 .. 2 and a whole power of 2: a 32nd from the table times the series of 2^(f / 32), |f| <= 1/2, whose
    // sixth term is 2^-49
    __device__ __forceinline__ double two_to(double y, int more) const
    {
        const double k = y + 0x1.8p52, f = y - (k - 0x1.8p52);   // rounded to a whole number, which the sum's lower half is
        const int n = __double2loint(k);
        double s = fma3(f, 3.973709984549416e-11, 9.172562701824643e-09);
        s = fma3(f, s, 1.693850972437182e-06);
        s = fma3(f, s, 0.0002345961982022468);
        s = fma3(f, s, 0.02166084939249829);
        s = fma(f, s, 1.0) * roots[n & 31];
        return __hiloint2double(__double2hiint(s) + (int)((uint32_t)n << 15 & 0xfff00000u) + (more << 20), __double2loint(s));
    }
    // 2^FB times the weight as a whole number, in the lower 52 bits of one with 0x433 above them; sums are taken of these, and the 0x433 taken off
    __device__ __forceinline__ u64 raw_weight(V v) const { return (u64)__double_as_longlong(two_to(power(v), bits) + 0x1p52); }
    __device__ __forceinline__ u64 weight(V v) const { return raw_weight(v) - RAW; }
    // falling logits in rising numbers, `scale` bins a unit and twice that a half; not a number or behind the bins where there is no weight
    __device__ __forceinline__ V bins(V v, V half, V scale) const { return __builtin_fma(v, (V)-0.5, half) * scale; }
    // the smallest number, up to the largest logit, for which `is` holds, which is for larger ones too: 64 are tried at a time
    template <typename F> __device__ __forceinline__ V smallest(F is) const
    {
        const int lane = threadIdx.x & 63;
        K lo = key_of(-(V)INFINITY), hi = key_of(top);   // of hi it holds
#pragma unroll 1
        while (hi - lo > 0) {
            const K step = (hi - lo) / 64, at = lo + step * (K)lane + (K)lane * ((hi - lo) % 64) / 64;   // rising from lo, below hi
            const u64 m = __ballot(is(of_key(at)));
            const int first = m ? __builtin_ctzll(m) : 64;
            const K here = first < 64 ? lane_key(at, first) : hi;
            lo = first > 0 ? lane_key(at, first - 1) + 1 : lo;
            hi = first == 0 ? lo : here;
        }
        return of_key(hi);
    }
    __device__ static uint32_t lane_key(uint32_t k, int lane) { return (uint32_t)__builtin_amdgcn_readlane((int)k, lane); }
    __device__ static u64 lane_key(u64 k, int lane) { return lane_of(k, lane); }
};

struct Shared {
    uint32_t count[BINS];
    u64 weight[BINS];
    u64 sums[WAVES];
    double roots[32];
    double values[FEW];
    u64 weights[FEW], kept[FEW];
    int ids[FEW];
    u64 above, least, most;
    double value;
    int bin, listed, index, found, reached;
};

// p in 0 .. 1 as a fraction of 2^64
__device__ __forceinline__ u64 fraction(double p) { return p >= 1.0 ? ~0ull : p > 0.0 ? (u64)(p * 18446744073709551616.0) : 0; }

// the first index at which the sum of one(logit, index) exceeds target(sum of all); piece(logits, first index): the sum over a lane's.  All threads; -1 if there is none
template <typename R, typename F, typename F1, typename G> __device__ __forceinline__ int locate(const R& r, Shared& s, u64* parts, F piece, F1 one, G target, u64* total)
{
    const int lane = threadIdx.x & 63, tid = threadIdx.x, chunks = r.perWave * WAVES, per = (chunks + THREADS - 1) / THREADS;
    for (int i = tid; i < chunks; i += THREADS) parts[i] = 0;
    if (tid == 0) s.found = -1;
    __syncthreads();
    r.each([&](int chunk, int i0, const typename R::V (&v)[R::VEC]) __attribute__((always_inline)) {
        const u64 w = wave_sum(piece(v, i0));
        if (lane == 0) parts[chunk] = w;
    });
    __syncthreads();
    u64 mine = 0;
    for (int i = tid * per; i < min(chunks, (tid + 1) * per); i++) mine += parts[i];
    u64 before = block_scan(mine, s.sums, total);
    const u64 want = target(*total);
    if (before <= want && want < before + mine)
        for (int i = tid * per; i < min(chunks, (tid + 1) * per); i++) {
            if (want < before + parts[i]) { s.found = i; s.above = before; break; }
            before += parts[i];
        }
    __syncthreads();
    const int chunk = s.found;
    const u64 start = s.above;
    __syncthreads();
    if (chunk < 0) return -1;
    if (tid < 64) {
        typename R::L_ raw[R::VEC];
        typename R::V v[R::VEC];
        u64 w[R::VEC], all = 0;
        const int i0 = chunk * R::CHUNK + lane * R::VEC;
        r.fetch(i0, raw);
        r.logits(raw, v);
#pragma unroll
        for (int e = 0; e < R::VEC; e++) {
            w[e] = one(v[e], i0 + e);
            all += w[e];
        }
        u64 at = start + wave_scan(all) - all;
#pragma unroll
        for (int e = 0; e < R::VEC; e++) {
            if (at <= want && want < at + w[e]) s.found = i0 + e;
            at += w[e];
        }
    }
    __syncthreads();
    const int i = s.found;
    __syncthreads();
    return i;
}
// the index of the `count`-th logit that is v0 and kept by `old`
template <typename R, typename B> __device__ __forceinline__ int locate_equal(const R& r, Shared& s, u64* parts, typename R::V v0, const B& old, u64 count)
{
    u64 total;
    return locate(r, s, parts, [&](const typename R::V (&v)[R::VEC], int i0) __attribute__((always_inline)) -> u64 {
        uint32_t n = 0;
#pragma unroll
        for (int e = 0; e < R::VEC; e++) n += v[e] == v0 && old.has(v[e], i0 + e);
        return n;
    }, [&](typename R::V v, int i) __attribute__((always_inline)) -> u64 { return v == v0 && old.has(v, i); }, [&](u64) { return count - 1; }, &total);
}

// what a row is drawn by
struct Settings {
    bool first, byK, byP;   // the largest logit alone; top-k, top-p
    u64 k, run, share;      // top-k's number; top-p's part and the random number, of 2^64
    double rate, least;     // Row's rate; min-p, 0: off
    __device__ __forceinline__ u64 run_of(u64 all) const { return max(1ull, __umul64hi(all, run) + (all * run ? 1 : 0)); }
};
template <typename N> __device__ __forceinline__ Settings settings_of(const SampleArgs& a, int row)
{
    const N heat = a.temperature ? ((const N*)a.temperature)[row] : (N)1, k = a.k ? ((const N*)a.k)[row] : (N)0, p = a.p ? ((const N*)a.p)[row] : (N)1;
    const N m = a.m ? ((const N*)a.m)[row] : (N)0, u = ((const N*)a.u)[row];
    Settings t;
    t.first = !(heat > (N)0) || m > (N)1;
    t.byK = !t.first && k >= (N)1 && k < (N)a.vocab;
    t.byP = !t.first && p < (N)1;
    t.k = t.byK ? (u64)k : 0;
    t.run = fraction((double)p);
    t.share = t.first ? 0 : fraction((double)u);
    t.rate = heat > (N)0 ? fmin(32 * 1.4426950408889634 / (double)heat, 1e300) : 0.0;
    t.least = !t.first && m > (N)0 ? (double)m : 0.0;
    return t;
}

// What is kept: logits above `at`, and equal ones up to index `last`
template <typename V> struct Border {
    V at;
    int last;
    __device__ __forceinline__ bool has(V v, int i) const { return v > at || (v == at && i <= last); }
};

// how the listed tokens, n <= FEW of them, stand to each other: of token i (of thread i << shift and the next ones, which all get the sums), what stands before it
struct Rank {
    int shift, i, part;
    bool mine, lead;
    double v;
    u64 w;
    int id;
    __device__ __forceinline__ Rank(const Shared& s, int n)
    {
        shift = n <= THREADS / 16 ? 4 : n <= THREADS / 8 ? 3 : 2;
        i = (int)threadIdx.x >> shift;
        part = (int)threadIdx.x & ((1 << shift) - 1);
        mine = i < n;
        lead = mine && part == 0;
        v = mine ? s.values[i] : 0;
        w = mine ? s.weights[i] : 0;
        id = mine ? s.ids[i] : 0;
    }
    template <typename F> __device__ __forceinline__ u64 sum(int n, F f) const   // of f(j) over all listed ones
    {
        u64 x = 0;
        if (mine)
            for (int j = part; j < n; j += 1 << shift) x += f(j);
        for (int o = 1; o < 1 << shift; o <<= 1) x += shfl_xor64(x, o);
        return x;
    }
    __device__ __forceinline__ bool before(const Shared& s, int j) const { return s.values[j] > v || (s.values[j] == v && s.ids[j] < id); }
};

// The border behind which the sum of counts (byWeight: of weights) of the kept tokens, in falling order, reaches the target.  It is looked for in bins of the
// logits, then in ever smaller ranges of keys, until so few are left that each is compared with each, or they are all equal.
// Bins reach over 12 octaves of weights (20 where they are added up), and only if the border is not among these over all of them: what is counted in LDS is a part of
// the vocabulary then.
// Where FEW tokens at most lie above the border's bin or in it, these are listed, and the border is not looked for.
// whole: all tokens are kept so far
template <typename R, typename G>
__device__ __forceinline__ Border<typename R::V> select(const R& r, Shared& s, u64* parts, const Border<typename R::V> old, const bool whole, const bool byWeight, u64* targetOut, int* few, G targetOf)
{
    typedef typename R::K K;
    typedef typename R::V V;
    const int tid = threadIdx.x, lane = tid & 63;
    auto clear = [&]() __attribute__((always_inline)) {
        __syncthreads();
        for (int i = tid; i < BINS; i += THREADS) { s.count[i] = 0; s.weight[i] = 0; }
        if (tid == 0) { s.listed = 0; s.bin = -1; s.least = ~0ull; s.most = 0; }
        __syncthreads();
    };
    // the bin in which the target is reached: s.bin, what is above it, and the number of tokens there and in it
    u64 target = 0, above = 0;
    auto pick = [&]() __attribute__((always_inline)) {
        constexpr int EACH = BINS / THREADS;
        __syncthreads();
        uint32_t n[EACH], mine = 0;
        u64 c[EACH], sum = 0, all, tokens = 0;
#pragma unroll
        for (int i = 0; i < EACH; i++) {
            mine += n[i] = s.count[EACH * tid + i];
            sum += c[i] = byWeight ? s.weight[EACH * tid + i] : n[i];
        }
        if (byWeight) tokens = block_scan(mine, s.sums, &all);
        u64 at = above + block_scan(sum, s.sums, &all);
        if (!byWeight) tokens = at - above;
#pragma unroll
        for (int i = 0; i < EACH; i++) {
            tokens += n[i];
            if (at < target && target <= at + c[i]) { s.bin = EACH * tid + i; s.above = at; s.reached = (int)tokens; }
            at += c[i];
        }
        __syncthreads();
        above = s.bin >= 0 ? s.above : above;
    };
    // the logits lo .. hi that `old` keeps: f(logit, index); few pieces have any
    auto among = [&](V lo, V hi, auto f) __attribute__((always_inline)) {
        r.each([&](int, int i0, const V (&v)[R::VEC]) __attribute__((always_inline)) {
            bool some = false;
#pragma unroll
            for (int e = 0; e < R::VEC; e++) some = some || (v[e] >= lo && v[e] <= hi);
            if (!__any(some)) return;
#pragma unroll
            for (int e = 0; e < R::VEC; e++)
                if (v[e] >= lo && v[e] <= hi && old.has(v[e], i0 + e)) f(v[e], i0 + e);
        });
    };
    auto list = [&](V lo, V hi) __attribute__((always_inline)) -> int {
        among(lo, hi, [&](V v, int i) __attribute__((always_inline)) {
            const int at = atomicAdd(&s.listed, 1);
            if (at < FEW) { s.values[at] = v; s.ids[at] = i; s.weights[at] = r.weight(v); }
        });
        __syncthreads();
        return min(s.listed, FEW);
    };
    // ---- bins of the logits ----
    const V half = r.top * (V)0.5;
    const double window = byWeight ? 20 : 12;
    V scale = 0;
    int bin = -1;
#pragma unroll 1
    for (int wide = 0; wide < 2 && bin < 0; wide++) {
        // twice the bins a unit of the logits; where that is beyond all numbers the largest logits are by themselves
        scale = (V)fmin(2.0 * r.rate * BINS / (wide ? -r.least : 32.0 * window), sizeof(V) == 4 ? 1e37 : 1e300);
        clear();
        u64 sum = 0;
        // straight on for all of a piece: the weights of its logits are made side by side
        if (byWeight && whole)
            r.each([&](int, int, const V (&v)[R::VEC]) __attribute__((always_inline)) {
#pragma unroll
                for (int e0 = 0; e0 < R::VEC; e0 += R::SIDE) {
                    u64 w[R::SIDE];
#pragma unroll
                    for (int e = 0; e < R::SIDE; e++) sum += w[e] = r.raw_weight(v[e0 + e]);
                    sum -= R::SIDE * RAW;
#pragma unroll
                    for (int e = 0; e < R::SIDE; e++) {
                        const V z = r.bins(v[e0 + e], half, scale);
                        if (!(z < (V)BINS)) continue;
                        atomicAdd(&s.count[(int)z], 1u);
                        atomicAdd(&s.weight[(int)z], w[e] - RAW);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            });
        else if (whole)
            r.each([&](int, int, const V (&v)[R::VEC]) __attribute__((always_inline)) {
#pragma unroll
                for (int e = 0; e < R::VEC; e++) {
                    const V z = r.bins(v[e], half, scale);
                    if (z < (V)BINS) atomicAdd(&s.count[(int)z], 1u);
                }
            });
        else
            among(old.at, r.top, [&](V v, int) __attribute__((always_inline)) {
                const u64 w = byWeight ? r.weight(v) : 0;
                sum += w;
                const V z = r.bins(v, half, scale);
                if (!(z < (V)BINS)) return;
                atomicAdd(&s.count[(int)z], 1u);
                if (byWeight) atomicAdd(&s.weight[(int)z], w);
            });
        if (!wide) {
            u64 all = 0;
            if (byWeight) block_scan(sum, s.sums, &all);
            target = targetOf(all);
        }
        pick();
        bin = s.bin;
    }
    *targetOut = target;
    *few = 0;
    if (bin < 0) return old;   // all of them, as far as they have weight
    // the bin's logits
    V lo = r.smallest([&](V v) __attribute__((always_inline)) { const V z = r.bins(v, half, scale); return z < (V)(bin + 1); });
    if (s.reached <= FEW) {
        *few = s.reached;
        list(lo, r.top);
        return old;
    }
    V hi = bin ? r.smallest([&](V v) __attribute__((always_inline)) { const V z = r.bins(v, half, scale); return z < (V)bin; }) : (V)INFINITY;
    hi = bin ? of_key((K)(key_of(hi) - 1)) : r.top;
    uint32_t n = s.count[bin];
#pragma unroll 1
    while (n > (uint32_t)FEW) {
        // their smallest and largest key
        clear();
        K least = ~(K)0, most = 0;
        among(lo, hi, [&](V v, int) __attribute__((always_inline)) {
            const K k = key_of(v + (V)0);   // -0 is 0
            least = min(least, k);
            most = max(most, k);
        });
        u64 a = least, b = most;
        for (int o = 32; o > 0; o >>= 1) {
            a = min(a, shfl_xor64(a, o));
            b = max(b, shfl_xor64(b, o));
        }
        if (lane == 0 && a <= b) { atomicMin(&s.least, a); atomicMax(&s.most, b); }
        __syncthreads();
        const K low = (K)s.least, high = (K)s.most;
        if (low == high) {
            // all equal: as many as it takes, by their index
            const V v0 = of_key(low);
            const u64 each = byWeight ? r.weight(v0) : 1;
            return Border<V>{v0, locate_equal(r, s, parts, v0, old, (target - above + each - 1) / each)};
        }
        int shift = 0;
        while (((high - low) >> shift) >= (K)BINS) shift++;
        clear();
        among(lo, hi, [&](V v, int) __attribute__((always_inline)) {
            const int at = (int)((high - key_of(v + (V)0)) >> shift);
            atomicAdd(&s.count[at], 1u);
            if (byWeight) atomicAdd(&s.weight[at], r.weight(v));
        });
        pick();
        const K to = high - ((K)s.bin << shift), span = ((K)1 << shift) - 1;
        hi = of_key(to);
        lo = of_key(to - low > span ? (K)(to - span) : low);
        n = s.count[s.bin];
    }
    // ---- so few that each is compared with each: the one at which the target is reached ----
    const int listed = list(lo, hi);
    const Rank me(s, listed);
    const u64 w = byWeight ? me.w : 1, at = above + me.sum(listed, [&](int j) __attribute__((always_inline)) -> u64 { return me.before(s, j) ? (byWeight ? s.weights[j] : 1) : 0; });
    if (me.lead && at < target && target <= at + w) { s.value = me.v; s.index = me.id; }
    __syncthreads();
    return Border<V>{(V)s.value, s.index};
}

// The draw from the listed tokens alone.  k: of them the first (0: all), targetOf(sum): the sum of weights at which top-p's run ends (0: all), least: weights from here on.
// Each is compared with each once, which says its place in both orders, by logit and by index; the rest are sums along these.
template <typename R, typename G> __device__ __forceinline__ int draw_of_few(const R& r, Shared& s, int n, u64 k, G targetOf, double least, u64 share, u64* total)
{
    const int tid = threadIdx.x;
    const Rank me(s, n);
    uint32_t at = 0;   // tokens before it, and 2^16 those of smaller indexes
    if (me.mine) {
#pragma unroll 4
        for (int j = me.part; j < n; j += 1 << me.shift) at += (me.before(s, j) ? 1u : 0u) + (s.ids[j] < me.id ? 0x10000u : 0u);
    }
    for (int o = 1; o < 1 << me.shift; o <<= 1) at += __shfl_xor(at, o);
    const int rank = at & 0xffff, place = at >> 16;
    uint32_t *tag = s.count, *ids = s.count + FEW;   // by rank: place and min-p's word; by place: index
    if (me.lead) {
        s.kept[rank] = me.w;
        tag[rank] = (uint32_t)place << 1 | (least == 0.0 || r.two_to(r.power((typename R::V)me.v), 0) >= least);
        ids[place] = me.id;
    }
    __syncthreads();
    const bool first = tid < n && (k == 0 || (u64)tid < k);
    const u64 w = first ? s.kept[tid] : 0;
    u64 all;
    const u64 better = block_scan(w, s.sums, &all), target = targetOf(all);
    if (tid < n) s.weight[tag[tid] >> 1] = first && (tid == 0 || ((target == 0 || better < target) && tag[tid] & 1)) ? w : 0;
    if (tid == 0) s.found = -1;
    __syncthreads();
    const u64 mine = tid < n ? s.weight[tid] : 0, before = block_scan(mine, s.sums, total), want = __umul64hi(*total, share);
    if (before <= want && want < before + mine) s.found = ids[tid];
    __syncthreads();
    return s.found;
}

// where a row's logits are, and whether it has any
template <typename L, typename N> __device__ __forceinline__ bool row_of(const SampleArgs& a, int row, Row<L>& r, const double* roots)
{
    const N which = a.rows ? ((const N*)a.rows)[row] : (N)row;
    const bool there = which >= (N)0 && which < (N)a.logitsRows;
    r.x = (const L*)a.x + (there ? (size_t)(int)which * a.stride : 0);
    r.vocab = a.vocab;
    r.perWave = a.perWave;
    r.bits = a.bits;
    r.least = -32.0 * (a.bits + 2);
    r.infinite = false;
    r.roots = roots;
    return there;
}
template <typename L> __device__ __forceinline__ void top_is(Row<L>& r, typename Row<L>::V top)
{
    typedef typename Row<L>::V V;
    r.infinite = top == (V)INFINITY;
    r.top = r.infinite ? (V)0 : top;
}
template <typename L, typename N> __device__ __forceinline__ void write_draw(const SampleArgs& a, int row, const Row<L>& r, const Settings& t, int id, u64 total)
{
    typedef typename Row<L>::V V;
    ((N*)a.ids)[row] = (N)id;
    if (!a.logs) return;
    const V v = r.infinite ? r.top : (V)read(r.x[id]);
    ((N*)a.logs)[row] = t.first ? (N)0 : (N)(fmin(((double)v - (double)r.top) * t.rate, 0.0) * (0.69314718055994530942 / 32) - log(ldexp((double)total, -a.bits)));
}
template <typename N> __device__ __forceinline__ void write_none(const SampleArgs& a, int row)
{
    ((N*)a.ids)[row] = (N)-1;
    if (a.logs) ((N*)a.logs)[row] = (N)0;
}
// sums of the weights that the border keeps, of a lane's piece
template <typename R> __device__ __forceinline__ u64 kept_weights(const R& r, const typename R::V (&v)[R::VEC], int i0, const Border<typename R::V>& border)
{
    typedef typename R::V V;
    u64 sum = 0;
    if (!(border.at > -(V)INFINITY)) {
#pragma unroll
        for (int e0 = 0; e0 < R::VEC; e0 += R::SIDE) {
#pragma unroll
            for (int e = 0; e < R::SIDE; e++) sum += r.raw_weight(v[e0 + e]);
            __builtin_amdgcn_sched_barrier(0);
        }
        return sum - R::VEC * RAW;
    }
    bool any = false;
#pragma unroll
    for (int e = 0; e < R::VEC; e++) any = any || v[e] >= border.at;
    if (__any(any))
#pragma unroll
        for (int e0 = 0; e0 < R::VEC; e0 += R::SIDE) {
#pragma unroll
            for (int e = e0; e < e0 + R::SIDE; e++) {
                const u64 w = r.weight(v[e]);
                sum += border.has(v[e], i0 + e) ? w : 0;
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    return sum;
}

// A row by one workgroup
template <typename L, typename N> __device__ __forceinline__ void sample_row(const SampleArgs& a, int row, Shared& s, u64* parts)
{
    typedef Row<L> R;
    typedef typename R::V V;
    __shared__ V sTop[WAVES];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    if (tid < 32) s.roots[tid] = ROOTS[tid];
    R r;
    const bool none = !row_of<L, N>(a, row, r, s.roots);
    // ---- the largest logit ----
    V top = -(V)INFINITY;
    if (!none)
        r.each([&](int, int, const V (&v)[R::VEC]) __attribute__((always_inline)) {
#pragma unroll
            for (int e = 0; e < R::VEC; e++) top = v[e] > top ? v[e] : top;
        });
    for (int o = 32; o > 0; o >>= 1) {
        const V t = __shfl_xor(top, o);
        top = t > top ? t : top;
    }
    if (lane == 0) sTop[wave] = top;
    __syncthreads();
    for (int i = 0; i < WAVES; i++) top = sTop[i] > top ? sTop[i] : top;
    if (!(top > -(V)INFINITY)) {   // no row, or nothing in it that could be drawn
        if (tid == 0) write_none<N>(a, row);
        return;
    }
    const Settings t = settings_of<N>(a, row);
    top_is(r, top);
    r.rate = t.rate;
    Border<V> border = {-(V)INFINITY, INT32_MAX};
    u64 total, target = 0;
    int id = -1, few;
#pragma unroll 1
    for (int filter = 0; filter < 2; filter++) {
        if (!(filter ? t.byP : t.byK)) continue;
        border = select(r, s, parts, border, !filter || !t.byK, filter != 0, &target, &few, [&](u64 all) __attribute__((always_inline)) -> u64 { return filter ? t.run_of(all) : t.k; });
        if (few) {
            id = draw_of_few(r, s, few, filter ? 0 : t.k, [&](u64 all) __attribute__((always_inline)) -> u64 { return filter ? target : t.byP ? t.run_of(all) : 0; }, t.least, t.share, &total);
            break;
        }
    }
    if (id < 0 && t.least > 0.0) {   // weights from here on are logits from here on
        const V at = r.smallest([&](V v) __attribute__((always_inline)) { return r.two_to(r.power(v), 0) >= t.least; });
        if (at > border.at) border = Border<V>{at, INT32_MAX};
    }
    if (t.first) id = locate_equal(r, s, parts, r.top, border, 1);
    else if (id < 0)
        id = locate(r, s, parts, [&](const V (&v)[R::VEC], int i0) __attribute__((always_inline)) -> u64 { return kept_weights(r, v, i0, border); },
                    [&](V v, int i) __attribute__((always_inline)) -> u64 { return border.has(v, i) ? r.weight(v) : 0; },
                    [&](u64 all) __attribute__((always_inline)) -> u64 { return __umul64hi(all, t.share); }, &total);
    if (tid == 0) write_draw<L, N>(a, row, r, t, id, total);
}
template <typename L, typename N> __global__ __launch_bounds__(THREADS) void sample_kernel(SampleArgs a)
{
    __shared__ Shared s;
    extern __shared__ u64 parts[];
    const long long row = (long long)blockIdx.y * gridDim.x + blockIdx.x;
    if (row < a.count) sample_row<L, N>(a, (int)row, s, parts);
}

// ---- a row by many workgroups ---------------------------------------------------------------------------------------------------------
// Logits of 16 and 32 bits: slices of a row, one a workgroup, in launches that read them one after the other:
//   top     the largest logit of every slice;
//   weigh   the weights: added up, or counted and added up in bins;
//   border  a workgroup a row: the draw, where neither top-k nor top-p is asked for, else the bin that has the border;
//   list    what lies above the border's bin and in it, if LISTED tokens at most, else what lies in the bin;
//   finish  a workgroup a row: the draw, with what is listed alone, or with that and the bins above it, slice by slice, and the logits of one slice; rows of which
//           too much would be listed as above, from their beginning.
// (No launch waits for its last workgroup: reading what the others have written past the caches, at the level that all XCDs share, at the end of every slice costs
// more than a launch.  256 rows of 131072, weigh with it 48 us.)  Sums are whole numbers: any order gives the same.
constexpr int CUT = 256, CUT_BINS = CUT, LISTED = 4096, COUNTERS = 32;   // (a row's counter has 128 bytes of its own)
enum RowMode { ROW_DONE, ROW_LIST_ALL, ROW_LIST_BIN, ROW_WHOLE };
struct RowState {
    int mode, last;       // min-p's border: logits above `at`, equal ones up to index `last`
    float top, lo, hi, at;
    u64 above, target;    // of what is listed of a bin: what is above it, and where top-k's or top-p's border is (0: not in it)
    int bins, none;       // whole bins that are kept
};

// a slice: EACH logits a thread of T, in pieces, in the order of the vocabulary from piece to piece and within one from thread to thread
template <typename L, int EACH, int T> struct Slice {
    typedef Row<L> R;
    static constexpr int VEC = R::VEC, PIECES = EACH / VEC, LOGITS = EACH * T, CELLS = PIECES * T / 64;   // cells: a wavefront's part of a piece
    __device__ static int index(int slice, int piece) { return slice * LOGITS + piece * T * VEC + (int)threadIdx.x * VEC; }
    L raw[PIECES][VEC];
    __device__ __forceinline__ void load(const R& r, int slice)   // all of it under way at once
    {
#pragma unroll
        for (int q = 0; q < PIECES; q++) r.fetch(index(slice, q), raw[q]);
    }
    template <typename F> __device__ __forceinline__ void each(const R& r, int slice, F f) const   // f(piece, first index, logits)
    {
#pragma unroll
        for (int q = 0; q < PIECES; q++) {
            float v[VEC];
            r.logits(raw[q], v);
            f(q, index(slice, q), v);
        }
    }
};

struct DrawShared { u64 sums[CUT / 64], before; int cell; };
// The draw of a row from the sums of its n cells: which it falls into, and, for one wavefront, where in it
template <typename L, int EACH>
__device__ __forceinline__ void draw_from(const SampleArgs& a, int row, const Row<L>& r, const Settings& t, const Border<float>& border, const u64* cells, int n, DrawShared& s)
{
    typedef Slice<L, EACH, CUT> C;
    constexpr int VEC = C::VEC;
    const int tid = threadIdx.x, per = (n + CUT - 1) / CUT, from = tid * per, to = min(n, from + per);
    u64 mine = 0, total;
#pragma unroll 8
    for (int i = from; i < to; i++) mine += cells[i];
    u64 before = block_scan<CUT / 64>(mine, s.sums, &total);
    const u64 want = __umul64hi(total, t.share);
    if (before <= want && want < before + mine)
        for (int i = from; i < to; i++) {
            const u64 x = cells[i];
            if (want < before + x) { s.cell = i; s.before = before; break; }
            before += x;
        }
    __syncthreads();
    if (tid >= 64) return;
    const int i0 = s.cell * 64 * VEC + tid * VEC;   // (the order of the cells is that of the vocabulary)
    L raw[VEC];
    float v[VEC];
    u64 w[VEC], sum = 0;
    r.fetch(i0, raw);
    r.logits(raw, v);
#pragma unroll
    for (int e = 0; e < VEC; e++) sum += w[e] = r.weight(v[e]);
    if (border.at > -INFINITY) {
        sum = 0;
#pragma unroll
        for (int e = 0; e < VEC; e++) sum += w[e] = border.has(v[e], i0 + e) ? w[e] : 0;
    }
    u64 at = s.before + wave_scan(sum) - sum;
    int id = -1;
#pragma unroll
    for (int e = 0; e < VEC; e++) {
        if (at <= want && want < at + w[e]) id = i0 + e;
        at += w[e];
    }
    if (id >= 0) write_draw<L, float>(a, row, r, t, id, total);
}

template <typename L, int EACH> __global__ __launch_bounds__(CUT) void sample_top_kernel(SampleArgs a, SampleCuts w)
{
    __shared__ float sTop[CUT / 64];
    const int tid = threadIdx.x, slice = blockIdx.x, row = blockIdx.y;
    Row<L> r;
    float top = -INFINITY;
    Slice<L, EACH, CUT> c;
    if (row_of<L, float>(a, row, r, nullptr)) {
        c.load(r, slice);
        c.each(r, slice, [&](int, int, const float (&v)[Row<L>::VEC]) __attribute__((always_inline)) {
#pragma unroll
            for (int e = 0; e < Row<L>::VEC; e++) top = v[e] > top ? v[e] : top;
        });
    }
    top = group_max<64>(top);
    if ((tid & 63) == 0) sTop[tid >> 6] = top;
    __syncthreads();
    if (tid == 0) {
        for (int i = 1; i < CUT / 64; i++) top = fmaxf(top, sTop[i]);
        w.tops[row * w.slices + slice] = top;
    }
    if (slice == 0 && tid == 0) w.listed[row * COUNTERS] = 0;
}

// smallest logit that the weights' share `least` keeps
template <typename R> __device__ __forceinline__ Border<float> border_of_least(const R& r, double least)
{
    Border<float> b = {-INFINITY, INT32_MAX};
    if (least > 0.0) b.at = r.smallest([&](float v) __attribute__((always_inline)) { return r.two_to(r.power(v), 0) >= least; });
    return b;
}

// the row's largest logit, and the first slice that has it, from that of slice i in thread i
constexpr int SLICES = 128;   // of a row, at most
static_assert(SLICES <= CUT && SAMPLE_VOCAB <= SLICES * 32 * CUT, "a thread a slice");
__device__ __forceinline__ float top_of_slice(const SampleCuts& w, int row) { return (int)threadIdx.x < w.slices ? w.tops[row * w.slices + threadIdx.x] : -INFINITY; }
__device__ __forceinline__ float top_of_row(float mine, int* first)
{
    __shared__ float sTop[SLICES / 64];
    __shared__ int sAt[SLICES / 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    if (tid < SLICES) {
        const float top = group_max<64>(mine);
        const u64 there = __ballot(mine == top);
        if (lane == 0) { sTop[wave] = top; sAt[wave] = tid + __builtin_ctzll(there | 1ull << 63); }
    }
    __syncthreads();
    float top = sTop[0];
    int at = sAt[0];
    for (int i = 1; i < SLICES / 64; i++)
        if (sTop[i] > top) { top = sTop[i]; at = sAt[i]; }
    *first = at;
    return top;
}
// bins a unit of the logits, twice: top-k's over all octaves of weights, and a little more than these, so that no rounding leaves out a token with weight; top-p's over 24
// (what lies below weighs too little to be reached, but for flat rows)
template <typename R> __device__ __forceinline__ float bins_of(const R& r, const Settings& t)
{
    return (float)fmin(2.0 * (1.0 - 0x1p-16) * r.rate * CUT_BINS / (t.byK ? -r.least : 32.0 * 24), 1e37);
}

// whether the bins' weights are added up: not where top-k leaves so few tokens that, with the others of the border's bin, they are all listed, but for flat rows
__device__ __forceinline__ bool weighs(const Settings& t) { return !t.byK || t.k > LISTED / 4; }

template <typename L, int EACH> __global__ __launch_bounds__(CUT) void sample_weigh_kernel(SampleArgs a, SampleCuts w)
{
    typedef Row<L> R;
    typedef Slice<L, EACH, CUT> C;
    __shared__ uint32_t sCount[CUT_BINS];
    __shared__ u64 sWeight[CUT_BINS], sSums[CUT / 64];
    __shared__ double sRoots[32];
    const int tid = threadIdx.x, slice = blockIdx.x, row = blockIdx.y;
    R r;
    const float mine = top_of_slice(w, row);
    if (!row_of<L, float>(a, row, r, sRoots)) return;
    const Settings t = settings_of<float>(a, row);
    C c;
    c.load(r, slice);   // (behind what is waited for first)
    if (t.first) return;
    if (tid < 32) sRoots[tid] = ROOTS[tid];
    sCount[tid] = 0;
    sWeight[tid] = 0;
    int first;
    const float top = top_of_row(mine, &first);   // (with the barrier that the lines above need)
    if (!(top > -INFINITY)) return;
    top_is(r, top);
    r.rate = t.rate;
    u64 sum = 0, all;
    if (!t.byK && !t.byP) {
        const Border<float> border = border_of_least(r, t.least);
        u64* cells = w.sums + (size_t)(row * w.slices + slice) * C::CELLS + (tid >> 6);
        c.each(r, slice, [&](int q, int i0, const float (&v)[R::VEC]) __attribute__((always_inline)) {
            const u64 x = wave_sum(kept_weights(r, v, i0, border));
            if ((tid & 63) == 0) cells[q * (CUT / 64)] = x;
        });
        return;
    }
    const bool byWeight = weighs(t);
    const float half = r.top * 0.5f, scale = bins_of(r, t);
    c.each(r, slice, [&](int, int, const float (&v)[R::VEC]) __attribute__((always_inline)) {
#pragma unroll
        for (int e0 = 0; e0 < R::VEC; e0 += R::SIDE) {
            u64 x[R::SIDE];
            if (byWeight) {
#pragma unroll
                for (int e = 0; e < R::SIDE; e++) sum += x[e] = r.raw_weight(v[e0 + e]);
                sum -= R::SIDE * RAW;
            }
#pragma unroll
            for (int e = 0; e < R::SIDE; e++) {
                const float z = r.bins(v[e0 + e], half, scale);
                if (!(z < (float)CUT_BINS)) continue;
                atomicAdd(&sCount[(int)z], 1u);
                if (byWeight) atomicAdd(&sWeight[(int)z], x[e] - RAW);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    });
    block_scan<CUT / 64>(sum, sSums, &all);
    const size_t bins = ((size_t)row * w.slices + slice) * CUT_BINS + tid;
    w.counts[bins] = sCount[tid];
    if (byWeight) {
        w.weights[bins] = sWeight[tid];
        if (tid == 0) w.sums[(size_t)(row * w.slices + slice) * C::CELLS] = all;
    }
}

template <typename L, int EACH> __global__ __launch_bounds__(CUT) void sample_border_kernel(SampleArgs a, SampleCuts w)
{
    typedef Row<L> R;
    typedef Slice<L, EACH, CUT> C;
    __shared__ DrawShared s;
    __shared__ int sFirst, sBin, sReached, sIn[CUT_BINS];
    __shared__ double sRoots[32];
    const int tid = threadIdx.x, row = blockIdx.x;
    R r;
    row_of<L, float>(a, row, r, sRoots);
    const Settings t = settings_of<float>(a, row);
    const bool bins = t.byK || t.byP;
    const float mine = top_of_slice(w, row);
    const u64* cells = w.sums + (size_t)row * w.slices * C::CELLS;
    // this thread's bin of the row, and its slice
    uint32_t n = 0;
    u64 x = 0, sum = 0, all = 0;
    if (bins) {
        constexpr int AHEAD = 16;   // slices read at once
        sum = !t.byK && tid < w.slices ? cells[tid * C::CELLS] : 0;
        for (int i0 = 0; i0 < w.slices; i0 += AHEAD) {
            uint32_t some[AHEAD];
            u64 heavy[AHEAD];
            const size_t at = (size_t)row * w.slices * CUT_BINS + tid;
#pragma unroll
            for (int j = 0; j < AHEAD; j++) some[j] = w.counts[at + min(i0 + j, w.slices - 1) * CUT_BINS];
            if (!t.byK)
#pragma unroll
                for (int j = 0; j < AHEAD; j++) heavy[j] = w.weights[at + min(i0 + j, w.slices - 1) * CUT_BINS];
#pragma unroll
            for (int j = 0; j < AHEAD; j++) {
                n += i0 + j < w.slices ? some[j] : 0;
                if (!t.byK) x += i0 + j < w.slices ? heavy[j] : 0;
            }
        }
    }
    if (tid < 32) sRoots[tid] = ROOTS[tid];
    sIn[tid] = n;
    if (tid == 0) { sFirst = INT32_MAX; sBin = -1; }
    int first;
    const float top = top_of_row(mine, &first);
    RowState st = {};
    st.mode = ROW_DONE;
    st.top = top;
    if (!(top > -INFINITY)) {   // no row, or nothing in it that could be drawn
        if (tid == 0) {
            write_none<float>(a, row);
            ((RowState*)w.state)[row] = st;
        }
        return;
    }
    top_is(r, top);
    r.rate = t.rate;
    if (t.first) {
        C c;
        c.load(r, first);
        c.each(r, first, [&](int, int i0, const float (&v)[R::VEC]) __attribute__((always_inline)) {
#pragma unroll
            for (int e = R::VEC - 1; e >= 0; e--)
                if (v[e] == r.top) atomicMin(&sFirst, i0 + e);
        });
        __syncthreads();
        if (tid == 0) write_draw<L, float>(a, row, r, t, sFirst, 0);
    } else if (!bins) {
        draw_from<L, EACH>(a, row, r, t, border_of_least(r, t.least), cells, w.slices * C::CELLS, s);
    } else {
        u64 any, weight;
        if (!t.byK) block_scan<CUT / 64>(sum, s.sums, &all);
        const u64 tokens = block_scan<CUT / 64>(n, s.sums, &any), before = t.byK ? tokens : block_scan<CUT / 64>(x, s.sums, &weight);
        const u64 target = t.byK ? t.k : t.run_of(all), amount = t.byK ? n : x;
        if (before < target && target <= before + amount) { sBin = tid; s.before = before; sReached = (int)tokens + n; }
        __syncthreads();
        const float half = r.top * 0.5f, scale = bins_of(r, t);
        const Border<float> least = border_of_least(r, t.least);
        const float z = r.bins(least.at, half, scale);
        const int leastBin = z < (float)CUT_BINS ? (int)z : CUT_BINS;
        st.at = least.at;
        st.last = least.last;
        // (top-k: no bin where there are not as many with weight, all of which stay then; top-p: none where it goes further down than the bins, unless min-p does not)
        int bin = sBin >= 0 ? sBin : t.byK ? CUT_BINS : leastBin < CUT_BINS ? leastBin : -1;
        const u64 reached = sBin >= 0 ? sReached : any;
        if (bin < 0) st.mode = ROW_WHOLE;
        else if (reached <= LISTED) {
            st.mode = ROW_LIST_ALL;
            st.target = target;
        } else if (t.byK && (t.byP || !weighs(t))) st.mode = ROW_WHOLE;
        else {
            st.above = s.before;
            st.target = sBin >= 0 && bin <= leastBin ? target : 0;
            bin = min(bin, leastBin);
            st.mode = bin < CUT_BINS && sIn[bin] > LISTED ? ROW_WHOLE : ROW_LIST_BIN;
        }
        st.bins = bin;
        auto from = [&](int b) __attribute__((always_inline)) { return r.smallest([&](float v) __attribute__((always_inline)) { return r.bins(v, half, scale) < (float)b; }); };
        if (bin < CUT_BINS) {
            st.lo = from(bin + 1);
            st.hi = bin > 0 ? of_key(key_of(from(bin)) - 1) : r.top;
        } else {   // no bin more
            st.lo = st.mode == ROW_LIST_ALL ? from(CUT_BINS) : INFINITY;
            st.hi = -INFINITY;
        }
    }
    if (tid == 0) ((RowState*)w.state)[row] = st;
}

// Logit (-0 is 0) and index as one number: falling logits, and rising indexes of equal ones, fall.  Few bits, so that few rounds tell them apart: 16 of a 16-bit logit
constexpr int INDEX_BITS = 20, LAST_INDEX = (1 << INDEX_BITS) - 1;
static_assert(SAMPLE_VOCAB <= LAST_INDEX + 1, "index");
template <typename L> __device__ __forceinline__ u64 place_of(float v, int i)
{
    const uint32_t k = key_of(v + 0.f);
    return (u64)(sizeof(L) == 2 ? k >> 16 : k) << INDEX_BITS | (uint32_t)(LAST_INDEX - i);
}
// of a logit that need not be one of L: the least place of those that are not below it
template <typename L> __device__ __forceinline__ u64 least_place(float v)
{
    const uint32_t k = key_of(v + 0.f);
    // the lower half of a 16-bit logit's key is 0, of a negative one all bits
    return sizeof(L) == 2 ? (u64)((k >> 16) + (k >> 31 && k & 0xffffu ? 1 : 0)) << INDEX_BITS : (u64)k << INDEX_BITS;
}
__device__ __forceinline__ int index_at(u64 place) { return LAST_INDEX - (int)(place & LAST_INDEX); }
template <typename L> __device__ __forceinline__ float logit_at(u64 place)
{
    const uint32_t k = (uint32_t)(place >> INDEX_BITS);
    return of_key(sizeof(L) == 2 ? k << 16 | (k & 0x8000u ? 0u : 0xffffu) : k);   // (of a negative one all bits are turned)
}

template <typename L, int EACH> __global__ __launch_bounds__(CUT) void sample_list_kernel(SampleArgs a, SampleCuts w)
{
    typedef Row<L> R;
    typedef Slice<L, EACH, CUT> C;
    __shared__ u64 sSums[CUT / 64];
    __shared__ int sBase;
    const int tid = threadIdx.x, slice = blockIdx.x, row = blockIdx.y;
    const RowState st = ((const RowState*)w.state)[row];
    if (st.mode != ROW_LIST_ALL && st.mode != ROW_LIST_BIN) return;
    R r;
    row_of<L, float>(a, row, r, nullptr);
    top_is(r, st.top);
    const float lo = st.lo, hi = st.mode == ROW_LIST_ALL ? r.top : st.hi;
    u64 hits = 0, all;
    C c;
    c.load(r, slice);
    c.each(r, slice, [&](int q, int, const float (&v)[R::VEC]) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < R::VEC; e++) hits |= (u64)(v[e] >= lo && v[e] <= hi) << (q * R::VEC + e);
    });
    int to = (int)block_scan<CUT / 64>(__popcll(hits), sSums, &all);
    if (!all) return;
    if (tid == 0) sBase = __hip_atomic_fetch_add(w.listed + row * COUNTERS, (int)all, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    to += sBase;
    if (hits)
        c.each(r, slice, [&](int q, int i0, const float (&v)[R::VEC]) __attribute__((always_inline)) {
#pragma unroll
            for (int e = 0; e < R::VEC; e++)
                if (hits >> (q * R::VEC + e) & 1) {
                    if (to < LISTED) w.list[(size_t)row * LISTED + to] = place_of<L>(v[e], i0 + e);
                    to++;
                }
        });
}

constexpr int OWN = LISTED / THREADS;
struct ReachShared { uint32_t count[THREADS]; u64 amount[THREADS], sums[WAVES], above, key, keys[64], amounts[64]; int bin, few; };
// Of numbers key[j], which are all different, with amounts: the one at which the sum of the amounts, from the largest number down, reaches the target; 0 if it does not.
// In ever smaller ranges, a bin a thread, until those of one wavefront are left, who look at each other.
template <typename F> __device__ __forceinline__ u64 reach(ReachShared& s, const u64 (&key)[OWN], F amount, u64 lo, u64 hi, u64 target)
{
    const int tid = threadIdx.x;
    u64 above = 0;
#pragma unroll 1
    for (;;) {
        const int shift = max(0, 64 - 10 - __builtin_clzll((hi - lo) | 1));
        __syncthreads();
        s.count[tid] = 0;
        s.amount[tid] = 0;
        if (tid == 0) { s.bin = -1; s.few = 0; }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < OWN; j++) {
            const u64 w = amount(j);
            if (!w || key[j] < lo || key[j] > hi) continue;
            const int b = (int)((hi - key[j]) >> shift);
            atomicAdd(&s.count[b], 1u);
            atomicAdd(&s.amount[b], w);
        }
        __syncthreads();
        u64 all;
        const u64 mine = s.amount[tid], at = above + block_scan(mine, s.sums, &all);
        if (at < target && target <= at + mine) { s.bin = tid; s.above = at; }
        __syncthreads();
        const int bin = s.bin;
        if (bin < 0) return 0;
        above = s.above;
        hi -= (u64)bin << shift;
        const u64 span = (1ull << shift) - 1;
        lo = hi - lo > span ? hi - span : lo;
        if (s.count[bin] <= 64) break;
    }
#pragma unroll
    for (int j = 0; j < OWN; j++) {
        const u64 w = amount(j);
        if (key[j] < lo || key[j] > hi || !w) continue;
        const int i = atomicAdd(&s.few, 1);
        s.keys[i] = key[j];
        s.amounts[i] = w;
    }
    __syncthreads();
    const int few = s.few;
    if (tid < few) {   // (of the first wavefront)
        const u64 mine = s.keys[tid];
        u64 at = above;
        for (int i = 0; i < few; i++) at += s.keys[i] > mine ? s.amounts[i] : 0;
        if (at < target && target <= at + s.amounts[tid]) s.key = mine;
    }
    __syncthreads();
    const u64 k = s.key;
    __syncthreads();
    return k;
}

template <typename L, int EACH> __global__ __launch_bounds__(THREADS) void sample_finish_kernel(SampleArgs a, SampleCuts w)
{
    static_assert(THREADS == 1024, "bins of reach()");
    typedef Row<L> R;
    __shared__ union { Shared row; ReachShared reach; } s;
    __shared__ double sRoots[32];
    extern __shared__ u64 parts[];
    const int tid = threadIdx.x, row = blockIdx.x;
    const RowState st = ((const RowState*)w.state)[row];
    // (read at once, whatever it is good for)
    const int n = min(w.listed[row * COUNTERS], LISTED);
    const u64* list = w.list + (size_t)row * LISTED;
    const Settings t = settings_of<float>(a, row);
    u64 key[OWN];
#pragma unroll
    for (int j = 0; j < OWN; j++) key[j] = list[tid + THREADS * j];
    if (st.mode == ROW_WHOLE) {
        sample_row<L, float>(a, row, s.row, parts);
        return;
    }
    if (st.mode != ROW_LIST_ALL && st.mode != ROW_LIST_BIN) return;
    R r;
    row_of<L, float>(a, row, r, sRoots);
    top_is(r, st.top);
    r.rate = t.rate;
    if (tid < 32) sRoots[tid] = ROOTS[tid];
    u64 weight[OWN], least = 0, all, total;
#pragma unroll
    for (int j = 0; j < OWN; j++) key[j] = tid + THREADS * j < n ? key[j] : 0;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < OWN; j++) weight[j] = key[j] ? r.weight(logit_at<L>(key[j])) : 0;
    auto one = [&](int j) __attribute__((always_inline)) -> u64 { return key[j] != 0; };
    auto kept = [&](int j) __attribute__((always_inline)) -> u64 { return key[j] >= least ? weight[j] : 0; };
    if (n <= FEW) {
        if (tid < n) {
            s.row.values[tid] = logit_at<L>(key[0]);
            s.row.weights[tid] = weight[0];
            s.row.ids[tid] = index_at(key[0]);
        }
        __syncthreads();
    }
    if (st.mode == ROW_LIST_ALL && n <= FEW) {
        const int id = draw_of_few(r, s.row, n, t.k, [&](u64 sum) __attribute__((always_inline)) -> u64 { return !t.byP ? 0 : t.byK ? t.run_of(sum) : st.target; }, t.least, t.share, &total);
        if (tid == 0) write_draw<L, float>(a, row, r, t, id, total);
        return;
    }
    const u64 from = place_of<L>(st.lo, LAST_INDEX), to = place_of<L>(st.mode == ROW_LIST_ALL ? r.top : st.hi, 0);
    if (st.mode == ROW_LIST_BIN) {
        Border<float> border = {st.at, st.last};
        if (st.target) {
            const u64 target = st.target - st.above, at = t.byK ? reach(s.reach, key, one, from, to, target) : reach(s.reach, key, kept, from, to, target);
            const Border<float> b = {logit_at<L>(at), index_at(at)};
            if (!(border.at > b.at)) border = b;
        }
        // what is left of every slice: whole bins, and of the bin that is listed what the border leaves
        constexpr int LOGITS = EACH * CUT, PER = LOGITS / THREADS;
        u64* slices = s.reach.amount;
        for (int i = tid >> 6; i < w.slices; i += WAVES) {
            const u64* bins = w.weights + ((size_t)row * w.slices + i) * CUT_BINS;
            u64 x = 0;
#pragma unroll
            for (int b = tid & 63; b < CUT_BINS; b += 64) x += b < st.bins ? bins[b] : 0;
            x = wave_sum(x);
            if ((tid & 63) == 0) slices[i] = x;
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < OWN; j++)
            if (key[j] && border.has(logit_at<L>(key[j]), index_at(key[j]))) atomicAdd(slices + index_at(key[j]) / LOGITS, weight[j]);
        __syncthreads();
        u64 mine = tid < w.slices ? slices[tid] : 0, at = block_scan(mine, s.reach.sums, &total);
        const u64 want = __umul64hi(total, t.share);
        if (at <= want && want < at + mine) { s.reach.bin = tid; s.reach.above = at; }
        __syncthreads();
        const int i0 = s.reach.bin * LOGITS + tid * PER;
        const u64 before = s.reach.above;
        u64 x[PER];
        mine = 0;
#pragma unroll
        for (int e = 0; e < PER; e++) {
            float v = i0 + e < a.vocab ? read(r.x[i0 + e]) : -INFINITY;
            if (r.infinite) v = v == INFINITY ? 0.f : -INFINITY;
            mine += x[e] = border.has(v, i0 + e) ? r.weight(v) : 0;
        }
        at = before + block_scan(mine, s.reach.sums, &all);
#pragma unroll
        for (int e = 0; e < PER; e++) {
            if (at <= want && want < at + x[e]) write_draw<L, float>(a, row, r, t, i0 + e, total);
            at += x[e];
        }
        return;
    }
    auto sum = [&]() __attribute__((always_inline)) -> u64 {
        u64 x = 0;
#pragma unroll
        for (int j = 0; j < OWN; j++) x += kept(j);
        block_scan(x, s.reach.sums, &all);
        return all;
    };
    if (t.byK) least = max(least, reach(s.reach, key, one, from, to, t.k));
    if (t.byP) least = max(least, reach(s.reach, key, kept, from, to, t.byK ? t.run_of(sum()) : st.target));
    if (t.least > 0.0) least = max(least, least_place<L>(st.at));
    total = sum();
    // in the order of the vocabulary: the sum up to the token drawn exceeds u times all
    u64 order[OWN];
#pragma unroll
    for (int j = 0; j < OWN; j++) order[j] = key[j] & LAST_INDEX;
    const u64 drawn = reach(s.reach, order, kept, LAST_INDEX + 1 - a.vocab, LAST_INDEX, __umul64hi(total, t.share) + 1);
    if (tid == 0) write_draw<L, float>(a, row, r, t, index_at(drawn), total);
}

}  // namespace

// bits of a weight behind the point: what the sum over the vocabulary leaves of 64
int sample_bits(int vocab)
{
    int log = 0;
    while ((1 << log) < vocab) log++;
    return std::min(50, 63 - log);
}

// When slices of rows are what workgroups have.  Where every CU has a row or two at most, a row alone takes as long as it is, and five launches some 25 us; more rows than that
// take turns.  us, a workgroup a row | slices, the same rows time and again: top-50 in fp32, 1 row of 32000 22.8 | 21.1, of 131072 48.7 | 23.5, 16 of 8000 17.8 | 22.0, 256 of 8000
// 18.6 | 24.4, of 32000 26.7 | 36.5, 1024 of 4000 62.2 | 48.9; temperature, top-k, top-p and min-p in 16 bits, 1 row of 32000 37.6 | 26.6, 16 46.3 | 32.6, 256 54.5 | 49.9, 4 of 131072 95.5 | 31.4,
// 16 of 8000 29.0 | 30.0, 1024 of 4000 92.8 | 64.8; top-p in fp32, 1 row of 32000 22.8 | 21.2, 64 36.7 | 33.6, 256 40.1 | 51.8.  (Above CUT_ROWS it is the scratch memory that costs.)
constexpr int CUT_ROWS = 4096, CUT_FEW = 128, CUT_TURNS = 512;
static bool cut(const SampleArgs& a) { return a.count <= CUT_ROWS && a.vocab >= (a.count <= CUT_FEW ? 24576 : a.count <= CUT_TURNS ? 49152 : 2048); }
// Logits a thread of a slice: few where there are few slices.  us, 8 | 32: 64 rows of 32000, the four settings 35.3 | 40.1, temperature alone 11.6 | 13.0, 1024 of 4000, the four 64.8 | 70.5; top-50,
// 256 rows of 32000 37.2 | 36.3, 1024 of 8000 59.1 | 58.0
static int cut_each(const SampleArgs& a)
{
    const long long slices = (long long)a.count * ((a.vocab + 8 * CUT - 1) / (8 * CUT));
    return slices < 4096 && a.vocab <= 128 * 8 * CUT ? 8 : 32;
}
static bool cut_bins(const SampleArgs& a) { return a.k || a.p; }

static size_t cells_of(SampleType type, int each) { return each / (type == SAMPLE_BF16 ? 8 : 4) * (CUT / 64); }

size_t sample_workspace_bytes(SampleType type, const SampleArgs& a)
{
    if (type == SAMPLE_F64 || !cut(a)) return 0;
    const int each = cut_each(a);
    const size_t slices = (a.vocab + each * CUT - 1) / (each * CUT), rows = a.count;
    return rows * (slices * (8 * cells_of(type, each) + 4) + sizeof(RowState) + 4 * COUNTERS + (cut_bins(a) ? LISTED * 8 + slices * CUT_BINS * 12 : 0));
}

hipError_t k_sample(hipStream_t s, SampleType type, SampleArgs a, void* workspace)
{
    const int chunk = 64 * 16 / (type == SAMPLE_BF16 ? 2 : type == SAMPLE_F32 ? 4 : 8);
    a.perWave = (a.vocab + chunk * WAVES - 1) / (chunk * WAVES);
    a.bits = sample_bits(a.vocab);
    const size_t parts = (size_t)a.perWave * WAVES * sizeof(u64);
    if (workspace) {
        const int each = cut_each(a);
        const size_t rows = a.count;
        SampleCuts w = {};
        w.slices = (a.vocab + each * CUT - 1) / (each * CUT);
        w.sums = (u64*)workspace;
        w.state = w.sums + rows * w.slices * cells_of(type, each);
        char* at = (char*)w.state + rows * sizeof(RowState);
        if (cut_bins(a)) {
            w.list = (u64*)at;
            w.weights = w.list + rows * LISTED;
            w.counts = (uint32_t*)(w.weights + rows * w.slices * CUT_BINS);
            at = (char*)(w.counts + rows * w.slices * CUT_BINS);
        }
        w.listed = (int*)at;
        w.tops = (float*)(w.listed + rows * COUNTERS);
        const dim3 grid(w.slices, a.count);
        auto go = [&](auto type, auto size) {
            typedef decltype(type) L;
            constexpr int EACH = decltype(size)::value;
            hipLaunchKernelGGL((sample_top_kernel<L, EACH>), grid, CUT, 0, s, a, w);
            hipLaunchKernelGGL((sample_weigh_kernel<L, EACH>), grid, CUT, 0, s, a, w);
            hipLaunchKernelGGL((sample_border_kernel<L, EACH>), a.count, CUT, 0, s, a, w);
            if (cut_bins(a)) {
                hipLaunchKernelGGL((sample_list_kernel<L, EACH>), grid, CUT, 0, s, a, w);
                hipLaunchKernelGGL((sample_finish_kernel<L, EACH>), a.count, THREADS, parts, s, a, w);
            }
        };
        auto sized = [&](auto type) {
            if (each == 8) go(type, std::integral_constant<int, 8>{});
            else go(type, std::integral_constant<int, 32>{});
        };
        if (type == SAMPLE_F32) sized(float());
        else sized(bf16_t());
        return hipGetLastError();
    }
    const int x = std::min(a.count, 1 << 21);   // an axis of a launch has less than 2^32 threads
    const dim3 grid(x, (a.count + x - 1) / x);
    if (type == SAMPLE_F32) hipLaunchKernelGGL((sample_kernel<float, float>), grid, THREADS, parts, s, a);
    else if (type == SAMPLE_BF16) hipLaunchKernelGGL((sample_kernel<bf16_t, float>), grid, THREADS, parts, s, a);
    else hipLaunchKernelGGL((sample_kernel<double, double>), grid, THREADS, parts, s, a);
    return hipGetLastError();
}

}  // namespace mch
