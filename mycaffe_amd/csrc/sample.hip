// The next token of every row of logits, drawn with a given random number.
//
// Weights w_i = exp((x_i - max x) / T).  Of the tokens in falling order of x, equal ones by their index: top-k keeps the first k, top-p of these the shortest run
// whose weights add up to at least p of theirs, min-p those with w >= m.  Drawn is the first token, in the order of the vocabulary, at which the sum of the weights of
// those that are left exceeds u times all of it.
//
// A draw compares u with sums over the whole vocabulary: a sum that is off by e moves every border by e, so with 100000 tokens fp32 sums draw another token every
// few hundred rows.  Weights are made in 64 bits and held as whole numbers of 2^-FB, which add up to the same in any order; their sums are exact.
#include <algorithm>

#include "kernels.h"

namespace mch {

namespace {

constexpr int THREADS = 1024, WAVES = THREADS / 64, BINS = 2048, FEW = 256;
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
__device__ __forceinline__ u64 block_scan(u64 v, u64* sums, u64* all)
{
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const u64 x = wave_scan(v);
    __syncthreads();
    if (lane == 63) sums[wave] = x;
    __syncthreads();
    u64 each = sums[lane & (WAVES - 1)];   // sums of the wavefronts up to the lane's
    each += dpp64<0x111, 0xf>(each);
    each += dpp64<0x112, 0xf>(each);
    each += dpp64<0x114, 0xf>(each);
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
        shift = n <= THREADS / 16 ? 4 : n <= THREADS / 4 ? 2 : 1;
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

// The draw from the listed tokens alone.  k: of them the first (0: all), targetOf(sum): the sum of weights at which top-p's run ends (0: all), least: weights from here on
template <typename R, typename G> __device__ __forceinline__ int draw_of_few(const R& r, Shared& s, int n, u64 k, G targetOf, double least, u64 share, u64* total)
{
    const int lane = threadIdx.x & 63;
    const Rank me(s, n);
    const u64 rank = me.sum(n, [&](int j) __attribute__((always_inline)) -> u64 { return me.before(s, j); });
    const u64 better = me.sum(n, [&](int j) __attribute__((always_inline)) -> u64 { return me.before(s, j) ? s.weights[j] : 0; });
    auto all = [&]() __attribute__((always_inline)) -> u64 {   // every wavefront for itself
        u64 x = 0;
        for (int j = lane; j < n; j += 64) x += s.kept[j];
        return wave_sum(x);
    };
    bool keep = me.mine && (k == 0 || rank < k);
    if (me.lead) s.kept[me.i] = keep ? me.w : 0;
    if (threadIdx.x == 0) s.found = -1;
    __syncthreads();
    const u64 target = targetOf(all());
    keep = keep && (rank == 0 || ((target == 0 || better < target) && (least == 0.0 || r.two_to(r.power((typename R::V)me.v), 0) >= least)));
    __syncthreads();
    if (me.lead) s.kept[me.i] = keep ? me.w : 0;
    __syncthreads();
    *total = all();
    const u64 want = __umul64hi(*total, share), before = me.sum(n, [&](int j) __attribute__((always_inline)) -> u64 { return s.ids[j] < me.id ? s.kept[j] : 0; });
    if (me.lead && keep && before <= want && want < before + me.w) s.found = me.id;
    __syncthreads();
    return s.found;
}

template <typename L, typename N> __global__ __launch_bounds__(THREADS) void sample_kernel(SampleArgs a)
{
    typedef Row<L> R;
    typedef typename R::V V;
    __shared__ Shared s;
    __shared__ V sTop[WAVES];
    extern __shared__ u64 parts[];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, row = blockIdx.x;
    N *ids = (N*)a.ids, *logs = (N*)a.logs;
    if (tid < 32) s.roots[tid] = ROOTS[tid];
    const N which = a.rows ? ((const N*)a.rows)[row] : (N)row;
    const bool none = !(which >= (N)0 && which < (N)a.logitsRows);
    R r;
    r.x = (const L*)a.x + (none ? 0 : (size_t)(int)which * a.stride);
    r.vocab = a.vocab;
    r.perWave = a.perWave;
    r.roots = s.roots;
    // ---- the largest logit ----
    r.infinite = false;
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
        if (tid == 0) {
            ids[row] = (N)-1;
            if (logs) logs[row] = (N)0;
        }
        return;
    }
    r.infinite = top == (V)INFINITY;
    top = r.infinite ? (V)0 : top;
    r.top = top;
    r.bits = a.bits;
    r.least = -32.0 * (a.bits + 2);
    const N heat = a.temperature ? ((const N*)a.temperature)[row] : (N)1, k = a.k ? ((const N*)a.k)[row] : (N)0, p = a.p ? ((const N*)a.p)[row] : (N)1;
    const N m = a.m ? ((const N*)a.m)[row] : (N)0;
    r.rate = heat > (N)0 ? fmin(32 * 1.4426950408889634 / (double)heat, 1e300) : 0.0;
    Border<V> border = {-(V)INFINITY, INT32_MAX};
    const bool first = !(heat > (N)0) || m > (N)1;   // of the largest logits the first one, whatever else
    const bool byK = !first && k >= (N)1 && k < (N)a.vocab, byP = !first && p < (N)1;
    const u64 run = fraction((double)p), share = first ? 0 : fraction((double)((const N*)a.u)[row]);
    const double least = !first && m > (N)0 ? (double)m : 0.0;
    auto run_of = [&](u64 all) __attribute__((always_inline)) -> u64 { return max(1ull, __umul64hi(all, run) + (all * run ? 1 : 0)); };
    u64 total, target = 0;
    int id = -1, few;
#pragma unroll 1
    for (int filter = 0; filter < 2; filter++) {
        if (!(filter ? byP : byK)) continue;
        border = select(r, s, parts, border, !filter || !byK, filter != 0, &target, &few, [&](u64 all) __attribute__((always_inline)) -> u64 { return filter ? run_of(all) : (u64)k; });
        if (few) {
            id = draw_of_few(r, s, few, filter ? 0 : (u64)k, [&](u64 all) __attribute__((always_inline)) -> u64 { return filter ? target : byP ? run_of(all) : 0; }, least, share, &total);
            break;
        }
    }
    if (id < 0 && least > 0.0) {   // weights from here on are logits from here on
        const V at = r.smallest([&](V v) __attribute__((always_inline)) { return r.two_to(r.power(v), 0) >= least; });
        if (at > border.at) border = Border<V>{at, INT32_MAX};
    }
    auto target_of = [&](u64 all) __attribute__((always_inline)) -> u64 { return __umul64hi(all, share); };
    if (first) id = locate_equal(r, s, parts, top, border, 1);
    else if (id < 0) {
        const bool some = border.at > -(V)INFINITY;
        id = locate(r, s, parts, [&](const V (&v)[R::VEC], int i0) __attribute__((always_inline)) -> u64 {
            u64 sum = 0;
            if (!some) {
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
        }, [&](V v, int i) __attribute__((always_inline)) -> u64 { return border.has(v, i) ? r.weight(v) : 0; }, target_of, &total);
    }
    if (tid == 0) {
        ids[row] = (N)id;
        if (logs) {
            const V v = r.infinite ? top : (V)read(r.x[id]);
            logs[row] = first ? (N)0 : (N)(fmin(((double)v - (double)top) * r.rate, 0.0) * (0.69314718055994530942 / 32) - log(ldexp((double)total, -a.bits)));
        }
    }
}

}  // namespace

// bits of a weight behind the point: what the sum over the vocabulary leaves of 64
int sample_bits(int vocab)
{
    int log = 0;
    while ((1 << log) < vocab) log++;
    return std::min(50, 63 - log);
}

hipError_t k_sample(hipStream_t s, SampleType type, SampleArgs a)
{
    const int chunk = 64 * 16 / (type == SAMPLE_BF16 ? 2 : type == SAMPLE_F32 ? 4 : 8);
    a.perWave = (a.vocab + chunk * WAVES - 1) / (chunk * WAVES);
    a.bits = sample_bits(a.vocab);
    const size_t parts = (size_t)a.perWave * WAVES * sizeof(u64);
    if (type == SAMPLE_F32) hipLaunchKernelGGL((sample_kernel<float, float>), a.count, THREADS, parts, s, a);
    else if (type == SAMPLE_BF16) hipLaunchKernelGGL((sample_kernel<bf16_t, float>), a.count, THREADS, parts, s, a);
    else hipLaunchKernelGGL((sample_kernel<double, double>), a.count, THREADS, parts, s, a);
    return hipGetLastError();
}

}  // namespace mch
