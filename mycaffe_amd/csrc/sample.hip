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

constexpr int THREADS = 1024, WAVES = THREADS / 64, BINS = 2048, LIST = 1024;
typedef unsigned long long u64;

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
// one that is not a number is never drawn; -0 is 0
template <typename V> __device__ __forceinline__ V clean(V x) { return x == x ? x + (V)0 : -(V)INFINITY; }
// whole numbers in the order of the logits
__device__ __forceinline__ uint32_t key_of(float x)
{
    const uint32_t u = __float_as_uint(x);
    return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ u64 key_of(double x)
{
    const u64 u = (u64)__double_as_longlong(x);
    return u ^ ((u64)((long long)u >> 63) | 0x8000000000000000ull);
}

__device__ __forceinline__ u64 shfl_up64(u64 v, int o)
{
    const uint32_t lo = __shfl_up((uint32_t)v, o), hi = __shfl_up((uint32_t)(v >> 32), o);
    return (u64)hi << 32 | lo;
}
__device__ __forceinline__ u64 shfl_xor64(u64 v, int o)
{
    const uint32_t lo = __shfl_xor((uint32_t)v, o), hi = __shfl_xor((uint32_t)(v >> 32), o);
    return (u64)hi << 32 | lo;
}
__device__ __forceinline__ u64 wave_sum(u64 v)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += shfl_xor64(v, o);
    return v;
}
__device__ __forceinline__ u64 wave_scan(u64 v)   // up to and with the lane's own
{
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const u64 y = shfl_up64(v, o);
        v += lane >= o ? y : 0;
    }
    return v;
}
// over the workgroup: the sum before the thread's own, and of all (sums: WAVES numbers, read until the next barrier)
__device__ __forceinline__ u64 block_scan(u64 v, u64* sums, u64* all)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const u64 x = wave_scan(v);
    __syncthreads();
    if (lane == 63) sums[wave] = x;
    __syncthreads();
    u64 before = 0, sum = 0;
#pragma unroll
    for (int i = 0; i < WAVES; i++) {
        before += i < wave ? sums[i] : 0;
        sum += sums[i];
    }
    *all = sum;
    return before + x - v;
}

// 2^(j / 16), rounded to nearest
__device__ const double ROOTS[16] = {1.0, 1.0442737824274138, 1.0905077326652577, 1.1387886347566916, 1.189207115002721, 1.2418578120734840, 1.2968395546510096, 1.3542555469368927,
                                     1.4142135623730951, 1.4768261459394993, 1.5422108254079407, 1.6104903319492543, 1.681792830507429, 1.7562521603732995, 1.8340080864093424,
                                     1.9152065613971474};

template <typename L> struct Row {
    typedef typename Logit<L>::V V;
    typedef typename Logit<L>::K K;
    static constexpr int VEC = 16 / (int)sizeof(L), CHUNK = 64 * VEC;   // logits of a lane's piece, of a wavefront's
    const L* x;
    int vocab, perWave;   // chunks of a wavefront, which has one run of them
    V top;
    double rate;          // log2(e) / T
    double scale;         // bins a unit of the logits
    int bits;             // FB
    const double* roots;

    // the pieces of the wavefront in the order of the vocabulary: f(chunk, first index, VEC logits (those behind the row's end -inf))
    template <typename F> __device__ __forceinline__ void each(F f) const
    {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        for (int j = 0; j < perWave; j++) {
            const int i0 = (wave * perWave + j) * CHUNK + lane * VEC;
            if (i0 - lane * VEC >= vocab) break;
            V v[VEC];
            piece(i0, v);
            f(wave * perWave + j, i0, v);
        }
    }
    __device__ __forceinline__ void piece(int i0, V (&v)[VEC]) const
    {
        if (i0 + VEC <= vocab) {
            L raw[VEC];
            __builtin_memcpy(raw, x + i0, sizeof(raw));
#pragma unroll
            for (int e = 0; e < VEC; e++) v[e] = clean<V>(read(raw[e]));
        } else
#pragma unroll
            for (int e = 0; e < VEC; e++) v[e] = i0 + e < vocab ? clean<V>(read(x[i0 + e])) : -(V)INFINITY;
    }
    // log2 of the weight
    __device__ __forceinline__ double power(V v) const
    {
        return v == top ? 0.0 : v > -(V)INFINITY ? ((double)v - (double)top) * rate : -INFINITY;
    }
    // 2^t, t <= 0: 2^(k/16) times the series of exp over +-ln(2)/32, whose seventh term is below 2^-51
    __device__ __forceinline__ double two_to(double t) const
    {
        const double k = rint(t * 16.0), z = fma(k, -0.0625, t) * 0.69314718055994530942;
        const int n = (int)k;
        double s = fma(z, 1.0 / 720, 1.0 / 120);
        s = fma(s, z, 1.0 / 24);
        s = fma(s, z, 1.0 / 6);
        s = fma(s, z, 0.5);
        s = fma(s, z, 1.0);
        s = fma(s, z, 1.0);
        return ldexp(s * roots[n & 15], n >> 4);
    }
    __device__ __forceinline__ u64 weight(V v) const
    {
        const double t = power(v);
        if (!(t > -(double)(bits + 2))) return 0;
        return (u64)(ldexp(two_to(t), bits) + 0.5);
    }
    // falling logits in rising bins; the last one: weight 0
    __device__ __forceinline__ int bin(V v) const
    {
        return v == top ? 0 : v > -(V)INFINITY ? (int)fmin(((double)top - (double)v) * scale, (double)(BINS - 1)) : BINS - 1;
    }
};

struct Shared {
    uint32_t count[BINS];
    u64 weight[BINS];
    u64 sums[WAVES];
    double roots[16];
    u64 keys[LIST], weights[LIST];
    int ids[LIST];
    u64 above, key, least, most;
    int bin, listed, index, found;
};

// p in 0 .. 1 as a fraction of 2^64
__device__ __forceinline__ u64 fraction(double p) { return p >= 1.0 ? ~0ull : p > 0.0 ? (u64)(p * 18446744073709551616.0) : 0; }

// the first index at which the sum of f exceeds `target` (total: asks for the target, given the sum of all).  All threads; -1 if there is none
template <typename R, typename F, typename G> __device__ int locate(const R& r, Shared& s, u64* parts, F f, G target, u64* total)
{
    const int lane = threadIdx.x & 63, tid = threadIdx.x, chunks = r.perWave * WAVES, per = (chunks + THREADS - 1) / THREADS;
    for (int i = tid; i < chunks; i += THREADS) parts[i] = 0;
    if (tid == 0) s.found = -1;
    __syncthreads();
    r.each([&](int chunk, int i0, const typename R::V (&v)[R::VEC]) {
        u64 w = 0;
#pragma unroll
        for (int e = 0; e < R::VEC; e++) w += f(v[e], i0 + e);
        w = wave_sum(w);
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
    __syncthreads();
    if (chunk < 0) return -1;
    if (tid < 64) {
        typename R::V v[R::VEC];
        u64 w[R::VEC], all = 0;
        const int i0 = chunk * R::CHUNK + lane * R::VEC;
        r.piece(min(i0, r.vocab), v);
#pragma unroll
        for (int e = 0; e < R::VEC; e++) {
            w[e] = i0 + e < r.vocab ? f(v[e], i0 + e) : 0;
            all += w[e];
        }
        u64 at = s.above + wave_scan(all) - all;
        if (at <= want && want < at + all)
#pragma unroll
            for (int e = 0; e < R::VEC; e++) {
                if (at <= want && want < at + w[e]) s.found = i0 + e;
                at += w[e];
            }
    }
    __syncthreads();
    const int r0 = s.found;
    __syncthreads();
    return r0;
}

// What is kept: logits with keys above `key`, and equal ones up to index `last`
template <typename K> struct Border {
    K key;
    int last;
    __device__ __forceinline__ bool has(K k, int i) const { return k > key || (k == key && i <= last); }
};

// The border behind which the sum of counts (byWeight: of weights) of the kept tokens, in falling order, reaches the target.  It is looked for in bins of the
// logits, then in ever smaller ranges of keys, until so few are left that each is compared with each, or they are all equal.
template <typename R, typename G> __device__ void select(const R& r, Shared& s, u64* parts, Border<typename R::K>& border, bool byWeight, G targetOf)
{
    typedef typename R::K K;
    typedef typename R::V V;
    const int tid = threadIdx.x, lane = tid & 63;
    const Border<K> old = border;
    // ---- bins of the logits ----
    auto clear = [&]() {
        __syncthreads();
        for (int i = tid; i < BINS; i += THREADS) { s.count[i] = 0; s.weight[i] = 0; }
        if (tid == 0) { s.listed = 0; s.bin = -1; s.least = ~0ull; s.most = 0; }
        __syncthreads();
    };
    clear();
    r.each([&](int, int i0, const V (&v)[R::VEC]) {
#pragma unroll
        for (int e = 0; e < R::VEC; e++) {
            const int b = r.bin(v[e]);
            if (b == BINS - 1 || !old.has(key_of(v[e]), i0 + e)) continue;
            atomicAdd(&s.count[b], 1u);
            if (byWeight) atomicAdd(&s.weight[b], r.weight(v[e]));
        }
    });
    __syncthreads();
    // the bin in which the target is reached: s.bin, and what is above it
    u64 target = 0, above = 0;
    auto pick = [&](bool first) {
        u64 c[2], all;
        for (int i = 0; i < 2; i++) c[i] = byWeight ? s.weight[2 * tid + i] : s.count[2 * tid + i];
        u64 at = above + block_scan(c[0] + c[1], s.sums, &all);
        if (first) target = targetOf(all);
        for (int i = 0; i < 2; i++) {
            if (at < target && target <= at + c[i]) { s.bin = 2 * tid + i; s.above = at; }
            at += c[i];
        }
        __syncthreads();
        above = s.bin >= 0 ? s.above : above;
    };
    pick(true);
    int bin = s.bin;
    if (bin < 0) return;   // all of them, as far as they have weight
    // alive: what of the old border's lies in the range of keys (first: in the bin)
    bool inBin = true;
    K lo = 0, hi = 0;
    uint32_t n = s.count[bin];
    auto alive = [&](V v, int i) -> bool {
        const K k = key_of(v);
        return (inBin ? r.bin(v) == bin : k >= lo && k <= hi) && old.has(k, i);
    };
    while (n > (uint32_t)LIST) {
        // their smallest and largest key
        clear();
        K least = ~(K)0, most = 0;
        r.each([&](int, int i0, const V (&v)[R::VEC]) {
#pragma unroll
            for (int e = 0; e < R::VEC; e++)
                if (i0 + e < r.vocab && alive(v[e], i0 + e)) {
                    const K k = key_of(v[e]);
                    least = min(least, k);
                    most = max(most, k);
                }
        });
        u64 a = least, b = most;
        for (int o = 32; o > 0; o >>= 1) {
            a = min(a, shfl_xor64(a, o));
            b = max(b, shfl_xor64(b, o));
        }
        if (lane == 0 && a <= b) { atomicMin(&s.least, a); atomicMax(&s.most, b); }
        __syncthreads();
        lo = (K)s.least;
        hi = (K)s.most;
        inBin = false;
        if (lo == hi) {
            // all equal: as many as it takes, by their index
            V v0;
            if constexpr (sizeof(K) == 4) v0 = __uint_as_float(lo ^ ((uint32_t)~((int32_t)lo >> 31) | 0x80000000u));
            else v0 = __longlong_as_double((long long)(lo ^ ((u64)~((long long)lo >> 63) | 0x8000000000000000ull)));
            const u64 each = byWeight ? r.weight(v0) : 1, more = (target - above + each - 1) / each;
            u64 total;
            const int last = locate(r, s, parts, [&](V v, int i) -> u64 { return key_of(v) == lo && old.has(lo, i); }, [&](u64) { return more - 1; }, &total);
            border = Border<K>{lo, last};
            return;
        }
        int shift = 0;
        while (((hi - lo) >> shift) >= (K)BINS) shift++;
        clear();
        r.each([&](int, int i0, const V (&v)[R::VEC]) {
#pragma unroll
            for (int e = 0; e < R::VEC; e++)
                if (i0 + e < r.vocab && alive(v[e], i0 + e)) {
                    const int b = (int)((hi - key_of(v[e])) >> shift);
                    atomicAdd(&s.count[b], 1u);
                    if (byWeight) atomicAdd(&s.weight[b], r.weight(v[e]));
                }
        });
        __syncthreads();
        pick(false);
        const K from = (K)s.bin << shift;
        hi -= from;
        const K span = ((K)1 << shift) - 1;
        lo = hi - lo > span ? hi - span : lo;
        n = s.count[s.bin];
    }
    // ---- the few: the one at which the target is reached ----
    __syncthreads();
    if (tid == 0) s.listed = 0;
    __syncthreads();
    r.each([&](int, int i0, const V (&v)[R::VEC]) {
#pragma unroll
        for (int e = 0; e < R::VEC; e++)
            if (i0 + e < r.vocab && alive(v[e], i0 + e)) {
                const int at = atomicAdd(&s.listed, 1);
                if (at < LIST) { s.keys[at] = key_of(v[e]); s.ids[at] = i0 + e; s.weights[at] = byWeight ? r.weight(v[e]) : 1; }
            }
    });
    __syncthreads();
    const int listed = min(s.listed, LIST);
    if (tid < listed) {
        const u64 k = s.keys[tid];
        const int id = s.ids[tid];
        u64 at = above;
        for (int i = 0; i < listed; i++) at += s.keys[i] > k || (s.keys[i] == k && s.ids[i] < id) ? s.weights[i] : 0;
        if (at < target && target <= at + s.weights[tid]) { s.key = k; s.index = id; }
    }
    __syncthreads();
    border = Border<K>{(K)s.key, s.index};
    __syncthreads();
}

template <typename L, typename N> __global__ __launch_bounds__(THREADS) void sample_kernel(SampleArgs a)
{
    typedef Row<L> R;
    typedef typename R::V V;
    typedef typename R::K K;
    __shared__ Shared s;
    __shared__ V sTop[WAVES];
    __shared__ int sAt[WAVES];
    extern __shared__ u64 parts[];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, row = blockIdx.x;
    N *ids = (N*)a.ids, *logs = (N*)a.logs;
    if (tid < 16) s.roots[tid] = ROOTS[tid];
    const N which = a.rows ? ((const N*)a.rows)[row] : (N)row;
    const bool none = !(which >= (N)0 && which < (N)a.logitsRows);
    R r;
    r.x = (const L*)a.x + (none ? 0 : (size_t)(int)which * a.stride);
    r.vocab = a.vocab;
    r.perWave = a.perWave;
    r.roots = s.roots;
    // ---- the largest logit, the first of equal ones ----
    V top = -(V)INFINITY;
    int at = INT32_MAX;
    if (!none)
        r.each([&](int, int i0, const V (&v)[R::VEC]) {
#pragma unroll
            for (int e = 0; e < R::VEC; e++)
                if (v[e] > top) { top = v[e]; at = i0 + e; }
        });
    for (int o = 32; o > 0; o >>= 1) {
        const V t = __shfl_xor(top, o);
        const int i = __shfl_xor(at, o);
        if (t > top || (t == top && i < at)) { top = t; at = i; }
    }
    if (lane == 0) { sTop[wave] = top; sAt[wave] = at; }
    __syncthreads();
    for (int i = 0; i < WAVES; i++)
        if (sTop[i] > top || (sTop[i] == top && sAt[i] < at)) { top = sTop[i]; at = sAt[i]; }
    if (!(top > -(V)INFINITY)) {   // no row, or nothing in it that could be drawn
        if (tid == 0) {
            ids[row] = (N)-1;
            if (logs) logs[row] = (N)0;
        }
        return;
    }
    const N heat = a.temperature ? ((const N*)a.temperature)[row] : (N)1;
    if (!(heat > (N)0)) {
        if (tid == 0) {
            ids[row] = (N)at;
            if (logs) logs[row] = (N)0;
        }
        return;
    }
    r.top = top;
    r.rate = 1.4426950408889634 / (double)heat;
    r.bits = a.bits;
    // logits below the last bin's edge have weights below half of 2^-FB
    r.scale = (BINS - 2) * r.rate / (a.bits + 2);
    const N k = a.k ? ((const N*)a.k)[row] : (N)0, p = a.p ? ((const N*)a.p)[row] : (N)1, m = a.m ? ((const N*)a.m)[row] : (N)0;
    Border<K> border = {0, INT32_MAX};
    if (m > (N)1) border = Border<K>{key_of(top), at};
    else {
        if (k >= (N)1 && k < (N)a.vocab) select(r, s, parts, border, false, [&](u64) { return (u64)k; });
        if (p < (N)1) {
            const u64 part = fraction((double)p);
            select(r, s, parts, border, true, [&](u64 all) { return max(1ull, __umul64hi(all, part) + (all * part ? 1 : 0)); });
        }
    }
    const bool least = m > (N)0 && m <= (N)1;
    const u64 part = fraction((double)((const N*)a.u)[row]);
    u64 total;
    const int id = locate(r, s, parts, [&](V v, int i) -> u64 {
        if (!border.has(key_of(v), i)) return 0;
        if (least && r.two_to(fmax(r.power(v), -1000.0)) < (double)m) return 0;
        return r.weight(v);
    }, [&](u64 all) { return __umul64hi(all, part); }, &total);
    if (tid == 0) {
        ids[row] = (N)id;
        if (logs) {
            const V v = clean<V>(read(r.x[id]));
            logs[row] = (N)(r.power(v) * 0.69314718055994530942 - log(ldexp((double)total, -a.bits)));
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
