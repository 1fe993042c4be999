// Norms of queries and keys for each head with the rotation of their position in the same pass, forward and backward, and the form
// for serving: rows of the q | k | v projection normalised, rotated and, keys and values, stored in the pages of a cache.
//
// For a head x of hs values at position p, with weights w (RMS norm) and the rotation R(p) of adjacent pairs:
//     r = 1 / sqrt(mean(x^2) + eps),   y = R(p) (w x r)
// and its gradient, with g = R(-p) dy:
//     dx = r (g w - x r mean(g w x r)),   dw = sum over the rows of g x r.
// Everything is held in fp32 and rounded once, when it is stored.
//
// All three read and write every value once and compute a handful of operations on it, so memory bounds them (50 MB forward in 10.1 us, 252 MB backward in 53,
// 201 MB appended in 46: 5.0, 4.7 and 4.3 TB/s, where a copy of 4 GiB has 4.5 - 4.8).  A head belongs to a group of
// LPH adjacent lanes, V values a lane (16 bytes), so that the mean is LPH's butterfly and a pair never leaves its lane.
#include <algorithm>
#include <type_traits>

#include "kernels.h"
#include "lane_ops.h"
#include "paged.h"

namespace mch {

namespace {

// V adjacent values of a head: 16 bytes at once where size and addresses allow it (VEC), else one by one up to the head's end
template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f<bf16_t>(bf16_t v) { return bf16_to_f32(v); }
template <typename T> __device__ __forceinline__ T of_f(float v);
template <> __device__ __forceinline__ float of_f<float>(float v) { return v; }
template <> __device__ __forceinline__ bf16_t of_f<bf16_t>(float v) { return f32_to_bf16(v); }

typedef uint32_t u4 __attribute__((ext_vector_type(4)));
template <typename T, int V> struct alignas(16) Piece { T e[V]; };
template <typename T, int V, bool VEC, bool ONCE = false> __device__ __forceinline__ Piece<T, V> piece_load(const T* p, int d0, int hs)
{
    Piece<T, V> r;
    if constexpr (VEC) {
        constexpr int W = (int)sizeof(T) * V / 4;
        uint32_t* w = (uint32_t*)&r;
        if (d0 < hs) {
#pragma unroll
            for (int i = 0; i < W; i += 4) {
                const u4* from = (const u4*)((const uint32_t*)(p + d0) + i);
                *(u4*)(w + i) = ONCE ? __builtin_nontemporal_load(from) : *from;
            }
        } else {
#pragma unroll
            for (int i = 0; i < W; i++) w[i] = 0u;
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; i++) r.e[i] = d0 + i < hs ? p[d0 + i] : T(0);
    }
    return r;
}
template <typename T, int V, bool VEC, bool AWAY = false> __device__ __forceinline__ void piece_store(T* p, int d0, int hs, const float (&v)[V])
{
    if constexpr (VEC) {
        Piece<T, V> r;
#pragma unroll
        for (int i = 0; i < V; i++) r.e[i] = of_f<T>(v[i]);
        constexpr int W = (int)sizeof(T) * V / 4;
        const uint32_t* w = (const uint32_t*)&r;
        if (d0 < hs) {
            if constexpr (W >= 4) {
#pragma unroll
                for (int i = 0; i < W; i += 4) {
                    u4* to = (u4*)((uint32_t*)(p + d0) + i);
                    if (AWAY) __builtin_nontemporal_store(*(const u4*)(w + i), to);
                    else *to = *(const u4*)(w + i);
                }
            } else *(uint2*)(p + d0) = *(const uint2*)w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; i++)
            if (d0 + i < hs) p[d0 + i] = of_f<T>(v[i]);
    }
}
template <typename T, int V> __device__ __forceinline__ void piece_floats(const Piece<T, V>& p, float (&v)[V])
{
#pragma unroll
    for (int i = 0; i < V; i++) v[i] = to_f<T>(p.e[i]);
}
// the weights of a lane's values (1 without weights, 0 past the head's end) and the cosines and sines of its pairs
template <typename T, int V, bool VEC> __device__ __forceinline__ void weights_of(const T* w, int d0, int hs, float (&v)[V])
{
    if (w && VEC) piece_floats<T, V>(piece_load<T, V, VEC>(w, d0, hs), v);
    else
#pragma unroll
        for (int i = 0; i < V; i++) v[i] = d0 + i >= hs ? 0.f : w ? to_f<T>(w[d0 + i]) : 1.f;
}
template <int V> __device__ __forceinline__ void turns_of(const float* turns, int pos, int d0, int hs, float (&c)[V / 2], float (&s)[V / 2])
{
    const float2* t = (const float2*)turns + (size_t)pos * (hs >> 1) + (d0 >> 1);
#pragma unroll
    for (int i = 0; i < V / 2; i++) {
        const float2 cs = turns && d0 + 2 * i < hs ? t[i] : make_float2(1.f, 0.f);
        c[i] = cs.x;
        s[i] = cs.y;
    }
}
template <int V> __device__ __forceinline__ void turn(float (&v)[V], const float (&c)[V / 2], const float (&s)[V / 2])
{
#pragma unroll
    for (int i = 0; i < V / 2; i++) {
        const float a = v[2 * i], b = v[2 * i + 1];
        v[2 * i] = a * c[i] - b * s[i];
        v[2 * i + 1] = a * s[i] + b * c[i];
    }
}
// 1 / sqrt(mean + eps) of a head spread over LPH lanes
template <int LPH, int V> __device__ __forceinline__ float head_rms(const float (&v)[V], float inv_hs, float eps)
{
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < V; i++) ss += v[i] * v[i];
    return 1.0f / sqrtf(group_sum<LPH>(ss) * inv_hs + eps);
}

__global__ void rope_turns_kernel(int n, int half, double theta, float2* turns)
{
    const int i = blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= n) return;
    const int pos = i / half, j = i - pos * half;
    double s, c;
    sincos(pos * pow(theta, -(double)j / half), &s, &c);
    turns[i] = make_float2((float)c, (float)s);
}

// ---- training form ---------------------------------------------------------------------------------------------------------------
struct HeadNormArgs {
    const void *q, *k, *wq, *wk, *dyq, *dyk;
    void *yq, *yk;            // outputs; backward: dx
    const float* turns;
    float* part;              // backward: sums of the weights' gradients, [workgroup][2][hs]
    int B, T, H, kvH, hs;
    float eps, inv_hs;
};
// Heads a lane group has in flight, and how the values that pass through once go by the caches: stores that are not kept there (forward, append),
// loads that are not (backward, whose two inputs are twice its output).  us for 8 x 1024 positions of 24 heads of 64, the gradient at 4 x 2048 of 40
// of 128, 8192 tokens of 48 of 128 appended, 16-bit storage:
//   plain, 4 heads 13.8 | 64 | 63     stores 11.5 (3 heads 10.7) | 60 | 47 (48)     loads 14.0 | 58 (2 heads 53.6) | 48     both 12.9 | 58 | 49
constexpr int AHEAD = 3, AHEAD_BWD = 2;      // heads a lane group has in flight

// A lane group keeps one position and walks the heads of its part, so that cosines, sines and weights are read once for all of them.
// grid: (groups of positions, parts of the heads, groups of positions beyond one axis)
template <typename T, int V, bool VEC, int LPH>
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(HeadNormArgs a)
{
    constexpr int GROUPS = 256 / LPH;
    const int d0 = (threadIdx.x % LPH) * V;
    const long long at = ((long long)blockIdx.z * gridDim.x + blockIdx.x) * GROUPS + threadIdx.x / LPH;
    const bool live = at < (long long)a.B * a.T;
    const int b = live ? (int)(at / a.T) : 0, t = live ? (int)(at - (long long)b * a.T) : 0;
    float c[V / 2], s[V / 2], w[2][V];
    turns_of<V>(a.turns, t, d0, a.hs, c, s);
    weights_of<T, V, VEC>((const T*)a.wq, d0, a.hs, w[0]);
    weights_of<T, V, VEC>((const T*)a.wk, d0, a.hs, w[1]);
    const int heads = a.H + a.kvH;
    // head h of all: where its row starts in its tensor
    const size_t step = (size_t)a.T * a.hs, inq = ((size_t)b * a.H * a.T + t) * a.hs, ink = ((size_t)b * a.kvH * a.T + t) * a.hs;
    auto row = [&](int h) { return h < a.H ? inq + h * step : ink + (h - a.H) * step; };
    Piece<T, V> x[AHEAD];
    auto request = [&](int i, int h) {
        if (h < heads) x[i] = piece_load<T, V, VEC>((h < a.H ? (const T*)a.q : (const T*)a.k) + row(h), live ? d0 : a.hs, a.hs);
    };
    for (int h0 = blockIdx.y; h0 < heads; h0 += AHEAD * gridDim.y) {
#pragma unroll
        for (int i = 0; i < AHEAD; i++) request(i, h0 + i * gridDim.y);
#pragma unroll
        for (int i = 0; i < AHEAD; i++) {
            const int h = h0 + i * gridDim.y;
            if (h >= heads) break;
            float v[V];
            piece_floats<T, V>(x[i], v);
            const float r = head_rms<LPH, V>(v, a.inv_hs, a.eps);
#pragma unroll
            for (int e = 0; e < V; e++) v[e] = v[e] * r * (h < a.H ? w[0][e] : w[1][e]);
            turn<V>(v, c, s);
            if (live) piece_store<T, V, VEC, true>((h < a.H ? (T*)a.yq : (T*)a.yk) + row(h), d0, a.hs, v);
        }
    }
}

// The gradient, with the same walk; a workgroup takes every gridDim.x-th group of positions and every gridDim.y-th head.  The weights' gradients stay in registers, meet
// in a fixed order, and leave as one row of sums a workgroup, which head_norm_dw_kernel adds in order: no sum depends on timing.
template <typename T, int V, bool VEC, int LPH>
__global__ __launch_bounds__(256) void qk_norm_rope_bwd_kernel(HeadNormArgs a)
{
    constexpr int GROUPS = 256 / LPH;
    __shared__ float red[4][2][LPH * V + 1];
    const int d0 = (threadIdx.x % LPH) * V, group = threadIdx.x / LPH;
    const int heads = a.H + a.kvH;
    float w[2][V], dw[2][V];
    weights_of<T, V, VEC>((const T*)a.wq, d0, a.hs, w[0]);
    weights_of<T, V, VEC>((const T*)a.wk, d0, a.hs, w[1]);
#pragma unroll
    for (int e = 0; e < V; e++) dw[0][e] = dw[1][e] = 0.f;
    const long long positions = (long long)a.B * a.T;
    for (long long at0 = (long long)blockIdx.x * GROUPS; at0 < positions; at0 += (long long)gridDim.x * GROUPS) {
        const long long at = at0 + group;
        const bool live = at < positions;
        const int b = live ? (int)(at / a.T) : 0, t = live ? (int)(at - (long long)b * a.T) : 0;
        float c[V / 2], s[V / 2];
        turns_of<V>(a.turns, t, d0, a.hs, c, s);
#pragma unroll
        for (int i = 0; i < V / 2; i++) s[i] = -s[i];
        const int dl = live ? d0 : a.hs;
        const size_t step = (size_t)a.T * a.hs, inq = ((size_t)b * a.H * a.T + t) * a.hs, ink = ((size_t)b * a.kvH * a.T + t) * a.hs;
        auto row = [&](int h) { return h < a.H ? inq + h * step : ink + (h - a.H) * step; };
        Piece<T, V> x[AHEAD_BWD], g[AHEAD_BWD];
        auto request = [&](int i, int h) {
            if (h >= heads) return;
            x[i] = piece_load<T, V, VEC, true>((h < a.H ? (const T*)a.q : (const T*)a.k) + row(h), dl, a.hs);
            g[i] = piece_load<T, V, VEC, true>((h < a.H ? (const T*)a.dyq : (const T*)a.dyk) + row(h), dl, a.hs);
        };
        for (int h0 = blockIdx.y; h0 < heads; h0 += AHEAD_BWD * gridDim.y) {
#pragma unroll
            for (int i = 0; i < AHEAD_BWD; i++) request(i, h0 + i * gridDim.y);
#pragma unroll
            for (int i = 0; i < AHEAD_BWD; i++) {
                const int h = h0 + i * gridDim.y;
                if (h >= heads) break;
                const bool isq = h < a.H;
                float xv[V], gv[V];
                piece_floats<T, V>(x[i], xv);
                piece_floats<T, V>(g[i], gv);
                turn<V>(gv, c, s);
                // a lane group without a position has no part in the sums, also where its zeros have no norm (eps 0)
                const float rms = head_rms<LPH, V>(xv, a.inv_hs, a.eps), r = live ? rms : 0.f;
                float dot = 0.f;
#pragma unroll
                for (int e = 0; e < V; e++) {
                    xv[e] *= r;
                    const float gx = gv[e] * xv[e];
                    if (isq) dw[0][e] += gx; else dw[1][e] += gx;
                    gv[e] *= isq ? w[0][e] : w[1][e];
                    dot += gv[e] * xv[e];
                }
                const float mean = group_sum<LPH>(dot) * a.inv_hs;
#pragma unroll
                for (int e = 0; e < V; e++) gv[e] = r * (gv[e] - xv[e] * mean);
                if (live) piece_store<T, V, VEC>((isq ? (T*)a.yq : (T*)a.yk) + row(h), d0, a.hs, gv);
            }
        }
    }
    if (!a.part) return;
    // the lane groups of a wavefront, then the wavefronts
#pragma unroll
    for (int x = 0; x < 2; x++)
#pragma unroll
        for (int e = 0; e < V; e++) {
            float v = dw[x][e];
            if constexpr (LPH <= 8) v = add_lane_xor<8>(v);
            if constexpr (LPH <= 16) v = add_lane_xor<16>(v);
            if constexpr (LPH <= 32) v = add_lane_xor<32>(v);
            if ((threadIdx.x & 63) < LPH) red[threadIdx.x >> 6][x][d0 + e] = v;
        }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * a.hs; i += 256) {
        const int x = i / a.hs, d = i - x * a.hs;
        a.part[((size_t)blockIdx.y * gridDim.x + blockIdx.x) * 2 * a.hs + i] = (red[0][x][d] + red[1][x][d]) + (red[2][x][d] + red[3][x][d]);
    }
}
// 16 columns by 64 lanes of workgroups; the lanes' sums are added in order
template <typename T>
__global__ __launch_bounds__(1024) void head_norm_dw_kernel(const float* part, int rows, int hs, T* dwq, T* dwk, int accum)
{
    __shared__ float red[64][17];
    const int c = threadIdx.x & 15, r = threadIdx.x >> 4, j = blockIdx.x * 16 + c;
    float acc = 0.f;
    if (j < 2 * hs)
#pragma unroll 8
        for (int i = r; i < rows; i += 64) acc += part[(size_t)i * 2 * hs + j];
    red[r][c] = acc;
    __syncthreads();
    if (r < 4) {
        float t = 0.f;
#pragma unroll
        for (int q = 0; q < 16; q++) t += red[16 * r + q][c];
        red[16 * r][c] = t;
    }
    __syncthreads();
    if (r == 0 && j < 2 * hs) {
        const float t = (red[0][c] + red[16][c]) + (red[32][c] + red[48][c]);
        T* dw = j < hs ? dwq : dwk;
        if (dw) {
            T* p = dw + (j < hs ? j : j - hs);
            *p = of_f<T>(accum ? to_f<T>(*p) + t : t);
        }
    }
}

// ---- serving form -----------------------------------------------------------------------------------------------------------------
struct AppendArgs {
    PagedCache c;
    const void *qkv, *wq, *wk;
    void* q;
    const float* turns;
    float eps, inv_hs;
    int norm;
};

// A wavefront has one token and every gridDim.y-th set of 64 / LPH of its heads.  What the position is and where its page lies takes three reads
// one after the other (starts, length, table entry); the rows' values are requested before that.
template <typename T, typename TC, int V, bool VEC, int LPH>
__global__ __launch_bounds__(256) void paged_append_kernel(AppendArgs a)
{
    constexpr int HPW = 64 / LPH;
    const PagedCache& c = a.c;
    const int lane = threadIdx.x & 63, d0 = (lane % LPH) * V, token = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (token >= c.tokens) return;
    const int heads = c.H + 2 * c.kvH, stride = HPW * gridDim.y;
    const T* row = (const T*)a.qkv + (size_t)token * heads * c.hs;
    int h0 = blockIdx.y * HPW + lane / LPH;
    Piece<T, V> x[AHEAD];
    auto request = [&](int i, int h) {
        if (h < heads) x[i] = piece_load<T, V, VEC>(row + (size_t)h * c.hs, d0, c.hs);
    };
#pragma unroll
    for (int i = 0; i < AHEAD; i++) request(i, h0 + i * stride);
    const int b = sequence_of(c.starts, c.batch, c.tokens, token);
    if (b < 0) return;
    const int positions = c.maxPages * c.pageSize;
    const PagedSpan sp = paged_span(c.starts[b], c.starts[b + 1], c.lens[b], c.tokens, positions);
    if (token >= sp.first + sp.count) return;   // a row behind the last sequence
    const int pos = sp.len - sp.count + (token - sp.first);
    const int entry = max(pos, 0) / c.pageSize;
    const int page = pos >= 0 ? paged_page(c.table[(size_t)b * c.maxPages + entry], c.pages) : -1;
    const long long at = page * c.sP + (max(pos, 0) - entry * c.pageSize) * c.sT;
    float cs[V / 2], sn[V / 2], w[2][V];
    turns_of<V>(a.turns, max(pos, 0), d0, c.hs, cs, sn);
    weights_of<T, V, VEC>((const T*)a.wq, d0, c.hs, w[0]);
    weights_of<T, V, VEC>((const T*)a.wk, d0, c.hs, w[1]);
    // the walk is the wavefront's (its butterflies want all lanes); a lane group past the last head stores nothing
    for (int first = blockIdx.y * HPW; first < heads; first += AHEAD * stride) {
#pragma unroll
        for (int i = 0; i < AHEAD; i++) {
            const int h = h0 + i * stride;
            if (first + i * stride >= heads) break;
            const bool isq = h < c.H, isk = !isq && h < c.H + c.kvH;
            float v[V];
            piece_floats<T, V>(x[i], v);
            const float r = a.norm ? head_rms<LPH, V>(v, a.inv_hs, a.eps) : 1.f;
            if (isq || isk) {
                if (a.norm)
#pragma unroll
                    for (int e = 0; e < V; e++) v[e] = v[e] * r * (isq ? w[0][e] : w[1][e]);
                turn<V>(v, cs, sn);
            }
            if (isq) piece_store<T, V, VEC, true>((T*)a.q + ((size_t)token * c.H + h) * c.hs, d0, c.hs, v);
            else if (h < heads && page >= 0)
                piece_store<TC, V, VEC, true>((TC*)(isk ? c.k : c.v) + at + (h - c.H - (isk ? 0 : c.kvH)) * c.sH, d0, c.hs, v);
        }
        h0 += AHEAD * stride;
#pragma unroll
        for (int i = 0; i < AHEAD; i++) request(i, h0 + i * stride);
    }
}

inline bool at16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// Values a lane: 8 in 16-bit storage, 4 in fp32, 16 bytes either way; lanes a head: the power of two from 8 up that covers hs
template <typename F> hipError_t with_lanes(int hs, int V, F f)
{
    const int need = (hs + V - 1) / V;
    if (need <= 8) return f(std::integral_constant<int, 8>{});
    if (need <= 16) return f(std::integral_constant<int, 16>{});
    if (need <= 32) return f(std::integral_constant<int, 32>{});
    if (need <= 64) return f(std::integral_constant<int, 64>{});
    return hipErrorInvalidValue;
}
template <typename F> hipError_t with_bool(bool b, F f) { return b ? f(std::integral_constant<bool, true>{}) : f(std::integral_constant<bool, false>{}); }
template <typename T> constexpr int values_a_lane() { return 16 / (int)sizeof(T); }

// workgroups of the backward pass, of `groups` positions at a time, and parts their heads are dealt to: enough for the chip, few enough rows of sums
constexpr int BWD_BLOCKS = 1024;
inline dim3 bwd_grid(long long positions, int groups, int heads)
{
    const int blocks = (int)std::min<long long>((positions + groups - 1) / groups, BWD_BLOCKS);
    return dim3(blocks, std::max(1, std::min(heads, BWD_BLOCKS / blocks)));
}

}  // namespace

hipError_t k_rope_turns(hipStream_t s, int seq, int hs, float theta, float* turns)
{
    const int n = seq * (hs / 2);
    hipLaunchKernelGGL(rope_turns_kernel, (n + 255) / 256, 256, 0, s, n, hs / 2, (double)theta, (float2*)turns);
    return hipGetLastError();
}

hipError_t k_qk_norm_rope(hipStream_t s, DType dt, int B, int T, int H, int kvH, int hs, const void* q, const void* k, const void* wq, const void* wk,
                          const float* turns, void* yq, void* yk, float eps)
{
    HeadNormArgs a = {};
    a.q = q; a.k = k; a.wq = wq; a.wk = wk; a.yq = yq; a.yk = yk; a.turns = turns;
    a.B = B; a.T = T; a.H = H; a.kvH = kvH; a.hs = hs; a.eps = eps; a.inv_hs = 1.0f / hs;
    auto go = [&](auto type) {
        typedef decltype(type) T_;
        constexpr int V = values_a_lane<T_>();
        const bool vec = hs % V == 0 && at16(q) && at16(k) && at16(yq) && at16(yk) && at16(wq) && at16(wk);
        return with_bool(vec, [&](auto vec_) {
            return with_lanes(hs, V, [&](auto lanes) {
                constexpr int LPH = decltype(lanes)::value, GROUPS = 256 / LPH;
                const long long blocks = ((long long)B * T + GROUPS - 1) / GROUPS;
                // few positions: their heads are dealt to several workgroups
                const int parts = (int)std::max<long long>(1, std::min<long long>(H + kvH, 2048 / blocks));
                const unsigned x = (unsigned)std::min<long long>(blocks, 1 << 23);   // an axis of a launch has less than 2^32 threads
                hipLaunchKernelGGL((qk_norm_rope_kernel<T_, V, decltype(vec_)::value, LPH>), dim3(x, parts, (unsigned)((blocks + x - 1) / x)), 256, 0, s, a);
                return hipGetLastError();
            });
        });
    };
    return dt == F32 ? go(float()) : go(bf16_t());
}

size_t k_qk_norm_rope_bwd_workspace_bytes(int hs) { return (size_t)BWD_BLOCKS * 2 * hs * sizeof(float); }

hipError_t k_qk_norm_rope_bwd(hipStream_t s, DType dt, int B, int T, int H, int kvH, int hs, const void* q, const void* k, const void* wq, const void* wk,
                              const float* turns, const void* dyq, const void* dyk, void* dxq, void* dxk, void* dwq, void* dwk, bool accum, float eps,
                              void* workspace)
{
    HeadNormArgs a = {};
    a.q = q; a.k = k; a.wq = wq; a.wk = wk; a.dyq = dyq; a.dyk = dyk; a.yq = dxq; a.yk = dxk; a.turns = turns;
    a.part = dwq || dwk ? (float*)workspace : nullptr;
    a.B = B; a.T = T; a.H = H; a.kvH = kvH; a.hs = hs; a.eps = eps; a.inv_hs = 1.0f / hs;
    auto go = [&](auto type) {
        typedef decltype(type) T_;
        constexpr int V = values_a_lane<T_>();
        const bool vec = hs % V == 0 && at16(q) && at16(k) && at16(dyq) && at16(dyk) && at16(dxq) && at16(dxk) && at16(wq) && at16(wk);
        dim3 grid;
        hipError_t e = with_bool(vec, [&](auto vec_) {
            return with_lanes(hs, V, [&](auto lanes) {
                constexpr int LPH = decltype(lanes)::value;
                grid = bwd_grid((long long)B * T, 256 / LPH, H + kvH);
                hipLaunchKernelGGL((qk_norm_rope_bwd_kernel<T_, V, decltype(vec_)::value, LPH>), grid, 256, 0, s, a);
                return hipGetLastError();
            });
        });
        if (e != hipSuccess || !a.part) return e;
        hipLaunchKernelGGL((head_norm_dw_kernel<T_>), (2 * hs + 15) / 16, 1024, 0, s, a.part, (int)(grid.x * grid.y), hs, (T_*)dwq, (T_*)dwk, accum ? 1 : 0);
        return hipGetLastError();
    };
    return dt == F32 ? go(float()) : go(bf16_t());
}

hipError_t k_paged_append(hipStream_t s, DType dt, const PagedCache& c, const void* qkv, void* q, const void* wq, const void* wk, bool norm, float eps,
                          const float* turns)
{
    AppendArgs a = {};
    a.c = c; a.qkv = qkv; a.wq = wq; a.wk = wk; a.q = q; a.turns = turns; a.eps = eps; a.inv_hs = 1.0f / c.hs; a.norm = norm;
    auto go = [&](auto type, auto ctype) {
        typedef decltype(type) T_;
        typedef decltype(ctype) TC_;
        constexpr int V = values_a_lane<T_>();
        const bool vec = c.hs % V == 0 && c.sP % V == 0 && c.sH % V == 0 && c.sT % V == 0 && at16(qkv) && at16(q) && at16(c.k) && at16(c.v) && at16(wq) && at16(wk);
        return with_bool(vec, [&](auto vec_) {
            return with_lanes(c.hs, V, [&](auto lanes) {
                constexpr int LPH = decltype(lanes)::value, HPW = 64 / LPH;
                const int sets = (c.H + 2 * c.kvH + HPW - 1) / HPW;
                // few tokens: their heads are dealt to several wavefronts
                const int parts = std::max(1, std::min(sets, 4096 / c.tokens));
                hipLaunchKernelGGL((paged_append_kernel<T_, TC_, V, decltype(vec_)::value, LPH>), dim3((c.tokens + 3) / 4, parts), 256, 0, s, a);
                return hipGetLastError();
            });
        });
    };
    if (dt == F32) return c.ct == F32 ? go(float(), float()) : go(float(), bf16_t());
    return go(bf16_t(), bf16_t());
}

}  // namespace mch
