// Attention of the new tokens of many sequences, one token or a chunk each, over keys and values in the pages of a cache.
//
// Token j of the n new ones of a sequence of len cached positions (the new ones last) is at position p = len - n + j:
//     y = sum over the positions t <= p whose page is given of softmax(scale q . k_t) v_t,   0 where there is none.
// What lies in positions that a token does not see (behind its own, behind the sequence, in pages not given) has no say, whatever it is; scores
// that are all -inf have no weights (0 / 0).
// Softmax statistics and sums are held in fp32; y is rounded once.
#include <algorithm>
#include <type_traits>

#include "kernels.h"
#include "lane_ops.h"
#include "paged.h"

namespace mch {

namespace {

struct PagedAttnArgs {
    PagedCache c;
    const void* q;
    void* y;
    float c2;   // scale * log2(e)
};

template <typename T> __device__ __forceinline__ float value_of(T v);
template <> __device__ __forceinline__ float value_of<float>(float v) { return v; }
template <> __device__ __forceinline__ float value_of<bf16_t>(bf16_t v) { return bf16_to_f32(v); }
template <typename T> __device__ __forceinline__ T stored(float v);
template <> __device__ __forceinline__ float stored<float>(float v) { return v; }
template <> __device__ __forceinline__ bf16_t stored<bf16_t>(float v) { return f32_to_bf16(v); }

// the sequence whose rows hold token `i`: the last one that starts at or before it.  All 64 lanes ask.
__device__ __forceinline__ int sequence_of(const float* starts, int batch, int tokens, int i)
{
    int n = 0;
    for (int b0 = 0; b0 < batch; b0 += 64) {
        const int b = b0 + (threadIdx.x & 63);
        const bool before = b < batch && paged_int(starts[b], 0, tokens) <= i;
        const uint64_t m = __ballot(before);
        if (!m) break;
        n = b0 + 64 - __builtin_clzll(m);
    }
    return n - 1;
}

// Any head size up to 256, any strides: a wavefront has one token's head, a group of LPH lanes every (64 / LPH)-th position, V values a lane.
template <typename T, typename TC, int V, int LPH>
__global__ __launch_bounds__(256) void attn_paged_any_kernel(PagedAttnArgs a)
{
    constexpr int GROUPS = 64 / LPH;
    const PagedCache& c = a.c;
    const int lane = threadIdx.x & 63, d0 = (lane % LPH) * V;
    const int token = blockIdx.x, h = blockIdx.y * 4 + (threadIdx.x >> 6);
    if (h >= c.H) return;
    const int b = sequence_of(c.starts, c.batch, c.tokens, token);
    if (b < 0) return;
    const PagedSpan sp = paged_span(c.starts[b], c.starts[b + 1], c.lens[b], c.tokens, c.maxPages * c.pageSize);
    if (token >= sp.first + sp.count) return;   // a row behind the last sequence
    const int last = sp.len - sp.count + (token - sp.first), kh = h / (c.H / c.kvH);
    const T* q = (const T*)a.q + ((size_t)token * c.H + h) * c.hs;
    float qv[V], acc[V], m = -INFINITY, l = 0.f;
    bool seen = false;
#pragma unroll
    for (int i = 0; i < V; i++) {
        qv[i] = d0 + i < c.hs ? value_of<T>(q[d0 + i]) : 0.f;
        acc[i] = 0.f;
    }
    for (int t = lane / LPH; t <= last; t += GROUPS) {
        const int entry = t / c.pageSize, page = paged_page(c.table[(size_t)b * c.maxPages + entry], c.pages);
        const bool given = page >= 0;
        const long long at = given ? page * c.sP + kh * c.sH + (t - entry * c.pageSize) * c.sT : 0;
        const TC *k = (const TC*)c.k + at, *v = (const TC*)c.v + at;
        float dot = 0.f;
#pragma unroll
        for (int i = 0; i < V; i++)
            if (d0 + i < c.hs) dot += qv[i] * value_of<TC>(k[d0 + i]);
        dot = group_sum<LPH>(dot) * a.c2;
        if (!given) continue;
        seen = true;
        const float mn = fmaxf(m, dot), ref = mn > -INFINITY ? mn : 0.f, f = exp2f(m - ref), w = exp2f(dot - ref);
        m = mn;
        l = l * f + w;
#pragma unroll
        for (int i = 0; i < V; i++) acc[i] = acc[i] * f + (d0 + i < c.hs ? w * value_of<TC>(v[d0 + i]) : 0.f);
    }
    // the groups' sums meet; a group without positions has weight 0
    float M = m;
#pragma unroll
    for (int o = LPH; o < 64; o <<= 1) M = fmaxf(M, __shfl_xor(M, o));
    const float f = exp2f(m - (M > -INFINITY ? M : 0.f));
    seen = __any(seen);
    l *= f;
#pragma unroll
    for (int o = LPH; o < 64; o <<= 1) l += __shfl_xor(l, o);
    T* y = (T*)a.y + ((size_t)token * c.H + h) * c.hs;
#pragma unroll
    for (int i = 0; i < V; i++) {
        float s = acc[i] * f;
#pragma unroll
        for (int o = LPH; o < 64; o <<= 1) s += __shfl_xor(s, o);
        if (lane < LPH && d0 + i < c.hs) y[d0 + i] = stored<T>(seen ? s / l : 0.f);
    }
}

}  // namespace

hipError_t k_attn_paged(hipStream_t s, DType dt, const PagedCache& c, const void* q, void* y, float scale)
{
    PagedAttnArgs a = {};
    a.c = c; a.q = q; a.y = y; a.c2 = scale * 1.44269504088896340736f;
    auto go = [&](auto type, auto ctype) {
        typedef decltype(type) T_;
        typedef decltype(ctype) TC_;
        const dim3 grid(c.tokens, (c.H + 3) / 4);
        if (c.hs <= 64) hipLaunchKernelGGL((attn_paged_any_kernel<T_, TC_, 4, 16>), grid, 256, 0, s, a);
        else if (c.hs <= 128) hipLaunchKernelGGL((attn_paged_any_kernel<T_, TC_, 4, 32>), grid, 256, 0, s, a);
        else hipLaunchKernelGGL((attn_paged_any_kernel<T_, TC_, 4, 64>), grid, 256, 0, s, a);
        return hipGetLastError();
    };
    if (dt == F32) return c.ct == F32 ? go(float(), float()) : go(float(), bf16_t());
    return go(bf16_t(), bf16_t());
}

}  // namespace mch
