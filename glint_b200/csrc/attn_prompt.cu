/* Causal attention over packed prompts with grouped heads.
 *
 * One warp per query row: a lane holds D / 32 values of q and of the output (element
 * lane + 32 i, so loads are coalesced at any alignment), each key's score is a shuffle
 * sum, and the running maximum and sum of the softmax rescale the output as they
 * change.  Simple and right for every case.
 */
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "../../include/glint_attn.h"
#include "common.cuh"
#include "glint_internal.h"

namespace glint {
namespace {

constexpr int kWarps = 4;

/* sequence of query token t and its bounds; false for a token outside every sequence */
struct Span {
    int q0, q1, k0, k1;
};
__device__ __forceinline__ int bound(const int *cu, int i, int most) { return min(max(cu[i], 0), most); }
__device__ __forceinline__ bool span_of(const GlintAttnPrompt &a, int t, Span &s)
{
    int lo = 0, hi = a.seqs; /* first i with cu_q[i + 1] > t */
    while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (bound(a.cu_q, mid + 1, a.q_tokens) > t)
            hi = mid;
        else
            lo = mid + 1;
    }
    if (lo >= a.seqs || t < bound(a.cu_q, lo, a.q_tokens))
        return false;
    s.q0 = bound(a.cu_q, lo, a.q_tokens), s.q1 = bound(a.cu_q, lo + 1, a.q_tokens);
    s.k0 = bound(a.cu_k, lo, a.k_tokens), s.k1 = max(s.k0, bound(a.cu_k, lo + 1, a.k_tokens));
    return true;
}

template <int D>
__device__ void plain_row(const GlintAttnPrompt &a, const Span &s, int t, int hq, int lane)
{
    const int h = hq / (a.heads / a.kv_heads);
    const int seen = a.causal ? min(s.k1 - s.k0, t - s.q0 + 1 + (s.k1 - s.k0) - (s.q1 - s.q0)) : s.k1 - s.k0;
    float q[D / 32], o[D / 32] = {}, m = -INFINITY, l = 0.f;
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
        q[i] = __bfloat162float(a.q[t * a.q_tok + hq * a.q_head + lane + 32 * i]);
    for (int j = 0; j < seen; ++j) {
        const __nv_bfloat16 *k = a.k + (int64_t)(s.k0 + j) * a.k_tok + h * a.k_head + lane;
        const __nv_bfloat16 *v = a.v + (int64_t)(s.k0 + j) * a.v_tok + h * a.v_head + lane;
        float x = 0.f;
#pragma unroll
        for (int i = 0; i < D / 32; ++i)
            x = fmaf(q[i], __bfloat162float(k[32 * i]), x);
        x = warp_sum(x) * a.scale;
        const float top = fmaxf(m, x);
        const float keep = m == -INFINITY ? 0.f : expf(m - top), p = x == -INFINITY ? 0.f : expf(x - top);
        l = l * keep + p;
#pragma unroll
        for (int i = 0; i < D / 32; ++i)
            o[i] = fmaf(p, __bfloat162float(v[32 * i]), o[i] * keep);
        m = top;
    }
    const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
        a.o[t * a.o_tok + hq * a.o_head + lane + 32 * i] = __float2bfloat16_rn(o[i] * inv);
    if (a.lse && lane == 0)
        a.lse[(int64_t)hq * a.q_tokens + t] = l == 0.f ? -INFINITY : m + logf(l);
}

template <int D>
__global__ void __launch_bounds__(kWarps * 32) attn_plain_kernel(const GlintAttnPrompt a)
{
    const int64_t w = (int64_t)blockIdx.x * kWarps + threadIdx.x / 32;
    if (w >= (int64_t)a.q_tokens * a.heads)
        return;
    Span s;
    const int t = (int)(w / a.heads);
    if (span_of(a, t, s))
        plain_row<D>(a, s, t, (int)(w % a.heads), threadIdx.x & 31);
}

int plain_launch(const GlintAttnPrompt &a, cudaStream_t st)
{
    const int64_t warps = (int64_t)a.q_tokens * a.heads;
    if ((warps + kWarps - 1) / kWarps > INT32_MAX)
        return kBadArg;
    const unsigned grid = (unsigned)((warps + kWarps - 1) / kWarps);
    if (a.head_dim == 128)
        attn_plain_kernel<128><<<grid, kWarps * 32, 0, st>>>(a);
    else
        attn_plain_kernel<64><<<grid, kWarps * 32, 0, st>>>(a);
    return cudaGetLastError() == cudaSuccess ? kOk : kLaunch;
}

} // namespace
} // namespace glint

using namespace glint;

extern "C" int glint_attn_prompt_stream(const GlintAttnPrompt *a, cudaStream_t stream)
{
    if (!a || a->seqs < 0 || a->q_tokens < 0 || a->k_tokens < 0 || a->heads < 1 || a->kv_heads < 1 ||
        a->heads % a->kv_heads)
        return kBadArg;
    if (a->head_dim != 64 && a->head_dim != 128)
        return kUnsupported;
    if (a->seqs == 0 || a->q_tokens == 0)
        return kOk;
    if (!a->q || !a->o || !a->cu_q || !a->cu_k || (a->k_tokens > 0 && (!a->k || !a->v)))
        return kBadArg;
    return plain_launch(*a, stream);
}
