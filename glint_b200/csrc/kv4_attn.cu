/* Attention of a sequence's newest tokens over its 4-bit cache.
 *
 * One warp per query row: a lane holds D / 32 neighbouring values of q and of the
 * output, each slot's score is a shuffle sum, and the running maximum and sum of the
 * softmax rescale the output as they change.  Simple and right for every case; the
 * cache is read once per query head.
 */
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "kv4.cuh"

namespace glint {
namespace {

constexpr int kWarps = 4;

struct Args {
    GlintKv4Cache c;
    GlintKv4Attn a;
};

/* lane's D / 32 values of one row */
template <int D>
__device__ __forceinline__ void row_values(const uint8_t *code, const uint16_t *meta, int64_t at, int t, int lane,
                                           float (&x)[D / 32])
{
    const int e = lane * (D / 32);
    const int64_t byte = at * (D / 2) + kv4_unit<D>(e / 64, t) + (e % 64) / 2;
    uint32_t w = D == 128 ? *reinterpret_cast<const uint16_t *>(code + byte) : code[byte];
    const uint32_t m = reinterpret_cast<const uint32_t *>(meta)[at * (D / 64) + e / 64];
    const float step = __uint_as_float(m << 16), lo = __uint_as_float(m & 0xFFFF0000u);
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
        x[i] = fmaf(step, (float)((w >> (4 * i)) & 15u), lo);
}

/* index of slot t's row (head h of sequence b), -1 where its page is outside the cache */
__device__ __forceinline__ int64_t row_of(const Args &g, int b, int h, int t)
{
    const int p = g.a.table[(int64_t)b * g.a.max_pages + t / g.c.page_size];
    if (p < 0 || p >= g.c.pages)
        return -1;
    return ((int64_t)p * g.c.kv_heads + h) * g.c.page_size + t % g.c.page_size;
}

__device__ __forceinline__ int length_of(const Args &g, int b)
{
    return min(max(g.a.lens[b], 0), g.a.max_pages * g.c.page_size);
}

template <int D>
__global__ void __launch_bounds__(kWarps * 32) kv4_attn_kernel(const Args g)
{
    const int lane = threadIdx.x & 31;
    const int64_t wq = (int64_t)blockIdx.x * kWarps + threadIdx.x / 32;
    const int heads = g.a.heads, rows = g.a.rows;
    if (wq >= (int64_t)g.a.seqs * rows * heads)
        return;
    const int b = (int)(wq / (rows * heads)), r = (int)(wq / heads % rows), hq = (int)(wq % heads);
    const int h = hq / (heads / g.c.kv_heads);
    const int seen = length_of(g, b) - rows + r + 1;
    float q[D / 32], o[D / 32] = {}, m = -INFINITY, l = 0.f;
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
        q[i] = __bfloat162float(g.a.q[b * g.a.q_seq + r * g.a.q_row + hq * g.a.q_head + lane * (D / 32) + i]);
    for (int t = 0; t < seen; ++t) {
        const int64_t at = row_of(g, b, h, t);
        if (at < 0)
            continue;
        float x[D / 32], s = 0.f;
        row_values<D>(g.c.k_code, g.c.k_meta, at, t, lane, x);
#pragma unroll
        for (int i = 0; i < D / 32; ++i)
            s = fmaf(q[i], x[i], s);
        s = warp_sum(s) * g.a.scale;
        const float top = fmaxf(m, s);
        const float keep = m == -INFINITY ? 0.f : expf(m - top), p = s == -INFINITY ? 0.f : expf(s - top);
        row_values<D>(g.c.v_code, g.c.v_meta, at, t, lane, x);
        l = l * keep + p;
#pragma unroll
        for (int i = 0; i < D / 32; ++i)
            o[i] = fmaf(p, x[i], o[i] * keep);
        m = top;
    }
    const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
        g.a.o[wq * D + lane * (D / 32) + i] = __float2bfloat16_rn(o[i] * inv);
    const int64_t li = ((int64_t)b * heads + hq) * rows + r;
    float *lse = reinterpret_cast<float *>(g.a.work);
    if (lane == 0) {
        const float v = l == 0.f ? -INFINITY : m + logf(l);
        if (g.a.lse)
            g.a.lse[li] = v;
        if (lse)
            lse[li] = v;
    }
}

/* weight_out: a thread per slot, the rows and heads of its group in order */
template <int D>
__global__ void __launch_bounds__(kWarps * 32) kv4_weight_kernel(const Args g)
{
    const int h = blockIdx.y, b = blockIdx.z, t = blockIdx.x * kWarps * 32 + threadIdx.x;
    const int len = length_of(g, b), group = g.a.heads / g.c.kv_heads;
    if (t >= len)
        return;
    const int64_t at = row_of(g, b, h, t);
    const float *lse = reinterpret_cast<const float *>(g.a.work);
    float sum = 0.f;
    if (at >= 0) {
        for (int j = 0; j < group; ++j) {
            const int hq = h * group + j;
            for (int r = 0; r < g.a.rows; ++r) {
                const float z = lse[((int64_t)b * g.a.heads + hq) * g.a.rows + r];
                if (t >= len - g.a.rows + r + 1 || z == -INFINITY)
                    continue;
                const __nv_bfloat16 *q = g.a.q + b * g.a.q_seq + r * g.a.q_row + hq * g.a.q_head;
                float s = 0.f;
                for (int e = 0; e < D; ++e) {
                    const uint32_t w = g.c.k_code[at * (D / 2) + kv4_unit<D>(e / 64, t) + (e % 64) / 2];
                    const uint32_t m = reinterpret_cast<const uint32_t *>(g.c.k_meta)[at * (D / 64) + e / 64];
                    const float x = fmaf(__uint_as_float(m << 16), (float)((w >> (4 * (e & 1))) & 15u),
                                         __uint_as_float(m & 0xFFFF0000u));
                    s = fmaf(__bfloat162float(q[e]), x, s);
                }
                sum += expf(s * g.a.scale - z);
            }
        }
    }
    const int64_t i = ((int64_t)b * g.c.kv_heads + h) * g.a.weight_stride + t;
    const float old = g.a.weight && t < len - g.a.rows ? g.a.weight[i] : 0.f;
    g.a.weight_out[i] = old + sum;
}

template <int D>
int launch(const Args &g, cudaStream_t st)
{
    const int64_t n = (int64_t)g.a.seqs * g.a.rows * g.a.heads;
    kv4_attn_kernel<D><<<(unsigned)((n + kWarps - 1) / kWarps), kWarps * 32, 0, st>>>(g);
    if (g.a.weight_out) {
        const int cap = g.a.max_pages * g.c.page_size;
        kv4_weight_kernel<D><<<dim3((cap + kWarps * 32 - 1) / (kWarps * 32), g.c.kv_heads, g.a.seqs), kWarps * 32, 0, st>>>(g);
    }
    return cudaGetLastError() == cudaSuccess ? kOk : kLaunch;
}

int check(const GlintKv4Cache *c, const GlintKv4Attn *a)
{
    const int rc = kv4_check(c);
    if (rc != kOk)
        return rc;
    if (!a || a->seqs < 0 || a->rows < 1 || a->heads < 1 || a->heads % c->kv_heads || a->max_pages < 1 ||
        (int64_t)a->heads / c->kv_heads * a->rows > 256 || (int64_t)a->max_pages * c->page_size > INT32_MAX ||
        a->seqs > 65535 || c->kv_heads > 65535)
        return kBadArg;
    return kOk;
}

} // namespace
} // namespace glint

using namespace glint;

extern "C" {

int64_t glint_kv4_attn_work_bytes(const GlintKv4Cache *c, const GlintKv4Attn *a)
{
    const int rc = check(c, a);
    if (rc != kOk)
        return rc;
    return a->weight_out ? (int64_t)a->seqs * a->heads * a->rows * 4 : 0;
}

int glint_kv4_attn_stream(const GlintKv4Cache *c, const GlintKv4Attn *a, cudaStream_t stream)
{
    const int rc = check(c, a);
    if (rc != kOk)
        return rc;
    if (a->seqs == 0)
        return kOk;
    if (!a->q || !a->o || !a->table || !a->lens || (a->weight_out && !a->work) ||
        (a->weight_out && a->weight_stride < (int64_t)a->max_pages * c->page_size))
        return kBadArg;
    Args g{*c, *a};
    if (!a->weight_out)
        g.a.work = nullptr;
    return c->head_dim == 128 ? launch<128>(g, stream) : launch<64>(g, stream);
}

} /* extern "C" */
