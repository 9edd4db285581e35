/* Rotary positions of query and key heads, with or without a norm of each head before them,
 * and the same with keys and values written to the 4-bit cache in the pass.
 *
 * A head x of D values, a = position * inv_freq[i], c = scale cos a, s = scale sin a:
 *
 *   y = x, or (x r) w with r = 1 / sqrt(mean(x^2) + eps)
 *   (o1, o2) = (y1 c - y2 s, y2 c + y1 s)   on the pairs (i, i + R / 2) or (2i, 2i + 1)
 *
 * A warp takes a token, or a part of its heads where tokens are few: 16 values a lane, so
 * 4 (D = 128) or 8 heads at a time, the next ones' loads under way.  Its angles are the
 * same for every head, so each is computed once, in 64 bits (a far position times a frequency
 * is hundreds of thousands of radians, of which f32 would keep two digits), and stays in
 * registers as (c, +-s) of the lane's 16 places.  A value's partner is in the same lane
 * (2i, 2i + 1), comes by shuffles (R / 2 a multiple of 16) or through shared memory.
 *
 * The mean is summed in 64 bits and products and sums are rounded one by one, as they stand
 * above: the result depends on no order, and what is then rounded to BF16 and to 4 bits is
 * the same whichever of the entry points computes it.
 */
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "kv4.cuh"

namespace glint {
namespace {

constexpr int kWarps = 8;

struct Args {
    GlintRope a;
    GlintKv4Cache c;
    const __nv_bfloat16 *v;
    const int *slots;
    int64_t v_tok, v_head;
    int page_log2;
    int rows;           /* heads of a token: q, k and, with the cache, v */
    int chunk, chunks;  /* of them a warp takes; such parts a token */
    int64_t warps;      /* tokens * chunks */
};

/* 16 values as BF16 pairs, by loads that may follow a store to the same place */
template <bool VEC>
__device__ __forceinline__ void get16(const __nv_bfloat16 *p, uint32_t (&x)[8])
{
    if constexpr (VEC) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint4 w = reinterpret_cast<const uint4 *>(p)[i];
            x[4 * i] = w.x, x[4 * i + 1] = w.y, x[4 * i + 2] = w.z, x[4 * i + 3] = w.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            x[i] = (uint32_t)__bfloat16_as_ushort(p[2 * i]) | ((uint32_t)__bfloat16_as_ushort(p[2 * i + 1]) << 16);
    }
}
template <bool VEC>
__device__ __forceinline__ void put16(__nv_bfloat16 *p, const uint32_t (&x)[8])
{
    if constexpr (VEC) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
            reinterpret_cast<uint4 *>(p)[i] = make_uint4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            p[2 * i] = __ushort_as_bfloat16((unsigned short)(x[i] & 0xFFFFu));
            p[2 * i + 1] = __ushort_as_bfloat16((unsigned short)(x[i] >> 16));
        }
    }
}

template <int D, bool VEC, bool APPEND>
__global__ void __launch_bounds__(kWarps * 32) rope_kernel(const Args g)
{
    constexpr int L = D / 16, N = 32 / L; /* lanes a head, heads a step */
    __shared__ float2 turns[kWarps][D / 2];
    __shared__ float4 mixed[kWarps][N * D / 4];
    const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
    const int64_t w = (int64_t)blockIdx.x * kWarps + warp;
    if (w >= g.warps)
        return; /* no barrier of the block follows */
    const GlintRope &a = g.a;
    const int t = (int)(w / g.chunks), r0 = (int)(w - (int64_t)t * g.chunks) * g.chunk, r1 = min(g.rows, r0 + g.chunk);
    const int e0 = lane % L * 16; /* the lane's first place in its head */
    const int keys = a.heads, values = a.heads + a.kv_heads;

    auto load = [&](int r, uint32_t (&x)[8]) {
        r += lane / L;
        const __nv_bfloat16 *p = r < keys ? a.q + t * a.q_tok + r * a.q_head
                                 : !APPEND || r < values ? a.k + t * a.k_tok + (r - keys) * a.k_head
                                                         : g.v + t * g.v_tok + (r - values) * g.v_head;
        if (r < r1) {
            get16<VEC>(p + e0, x);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                x[i] = 0u;
        }
    };
    uint32_t x[8];
    load(r0, x);

    const double pos = (double)a.positions[t];
    for (int i = lane; i < a.half; i += 32) {
        double s, c;
        sincos(pos * (double)a.inv_freq[i], &s, &c);
        turns[warp][i] = make_float2((float)(c * a.scale), (float)(s * a.scale));
    }
    __syncwarp();
    /* o = y c + partner s; behind the rotated part c = 1, the partner 0 and s = -0: -0 is what
     * may be added to any y */
    uint64_t c2[8], s2[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        float c[2], s[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int e = e0 + 2 * i + j;
            const bool second = a.interleaved ? j : e >= a.half;
            const float2 v = turns[warp][e < 2 * a.half ? (a.interleaved ? e / 2 : second ? e - a.half : e) : 0];
            c[j] = e < 2 * a.half ? v.x : 1.f;
            s[j] = e < 2 * a.half ? (second ? v.y : -v.y) : -0.f;
        }
        c2[i] = pack2f(c[0], c[1]), s2[i] = pack2f(s[0], s[1]);
    }
    const bool shuffled = a.half % 16 == 0;
    const int away = a.half / 16, from = e0 < a.half ? lane + away : e0 < 2 * a.half ? lane - away : lane;

    /* 16 values of a head, normed with its weights (NULL: not) and rotated, as BF16 pairs */
    auto turned = [&](const uint32_t (&x)[8], const float *weight, uint32_t (&o)[8]) {
        uint64_t y[8], p[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
            y[i] = pack2f(low_half(x[i]), high_half(x[i]));
        if (a.q_norm || a.k_norm) {
            double sum = 0.;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const double u = (double)low_half(x[i]), v = (double)high_half(x[i]);
                sum = fma(u, u, sum), sum = fma(v, v, sum);
            }
#pragma unroll
            for (int off = 1; off < L; off *= 2)
                sum += __shfl_xor_sync(0xFFFFFFFFu, sum, off);
            const float r = (float)(1. / sqrt(sum * (1. / D) + a.eps));
            if (weight) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float4 w4 = reinterpret_cast<const float4 *>(weight + e0)[i];
                    y[2 * i] = mul2(mul2(y[2 * i], pack2f(r, r)), pack2f(w4.x, w4.y));
                    y[2 * i + 1] = mul2(mul2(y[2 * i + 1], pack2f(r, r)), pack2f(w4.z, w4.w));
                }
            }
        }
        if (a.interleaved) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float u, v;
                unpack2f(y[i], u, v);
                p[i] = pack2f(v, u);
            }
        } else if (shuffled) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                p[i] = __shfl_sync(0xFFFFFFFFu, y[i], from);
        } else {
            float4 *mine = mixed[warp] + (lane * 16) / 4;
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float4 v;
                unpack2f(y[2 * i], v.x, v.y), unpack2f(y[2 * i + 1], v.z, v.w);
                mine[i] = v;
            }
            __syncwarp();
            const float *head = reinterpret_cast<const float *>(mixed[warp]) + lane / L * D;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int e = e0 + 2 * i;
                const int f = e < a.half ? e + a.half : e < 2 * a.half ? e - a.half : e;
                const int f1 = e + 1 < a.half ? e + 1 + a.half : e + 1 < 2 * a.half ? e + 1 - a.half : e + 1;
                p[i] = pack2f(head[f], head[f1]);
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float u, v, pu, pv;
            unpack2f(p[i], pu, pv);
            if (e0 + 2 * i >= 2 * a.half) /* nothing that is not finite comes by here */
                pu = pv = 0.f;
            /* three roundings, as they stand in the definition: no fma */
            unpack2f(add2(mul2(y[i], c2[i]), mul2(pack2f(pu, pv), s2[i])), u, v);
            const __nv_bfloat162 b = __floats2bfloat162_rn(u, v);
            o[i] = *reinterpret_cast<const uint32_t *>(&b);
        }
    };

    const int slot = APPEND ? g.slots[t] : -1;
    for (int r = r0; r < r1; r += N) {
        uint32_t next[8], o[8];
        load(r + N, next); /* zeros past the last */
        const int row = r + lane / L;
        const bool key = row >= keys && row < values;
        if (!APPEND || r < values) {
            turned(x, row < keys ? a.q_norm : key ? a.k_norm : nullptr, o);
            if (row < r1) {
                if (row < keys)
                    put16<VEC>(a.q_out + t * a.qo_tok + row * a.qo_head + e0, o);
                else if (key && (!APPEND || a.k_out))
                    put16<VEC>(a.k_out + t * a.ko_tok + (row - keys) * a.ko_head + e0, o);
            }
        }
        if constexpr (APPEND) {
            if (r + N > keys) { /* the whole warp */
                if (row >= values) {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        o[i] = x[i];
                }
                uint32_t meta;
                const uint2 code = quantise16(o, meta);
                if (row >= keys && row < r1 && slot >= 0 && slot < g.c.pages * g.c.page_size) {
                    const int page = slot >> g.page_log2, at = slot & (g.c.page_size - 1);
                    const int h = key ? row - keys : row - values;
                    const int64_t place = (((int64_t)page * g.c.kv_heads + h) << g.page_log2) + at;
                    uint8_t *codes = key ? g.c.k_code : g.c.v_code;
                    uint16_t *metas = key ? g.c.k_meta : g.c.v_meta;
                    *reinterpret_cast<uint2 *>(codes + place * (D / 2) + kv4_unit<D>(e0 / 64, at) + e0 % 64 / 2) = code;
                    if (e0 % 64 == 0)
                        reinterpret_cast<uint32_t *>(metas)[place * (D / 64) + e0 / 64] = meta;
                }
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
            x[i] = next[i];
    }
}

int launch(Args &g, bool append, bool vec, cudaStream_t st)
{
    const GlintRope &a = g.a;
    const int n = 32 / (a.head_dim / 16); /* heads a step */
    g.rows = a.heads + a.kv_heads + (append ? a.kv_heads : 0);
    /* as many parts of a token as give every SM two warps of each scheduler, while there is a step for each */
    const int steps = (g.rows + n - 1) / n;
    const int64_t want = (8LL * sm_count() + a.tokens - 1) / a.tokens;
    g.chunk = (int)((steps + std::min<int64_t>(want, steps) - 1) / std::min<int64_t>(want, steps)) * n;
    g.chunks = (g.rows + g.chunk - 1) / g.chunk;
    g.warps = (int64_t)a.tokens * g.chunks;
    const int64_t grid = (g.warps + kWarps - 1) / kWarps;
    if (grid > INT32_MAX)
        return kBadArg;
    const auto kernel = [&](auto d) {
        constexpr int D = decltype(d)::value;
        return append ? (vec ? rope_kernel<D, true, true> : rope_kernel<D, false, true>)
                      : (vec ? rope_kernel<D, true, false> : rope_kernel<D, false, false>);
    };
    const auto k = a.head_dim == 128 ? kernel(std::integral_constant<int, 128>()) : kernel(std::integral_constant<int, 64>());
    k<<<(unsigned)grid, kWarps * 32, 0, st>>>(g);
    return cudaGetLastError() == cudaSuccess ? kOk : kLaunch;
}

/* kOk, or what an entry point returns for these arguments; keys: k_out must be there */
int check(const GlintRope *a, bool keys)
{
    if (!a)
        return kBadArg;
    if (a->head_dim != 64 && a->head_dim != 128)
        return kUnsupported;
    if (a->tokens < 0 || a->heads < 1 || a->kv_heads < 0 || a->half < 0 || a->half > a->head_dim / 2 || !(a->eps > 0.) ||
        (int64_t)a->heads + 2 * (int64_t)a->kv_heads > INT32_MAX / 4)
        return kBadArg;
    if (a->tokens == 0)
        return kOk;
    if (!a->q || !a->q_out || !a->positions || (a->half && !a->inv_freq) || (a->kv_heads && (!a->k || (keys && !a->k_out))) ||
        !aligned_to(a->q_norm, 16) || !aligned_to(a->k_norm, 16))
        return kBadArg;
    return kOk;
}
bool vectors(const GlintRope &a)
{
    return aligned_to(a.q, 16) && aligned_to(a.k, 16) && aligned_to(a.q_out, 16) && aligned_to(a.k_out, 16) &&
           (a.q_tok | a.q_head | a.k_tok | a.k_head | a.qo_tok | a.qo_head | a.ko_tok | a.ko_head) % 8 == 0;
}

} // namespace
} // namespace glint

using namespace glint;

int glint_rope_stream(const GlintRope *a, cudaStream_t stream)
{
    const int rc = check(a, true);
    if (rc != kOk || a->tokens == 0)
        return rc;
    Args g{};
    g.a = *a;
    return launch(g, false, vectors(*a), stream);
}

int glint_kv4_rope_append_stream(const GlintKv4Cache *c, const GlintRope *a, const glint_bf16_t *v, int64_t v_tok,
                                 int64_t v_head, const int *slots, cudaStream_t stream)
{
    int rc = kv4_check(c);
    if (rc == kOk)
        rc = check(a, false);
    if (rc != kOk)
        return rc;
    if (a->kv_heads != c->kv_heads || a->head_dim != c->head_dim)
        return kBadArg;
    if (a->tokens == 0)
        return kOk;
    if (!v || !slots)
        return kBadArg;
    Args g{};
    g.a = *a, g.c = *c, g.v = v, g.slots = slots, g.v_tok = v_tok, g.v_head = v_head;
    g.page_log2 = log2_of(c->page_size);
    return launch(g, true, vectors(*a) && aligned_to(v, 16) && (v_tok | v_head) % 8 == 0, stream);
}
