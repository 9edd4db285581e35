/* Rotary positions of query and key heads, with or without a norm of each head before them,
 * and the same with keys and values written to the 4-bit cache in the pass.
 *
 * A head x of D values, a = position * inv_freq[i], c = scale cos a, s = scale sin a:
 *
 *   y = x, or (x r) w with r = 1 / sqrt(mean(x^2) + eps)
 *   (o1, o2) = (y1 c - y2 s, y2 c + y1 s)   on the pairs (i, i + R / 2) or (2i, 2i + 1)
 *
 * A warp takes a token, or a part of its heads where tokens are few: 16 values a lane, so
 * 4 (D = 128) or 8 heads a step, the next step's loads under way.  Its angles are the
 * same for every head, so each is computed once, in 64 bits (a far position times a frequency
 * is hundreds of thousands of radians, of which f32 would keep two digits), and (c, s) of the
 * lane's 8 pairs stay in registers.  A lane's 16 values are two runs of 8 that are partners of
 * one another (i, i + R / 2; R / 2 a multiple of 8) or 16 neighbours (2i, 2i + 1), so no value
 * leaves its lane; other R exchange through shared memory.
 *
 * The mean is summed in 64 bits and products and sums are rounded one by one, as they stand
 * above: the result depends on no order, and what is then rounded to BF16 and to 4 bits is
 * the same whichever of the entry points computes it.
 *
 * Bytes bound it: q and k read and written once, v read, codes written.  32768 tokens, 32 / 8 heads of 128,
 * norms: 124 us, 5.4 TB/s where a copy reaches 6.4 (its floor 105); 16383 tokens into the cache 89 us of 61, the
 * quantisation's shuffles and conversions in the way; few tokens are launch and latency: 1 token 2.6 us, 513
 * 4.7, 7 into the cache 3.6.  Partners that are no runs of 8, through shared memory: 32768 tokens (no norms, 122 us with
 * runs) 261 us; operands at odd addresses, value by value, 302, both 638, side by side 940.  CTAs of 4 warps, 6 an SM (5 with the cache): of 8 warps 127 to 150 us for the 124, more
 * CTAs with fewer registers 154.
 */
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "kv4.cuh"

namespace glint {
namespace {

constexpr int kWarps = 4;
constexpr double kLeastEps = 0x1p-250; /* r of a head of zeros is a number in f32 */
/* where a value's partner is: R / 2 places on, in whole runs of 8 or not; beside it */
enum Pairing : int { kRuns, kAny, kBeside };

struct Args {
    GlintRope a;
    GlintKv4Cache c;
    const __nv_bfloat16 *v;
    const int *slots;
    int64_t v_tok, v_head;
    int page_log2;
    int q_steps, k_steps;     /* of a token's heads; v, with the cache, takes as many as k */
    int steps, chunk, chunks; /* in all; of them a warp takes; such parts a token */
    int64_t warps;            /* tokens * chunks */
    uint64_t none;            /* -0 twice, see product2() */
};

/* 8 values as BF16 pairs, by loads that may follow a store to the same place */
template <bool VEC>
__device__ __forceinline__ void get8(const __nv_bfloat16 *p, uint32_t *x)
{
    if constexpr (VEC) {
        const uint4 w = *reinterpret_cast<const uint4 *>(p);
        x[0] = w.x, x[1] = w.y, x[2] = w.z, x[3] = w.w;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            x[i] = (uint32_t)__bfloat16_as_ushort(p[2 * i]) | ((uint32_t)__bfloat16_as_ushort(p[2 * i + 1]) << 16);
    }
}
template <bool VEC>
__device__ __forceinline__ void put8(__nv_bfloat16 *p, const uint32_t *x)
{
    if constexpr (VEC) {
        *reinterpret_cast<uint4 *>(p) = make_uint4(x[0], x[1], x[2], x[3]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            p[2 * i] = __ushort_as_bfloat16((unsigned short)(x[i] & 0xFFFFu));
            p[2 * i + 1] = __ushort_as_bfloat16((unsigned short)(x[i] >> 16));
        }
    }
}
__device__ __forceinline__ uint64_t sub2(uint64_t a, uint64_t b)
{
    uint64_t r;
    asm("sub.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
/* a b, rounded, that no sum behind it takes into an fma (of mul.rn.f32x2 the assembler makes one): none is -0
 * twice, from the host, so that no compiler knows it */
__device__ __forceinline__ uint64_t product2(uint64_t a, uint64_t b, uint64_t none) { return fma2(a, b, none); }
__device__ __forceinline__ uint32_t round2(float lo, float hi)
{
    const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&b);
}
__device__ __forceinline__ uint32_t round2(uint64_t v)
{
    float lo, hi;
    unpack2f(v, lo, hi);
    return round2(lo, hi);
}

template <int D, Pairing P, bool VEC, bool APPEND>
__global__ void __launch_bounds__(kWarps * 32, APPEND ? 5 : 6) rope_kernel(const Args g)
{
    constexpr int L = D / 16, N = 32 / L; /* lanes a head, heads a step */
    constexpr bool kMoves = APPEND && P == kRuns; /* values go to the lanes that quantise them */
    __shared__ float2 turns[kWarps][D / 2];
    /* a step's heads, f32 values for partners to read or BF16 ones; 16 bytes keep rows off one another's banks */
    constexpr int kRow = (P == kAny ? 4 : 2) * D + 16;
    __shared__ __align__(16) uint8_t mixed[P == kAny || kMoves ? kWarps : 1][N * kRow];
    const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
    const int64_t w = (int64_t)blockIdx.x * kWarps + warp;
    if (w >= g.warps)
        return; /* no barrier of the block follows */
    const GlintRope &a = g.a;
    const int t = (int)(w / g.chunks), s0 = (int)(w - (int64_t)t * g.chunks) * g.chunk, s1 = min(g.steps, s0 + g.chunk);
    const int l = lane % L, in = lane / L, half = a.half;
    /* the lane's runs of 8 values: partners while there are any (then the lane turns them), else neighbours */
    const bool partners = P == kRuns && l < half / 8;
    const int ea = P != kRuns ? 16 * l : partners ? 8 * l : 2 * half + 16 * (l - half / 8);
    const int eb = partners ? ea + half : ea + 8;

    const int k0 = g.q_steps, v0 = g.q_steps + g.k_steps; /* first steps of k and v */
    /* a step's heads: this lane's one of them, which lies `by` behind that of the step before of the same kind */
    struct Heads {
        const __nv_bfloat16 *p;
        int64_t by;
        int left; /* heads of its kind from this lane's on; none: <= 0 */
    };
    auto heads_at = [&](int s) {
        const int row = (s - (s < k0 ? 0 : !APPEND || s < v0 ? k0 : v0)) * N + in;
        if (s < k0)
            return Heads{a.q + t * a.q_tok + row * a.q_head, N * a.q_head, a.heads - row};
        if (!APPEND || s < v0)
            return Heads{a.k + t * a.k_tok + row * a.k_head, N * a.k_head, a.kv_heads - row};
        return Heads{g.v + t * g.v_tok + row * g.v_head, N * g.v_head, a.kv_heads - row};
    };
    Heads from = heads_at(s0);
    auto load = [&](int s, uint32_t (&x)[8]) { /* of `from`, the heads of step s, which moves on */
        if (from.left > 0 && s < s1) {
            const bool value = APPEND && s >= v0;
            get8<VEC>(from.p + (value ? 16 * l : ea), x);
            get8<VEC>(from.p + (value ? 16 * l + 8 : eb), x + 4);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                x[i] = 0u;
        }
        from.p += from.by, from.left -= N;
        if (s + 1 == k0 || (APPEND && s + 1 == v0))
            from = heads_at(s + 1);
    };
    uint32_t x[8];
    load(s0, x);

    if (s0 < v0) {
        const double pos = (double)a.positions[t];
        for (int i = lane; i < half; i += 32) {
            double s, c;
            sincos(pos * (double)a.inv_freq[i], &s, &c);
            turns[warp][i] = make_float2((float)(c * a.scale), (float)(s * a.scale));
        }
        __syncwarp();
    }
    uint64_t c2[4], s2[4]; /* of pairs 8 l .. 8 l + 7 */
    if constexpr (P != kAny) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int f = 8 * l + 2 * i;
            const float2 e = turns[warp][f < half ? f : 0], o = turns[warp][f + 1 < half ? f + 1 : 0];
            c2[i] = pack2f(e.x, o.x), s2[i] = pack2f(e.y, o.y);
        }
    }

    const uint64_t none = g.none;
    /* the lane's values of a head, normed with its weights (NULL: not) and turned, as BF16 pairs */
    auto turned = [&](const uint32_t (&x)[8], const float *weight, uint32_t (&o)[8]) {
        /* first and second values of pairs 2 i, 2 i + 1 */
        uint64_t y1[4], y2[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (P == kBeside) {
                y1[i] = pack2f(low_half(x[2 * i]), low_half(x[2 * i + 1]));
                y2[i] = pack2f(high_half(x[2 * i]), high_half(x[2 * i + 1]));
            } else {
                y1[i] = pack2f(low_half(x[i]), high_half(x[i]));
                y2[i] = pack2f(low_half(x[4 + i]), high_half(x[4 + i]));
            }
        }
        if (weight) {
            double sum = 0.;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const double u = (double)low_half(x[i]), v = (double)high_half(x[i]);
                sum = fma(u, u, sum), sum = fma(v, v, sum);
            }
#pragma unroll
            for (int off = 1; off < L; off *= 2)
                sum += __shfl_xor_sync(0xFFFFFFFFu, sum, off);
            const float r = (float)rsqrt(sum * (1. / D) + a.eps);
            const uint64_t r2 = pack2f(r, r);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float4 u = __ldg(reinterpret_cast<const float4 *>(weight + ea) + i);
                const float4 v = __ldg(reinterpret_cast<const float4 *>(weight + eb) + i);
                if constexpr (P == kBeside) { /* u is pairs 2 i, 2 i + 1 of the first run, v of the second */
                    y1[i] = mul2(mul2(y1[i], r2), pack2f(u.x, u.z)), y2[i] = mul2(mul2(y2[i], r2), pack2f(u.y, u.w));
                    y1[2 + i] = mul2(mul2(y1[2 + i], r2), pack2f(v.x, v.z));
                    y2[2 + i] = mul2(mul2(y2[2 + i], r2), pack2f(v.y, v.w));
                } else {
                    y1[2 * i] = mul2(mul2(y1[2 * i], r2), pack2f(u.x, u.y));
                    y1[2 * i + 1] = mul2(mul2(y1[2 * i + 1], r2), pack2f(u.z, u.w));
                    y2[2 * i] = mul2(mul2(y2[2 * i], r2), pack2f(v.x, v.y));
                    y2[2 * i + 1] = mul2(mul2(y2[2 * i + 1], r2), pack2f(v.z, v.w));
                }
            }
        }
        if constexpr (P == kAny) { /* 16 neighbours a lane, whose partners may be anywhere */
            float *head = reinterpret_cast<float *>(mixed[warp] + in * kRow);
            float y[16];
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 4; ++i)
                unpack2f(y1[i], y[2 * i], y[2 * i + 1]), unpack2f(y2[i], y[8 + 2 * i], y[9 + 2 * i]);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                reinterpret_cast<float4 *>(head + ea)[i] = make_float4(y[4 * i], y[4 * i + 1], y[4 * i + 2], y[4 * i + 3]);
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int e = ea + i;
                if (e < 2 * half) {
                    const float2 cs = turns[warp][e < half ? e : e - half];
                    /* roundings one by one, as everywhere here: no fma */
                    y[i] = e < half ? __fsub_rn(__fmul_rn(y[i], cs.x), __fmul_rn(head[e + half], cs.y))
                                    : __fadd_rn(__fmul_rn(y[i], cs.x), __fmul_rn(head[e - half], cs.y));
                }
            }
#pragma unroll
            for (int i = 0; i < 8; ++i)
                o[i] = round2(y[2 * i], y[2 * i + 1]);
        } else {
            uint64_t o1[4], o2[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                o1[i] = sub2(product2(y1[i], c2[i], none), product2(y2[i], s2[i], none));
                o2[i] = add2(product2(y2[i], c2[i], none), product2(y1[i], s2[i], none));
            }
            if (half != D / 2) { /* places behind the rotated ones stay, whatever their values */
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const bool first = P == kRuns ? partners : 8 * l + 2 * i < half;
                    const bool second = P == kRuns ? partners : 8 * l + 2 * i + 1 < half;
                    float f[2], y[2];
                    unpack2f(o1[i], f[0], f[1]), unpack2f(y1[i], y[0], y[1]);
                    o1[i] = pack2f(first ? f[0] : y[0], second ? f[1] : y[1]);
                    unpack2f(o2[i], f[0], f[1]), unpack2f(y2[i], y[0], y[1]);
                    o2[i] = pack2f(first ? f[0] : y[0], second ? f[1] : y[1]);
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (P == kBeside) {
                    float a0, a1, b0, b1;
                    unpack2f(o1[i], a0, a1), unpack2f(o2[i], b0, b1);
                    o[2 * i] = round2(a0, b0), o[2 * i + 1] = round2(a1, b1);
                } else {
                    o[i] = round2(o1[i]), o[4 + i] = round2(o2[i]);
                }
            }
        }
    };

    const int slot = APPEND && s1 > k0 ? g.slots[t] : -1;
    const bool cached = APPEND && slot >= 0 && slot < g.c.pages * g.c.page_size;
    __nv_bfloat16 *out = nullptr; /* where this step's heads go */
    int64_t by = 0;
    int row = 0; /* this lane's head of its kind */
    for (int s = s0; s < s1; ++s) {
        uint32_t next[8], o[8];
        load(s + 1, next);
        const bool query = s < k0, value = APPEND && s >= v0;
        if (s == s0 || s == k0 || (APPEND && s == v0)) {
            row = (s - (query ? 0 : value ? v0 : k0)) * N + in;
            by = N * (query ? a.qo_head : a.ko_head);
            out = query ? a.q_out + t * a.qo_tok + row * a.qo_head : a.k_out + t * a.ko_tok + row * a.ko_head;
        }
        const bool live = row < (query ? a.heads : a.kv_heads);
        if (value) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                o[i] = x[i];
        } else {
            turned(x, query ? a.q_norm : a.k_norm, o);
            if (live && (query || !APPEND || a.k_out)) {
                put8<VEC>(out + ea, o);
                put8<VEC>(out + eb, o + 4);
            }
            out += by;
        }
        if (APPEND && !query) {
            if constexpr (kMoves) {
                if (!value) { /* 16 neighbours a lane */
                    uint8_t *head = mixed[warp] + in * kRow;
                    __syncwarp();
                    *reinterpret_cast<uint4 *>(head + 2 * ea) = make_uint4(o[0], o[1], o[2], o[3]);
                    *reinterpret_cast<uint4 *>(head + 2 * eb) = make_uint4(o[4], o[5], o[6], o[7]);
                    __syncwarp();
                    const uint4 u = *reinterpret_cast<const uint4 *>(head + 32 * l);
                    const uint4 v = *reinterpret_cast<const uint4 *>(head + 32 * l + 16);
                    o[0] = u.x, o[1] = u.y, o[2] = u.z, o[3] = u.w, o[4] = v.x, o[5] = v.y, o[6] = v.z, o[7] = v.w;
                }
            }
            uint32_t meta;
            const uint2 code = quantise16(o, meta);
            if (live && cached) {
                const int page = slot >> g.page_log2, at = slot & (g.c.page_size - 1), e0 = 16 * l;
                const int64_t place = (((int64_t)page * g.c.kv_heads + row) << g.page_log2) + at;
                uint8_t *codes = value ? g.c.v_code : g.c.k_code;
                uint16_t *metas = value ? g.c.v_meta : g.c.k_meta;
                *reinterpret_cast<uint2 *>(codes + place * (D / 2) + kv4_unit<D>(e0 / 64, at) + e0 % 64 / 2) = code;
                if (e0 % 64 == 0)
                    reinterpret_cast<uint32_t *>(metas)[place * (D / 64) + e0 / 64] = meta;
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
            x[i] = next[i];
        row += N;
    }
}

template <int D, Pairing P>
auto kernel_of(bool append, bool vec)
{
    return append ? (vec ? rope_kernel<D, P, true, true> : rope_kernel<D, P, false, true>)
                  : (vec ? rope_kernel<D, P, true, false> : rope_kernel<D, P, false, false>);
}
template <int D>
auto kernel_of(const GlintRope &a, bool append, bool vec)
{
    return a.interleaved       ? kernel_of<D, kBeside>(append, vec)
           : a.half % 8 == 0 ? kernel_of<D, kRuns>(append, vec)
                               : kernel_of<D, kAny>(append, vec);
}

int launch(Args &g, bool append, bool vec, cudaStream_t st)
{
    const GlintRope &a = g.a;
    const int n = 32 / (a.head_dim / 16); /* heads a step */
    g.q_steps = (a.heads + n - 1) / n, g.k_steps = (a.kv_heads + n - 1) / n;
    g.steps = g.q_steps + (append ? 2 : 1) * g.k_steps;
    /* as many parts of a token as give every SM eight warps, while there is a step for each */
    const int64_t want = std::min<int64_t>((8LL * sm_count() + a.tokens - 1) / a.tokens, g.steps);
    g.chunk = (int)((g.steps + want - 1) / want);
    g.chunks = (g.steps + g.chunk - 1) / g.chunk;
    g.warps = (int64_t)a.tokens * g.chunks;
    g.none = 0x8000000080000000u;
    const int64_t grid = (g.warps + kWarps - 1) / kWarps;
    if (grid > INT32_MAX)
        return kBadArg;
    const auto kernel = a.head_dim == 128 ? kernel_of<128>(a, append, vec) : kernel_of<64>(a, append, vec);
    kernel<<<(unsigned)grid, kWarps * 32, 0, st>>>(g);
    return cudaGetLastError() == cudaSuccess ? kOk : kLaunch;
}

/* kOk, or what an entry point returns for these arguments; keys: k_out must be there */
int check(const GlintRope *a, bool keys)
{
    if (!a)
        return kBadArg;
    if (a->head_dim != 64 && a->head_dim != 128)
        return kUnsupported;
    if (a->tokens < 0 || a->heads < 1 || a->kv_heads < 0 || a->half < 0 || a->half > a->head_dim / 2 ||
        !(a->eps >= kLeastEps) ||
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
