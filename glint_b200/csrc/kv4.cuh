/* The 4-bit key/value cache's layout, shared by the kernels that fill, read and
 * shrink it (kv4_cache.cu, rope.cu) and the attention over it (kv4_attn.cu), and the
 * quantisation of a block.
 *
 * Rows of one (page, head) lie one after another, so a page is one contiguous run per
 * head for codes and one for (step, lo).  At head_dim 128 a row is 64 bytes and the
 * halves are swapped in slots with slot & 2: rows t, t + 1, t + 2, t + 3 then put any
 * one 32-byte half in four different quarters of the 32 shared-memory banks, so the
 * attention kernel's fragment loads (four rows, the same 32 columns) meet no conflict. */
#ifndef GLINT_B200_KV4_CUH_
#define GLINT_B200_KV4_CUH_

#include "../../include/glint_attn.h"
#include "common.cuh"
#include "glint_internal.h"

namespace glint {

constexpr int kKv4Block = 64; /* values per (step, lo) */

/* byte offset in a row of the 32-byte unit u of 64 values, for the row of slot t */
template <int D>
__device__ __forceinline__ int kv4_unit(int u, int t)
{
    return D == 128 ? ((u ^ ((t >> 1) & 1)) * 32) : 0;
}

inline bool kv4_supported(const GlintKv4Cache &c)
{
    return (c.head_dim == 64 || c.head_dim == 128) &&
           (c.page_size == 16 || c.page_size == 32 || c.page_size == 64 || c.page_size == 128);
}
inline bool kv4_valid(const GlintKv4Cache &c)
{
    return c.k_code && c.k_meta && c.v_code && c.v_meta && c.pages >= 1 && c.kv_heads >= 1 &&
           aligned_to(c.k_code, 16) && aligned_to(c.v_code, 16) && aligned_to(c.k_meta, 16) &&
           aligned_to(c.v_meta, 16) && (int64_t)c.pages * c.page_size <= INT32_MAX;
}
/* kOk, or the code an entry point returns for this cache */
inline int kv4_check(const GlintKv4Cache *c)
{
    if (!c)
        return kBadArg;
    if (!kv4_supported(*c))
        return kUnsupported;
    return kv4_valid(*c) ? kOk : kBadArg;
}

inline int log2_of(int n)
{
    int l = 0;
    while ((1 << l) < n)
        ++l;
    return l;
}

/* ---- quantisation, for the kernels that fill the cache (kv4_cache.cu, rope.cu) */

/* 16 values of a row as BF16 pairs; ALIGNED: two 16-byte loads */
template <bool ALIGNED>
__device__ __forceinline__ void load16(const __nv_bfloat16 *p, uint32_t (&x)[8])
{
    if constexpr (ALIGNED) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint4 w = __ldg(reinterpret_cast<const uint4 *>(p) + i);
            x[4 * i] = w.x, x[4 * i + 1] = w.y, x[4 * i + 2] = w.z, x[4 * i + 3] = w.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            x[i] = (uint32_t)__bfloat16_as_ushort(p[2 * i]) | ((uint32_t)__bfloat16_as_ushort(p[2 * i + 1]) << 16);
    }
}
__device__ __forceinline__ uint32_t min2(uint32_t a, uint32_t b)
{
    asm("min.bf16x2 %0, %0, %1;" : "+r"(a) : "r"(b));
    return a;
}
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b)
{
    asm("max.bf16x2 %0, %0, %1;" : "+r"(a) : "r"(b));
    return a;
}
__device__ __forceinline__ uint64_t pack2f(float lo, float hi)
{
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void unpack2f(uint64_t v, float &lo, float &hi)
{
    asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b)
{
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c)
{
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b)
{
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float low_half(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float high_half(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }

/* One block's 16 values of this lane -> 16 nibbles; (step, lo) of the block the same in
 * all 4 lanes of the aligned group. */
__device__ __forceinline__ uint2 quantise16(const uint32_t (&x)[8], uint32_t &meta)
{
    uint32_t mn = x[0], mx = x[0], odd = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        mn = min2(mn, x[i]), mx = max2(mx, x[i]);
        odd |= (x[i] & 0x7F807F80u) + 0x00800080u; /* NaN, infinity: an exponent of ones carries into bit 15 or 31 */
    }
#pragma unroll
    for (int off = 2; off > 0; off >>= 1) {
        mn = min2(mn, __shfl_xor_sync(0xFFFFFFFFu, mn, off));
        mx = max2(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, off));
    }
    const bool any = (__ballot_sync(0xFFFFFFFFu, (odd & 0x80008000u) != 0) >> (lane_id() & 28u) & 15u) != 0;
    const float lo = fminf(low_half(mn), high_half(mn)), hi = fmaxf(low_half(mx), high_half(mx));
    /* Quotients as f32 division gives them, from the correctly rounded reciprocal y of the
     * divisor s: q = n y, then q + (n - q s) y (P. Markstein, IBM J. Res. Dev. 34(1), 1990);
     * exact where y, s and n are normal numbers with room to spare. */
    const float range = hi - lo;
    float fifteenth;
    if (range > 1e-28f && range < 1e30f) {
        const float y = 1.f / 15.f, q = range * y;
        fifteenth = fmaf(fmaf(-q, 15.f, range), y, q);
    } else {
        fifteenth = __fdiv_rn(range, 15.f);
    }
    const __nv_bfloat16 sb = __float2bfloat16_rn(fifteenth);
    const float step = __bfloat162float(sb);
    if (any || step - step != 0.f) { /* not finite: the block reads as NaN */
        meta = 0x7FC00000u;
        return make_uint2(0u, 0u);
    }
    /* lo is one of the BF16 inputs, so its upper half is all of it */
    meta = (__float_as_uint(lo) & 0xFFFF0000u) | (uint32_t)__bfloat16_as_ushort(sb);
    /* (x - lo) / step, at most 15.06, plus 1.5 * 2^23 is rounded to an integer, ties to even:
     * no clamp.  Four codes at a time are added up as c0 + 16 c1 + 256 c2 + 4096 c3, exact in
     * f32; plus 2^23 they stand in the low bits. */
    float c[16];
    if (step > 1e-30f && step < 1e30f) {
        const float y = __frcp_rn(step);
        const uint64_t y2 = pack2f(y, y), lo2 = pack2f(-lo, -lo), less = pack2f(-step, -step);
        const uint64_t magic = pack2f(12582912.f, 12582912.f), minus = pack2f(-12582912.f, -12582912.f);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint64_t d = add2(pack2f(low_half(x[i]), high_half(x[i])), lo2), q = mul2(d, y2);
            unpack2f(add2(add2(fma2(fma2(q, less, d), y2, q), magic), minus), c[2 * i], c[2 * i + 1]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float v = i & 1 ? high_half(x[i / 2]) : low_half(x[i / 2]);
            c[i] = step > 0.f ? fminf(fmaxf(rintf(__fdiv_rn(v - lo, step)), 0.f), 15.f) : 0.f;
        }
    }
    uint32_t four[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        four[i] = __float_as_uint(fmaf(4096.f, c[4 * i + 3], fmaf(256.f, c[4 * i + 2], fmaf(16.f, c[4 * i + 1], c[4 * i]))) +
                                  8388608.f);
    return make_uint2(__byte_perm(four[0], four[1], 0x5410), __byte_perm(four[2], four[3], 0x5410));
}

} // namespace glint

#endif
