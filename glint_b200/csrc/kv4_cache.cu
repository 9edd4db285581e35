/* The 4-bit key/value cache: append (quantise rows into their slots), read (slots back
 * to BF16) and eviction by accumulated attention weight.
 *
 * Append and read move each byte once.  Append: a thread takes 16 neighbouring values of a
 * row (32 bytes of BF16, 8 bytes of codes), the 4 threads of a 64-value block find its
 * minimum and maximum with two shuffles, and K and V go through one thread so that four
 * loads are in flight.  Read: 8 values a thread, one 16-byte store each for K and V (16
 * values and two stores: 22 us in place of 18).
 *
 * HBM's bound is 2 * (2 D + D / 2 + D / 16) bytes a token and head.  At 16383 tokens, 8
 * heads of 128: append 21 us = 4.1 TB/s, bound by its instructions (8 values a thread:
 * 28 us), read 18 us = 4.8 TB/s.
 */
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "kv4.cuh"

namespace glint {
namespace {

constexpr int kThreads = 256;

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

struct AppendArgs {
    GlintKv4Cache c;
    const __nv_bfloat16 *k, *v;
    int64_t k_tok, k_head, v_tok, v_head;
    const int *slots;
    uint32_t chunks; /* tokens * kv_heads * D / 16 */
    int page_log2;
};
/* 32-bit chunk numbers: longer calls go in slices of this many tokens */
inline int slice_tokens(const GlintKv4Cache &c) { return (int)std::max((int64_t)1, (int64_t)0x7FFFFFFF / ((int64_t)c.kv_heads * (c.head_dim / 8))); }
inline int log2_of(int n)
{
    int l = 0;
    while ((1 << l) < n)
        ++l;
    return l;
}

template <int D, bool ALIGNED>
__global__ void __launch_bounds__(kThreads) kv4_append_kernel(const AppendArgs a)
{
    constexpr int CH = D / 16; /* chunks a row: a power of two, so a block's 4 lanes stay in one row */
    const uint32_t i = blockIdx.x * kThreads + threadIdx.x;
    const bool live = i < a.chunks;
    const int ch = (int)(i % CH);
    const uint32_t row = live ? i / CH : 0, t = row / (uint32_t)a.c.kv_heads;
    const int h = (int)(row - t * (uint32_t)a.c.kv_heads);
    uint32_t x[8] = {}, y[8] = {};
    const int slot = live ? a.slots[t] : -1;
    if (live) {
        load16<ALIGNED>(a.k + t * a.k_tok + h * a.k_head + ch * 16, x);
        load16<ALIGNED>(a.v + t * a.v_tok + h * a.v_head + ch * 16, y);
    }
    uint32_t km, vm;
    const uint2 kw = quantise16(x, km), vw = quantise16(y, vm);
    if (slot < 0 || slot >= a.c.pages * a.c.page_size)
        return;
    const int page = slot >> a.page_log2, r = slot & (a.c.page_size - 1);
    const int64_t at = (((int64_t)page * a.c.kv_heads + h) << a.page_log2) + r;
    const int64_t byte = at * (D / 2) + kv4_unit<D>(ch / 4, r) + (ch % 4) * 8;
    *reinterpret_cast<uint2 *>(a.c.k_code + byte) = kw;
    *reinterpret_cast<uint2 *>(a.c.v_code + byte) = vw;
    if (ch % 4 == 0) {
        reinterpret_cast<uint32_t *>(a.c.k_meta)[at * (D / 64) + ch / 4] = km;
        reinterpret_cast<uint32_t *>(a.c.v_meta)[at * (D / 64) + ch / 4] = vm;
    }
}

__device__ __forceinline__ uint4 values8(uint32_t w, uint32_t meta)
{
    const float step = __uint_as_float(meta << 16), lo = __uint_as_float(meta & 0xFFFF0000u);
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        /* step * code is exact (8 + 4 bits), so the fma rounds as lo + step * code does */
        const float a = fmaf(step, (float)((w >> (8 * i)) & 15u), lo);
        const float b = fmaf(step, (float)((w >> (8 * i + 4)) & 15u), lo);
        const __nv_bfloat162 p = __floats2bfloat162_rn(a, b);
        u[i] = *reinterpret_cast<const uint32_t *>(&p);
    }
    return make_uint4(u[0], u[1], u[2], u[3]);
}

template <int D>
__global__ void __launch_bounds__(kThreads) kv4_read_kernel(const GlintKv4Cache c, const int *slots, uint32_t chunks,
                                                            int page_log2, uint4 *ko, uint4 *vo)
{
    constexpr int CH = D / 8;
    const uint32_t i = blockIdx.x * kThreads + threadIdx.x;
    if (i >= chunks)
        return;
    const int ch = (int)(i % CH);
    const uint32_t row = i / CH, t = row / (uint32_t)c.kv_heads;
    const int h = (int)(row - t * (uint32_t)c.kv_heads);
    const int slot = slots[t];
    uint4 k = make_uint4(0u, 0u, 0u, 0u), v = k;
    if (slot >= 0 && slot < c.pages * c.page_size) {
        const int page = slot >> page_log2, r = slot & (c.page_size - 1);
        const int64_t at = (((int64_t)page * c.kv_heads + h) << page_log2) + r;
        const int64_t byte = at * (D / 2) + kv4_unit<D>(ch / 8, r) + (ch % 8) * 4;
        const int64_t m = at * (D / 64) + ch / 8;
        const uint32_t kw = *reinterpret_cast<const uint32_t *>(c.k_code + byte);
        const uint32_t vw = *reinterpret_cast<const uint32_t *>(c.v_code + byte);
        k = values8(kw, reinterpret_cast<const uint32_t *>(c.k_meta)[m]);
        v = values8(vw, reinterpret_cast<const uint32_t *>(c.v_meta)[m]);
    }
    ko[i] = k, vo[i] = v;
}

/* ---- eviction --------------------------------------------------------------------
 * A cluster of 1 to 8 CTAs per (sequence, kv head), each with an equal stretch of the
 * slots.  The n-th largest key is found by four passes over 8-bit digits: a histogram in
 * every CTA, summed through the others' shared memory.  A bit per slot (kept) and the
 * running count of bits then number the free slots below n and the kept ones from n on;
 * the free ones are listed across the cluster's shared memory, and the k-th kept one is
 * moved into the k-th of the list.  Sources lie at n and above, destinations below, so
 * the moves do not depend on one another.
 *
 * Floor: 8 bytes a slot and head read (weight and position), 8 + D + D / 8 read and
 * written a slot moved.  Bound: latency, of the seven cluster barriers that this way of
 * finding the n-th key takes whatever the keys, and of what each waits for: for a sequence of 32768 slots about 50000 clocks, 8400 of them for the keys and the
 * first digit's counts, 16000 for the digits, 3000 for the bits, 6600 for the list (the
 * first CTA's slots, mostly), 8700 for the moves (16 bytes a lane; a slot a lane: 14000).
 * 16 ragged sequences of up to 32768 slots to 4096, 8 heads of 128: 33 us (512 threads a
 * CTA: 37, though 27 in place of 32 for two such sequences alone).  8 of 1025 to 1024: 12.6.
 */
constexpr int kEvThreads = 256, kEvWarps = kEvThreads / 32;
constexpr int kEvSlots = 4; /* slots a thread that another CTA is taken for */
constexpr int kEvMaxSlots = 524288;
constexpr int kEvKeys = 40960; /* keys a CTA holds in shared memory; with more it reads weights again */

struct EvictArgs {
    GlintKv4Cache c;
    GlintKv4Evict e;
    int cluster, stretch; /* CTAs a head; slots a CTA at most, a multiple of kEvThreads */
    int page_log2;
};

/* larger key = kept first: protected, then by weight, NaN last */
__device__ __forceinline__ uint32_t evict_key(float w, int pos, int64_t guard)
{
    if (pos >= guard)
        return 0xFFFFFFFFu;
    if (w != w)
        return 0u;
    const uint32_t u = __float_as_uint(w + 0.f); /* -0 and +0 tie */
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ void cluster_barrier()
{
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t there(const void *p, uint32_t cta) /* the same place in another CTA */
{
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(cta));
    return r;
}
__device__ __forceinline__ int load_there(uint32_t a)
{
    int v;
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ void store_there(uint32_t a, int v)
{
    asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(a), "r"(v) : "memory");
}
/* sum over the lanes below this one */
__device__ __forceinline__ int warp_before(int v)
{
    int s = v;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const int o = __shfl_up_sync(0xFFFFFFFFu, s, off);
        if ((int)lane_id() >= off)
            s += o;
    }
    return s - v;
}
template <int D>
__global__ void __launch_bounds__(kEvThreads, 4) kv4_evict_kernel(const EvictArgs a)
{
    extern __shared__ uint32_t ev_smem[];
    __shared__ int hist[2][256];
    __shared__ __align__(16) int tot[256];
    __shared__ int near_of[kEvWarps], far_of[kEvWarps], eq_of[kEvWarps]; /* per warp: free below n, kept from n on, keys equal to the n-th */
    __shared__ int s_free, s_far, s_need, s_same;
    __shared__ uint32_t s_prefix;
    const GlintKv4Cache &c = a.c;
    const GlintKv4Evict &e = a.e;
    const int rank = blockIdx.x % a.cluster, bh = blockIdx.x / a.cluster;
    const int b = bh / c.kv_heads, h = bh - b * c.kv_heads;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int L = min(max(e.lens[b], 0), e.max_pages << a.page_log2), n = min(L, e.budget);
    /* as many CTAs as the length is worth, with an equal stretch of the slots each (a multiple
     * of kEvThreads, no more than a.stretch); the others make room at once, and a cluster's
     * barriers do not wait for them */
    const int ctas = min(a.cluster, max(1, (L + kEvSlots * kEvThreads - 1) / (kEvSlots * kEvThreads)));
    if (rank >= ctas)
        return;
    const int stretch = max(1, (L + ctas * kEvThreads - 1) / (ctas * kEvThreads)) * kEvThreads;
    const int begin = rank * stretch, end = min(L, begin + stretch); /* this CTA's; none where end <= begin */
    const int words = stretch / 32, per_warp = words / kEvWarps;
    uint32_t *bits = ev_smem;                                      /* kept, a bit a slot */
    int *free_at = reinterpret_cast<int *>(bits + a.stretch / 32); /* this warp's free slots below n before a word */
    int *far_at = free_at + a.stretch / 32;                        /* its kept slots from n on before a word */
    uint32_t *keys = reinterpret_cast<uint32_t *>(far_at + a.stretch / 32); /* later this CTA's part of the list of free slots */
    int *list = reinterpret_cast<int *>(keys);
    const bool held = a.stretch <= kEvKeys;
    const int64_t row = (int64_t)bh * e.stride;
    const float *w = e.weight + row;
    const int *pos = e.pos + row;
    const int64_t guard = (int64_t)e.seen[b] - e.recent;
    auto key = [&](int t) { return held ? keys[t - begin] : evict_key(__ldg(w + t), __ldg(pos + t), guard); };
    if (h == 0 && rank == 0 && tid == 0)
        e.new_lens[b] = n;
    for (int i = tid; i < 256; i += kEvThreads)
        hist[0][i] = 0;
    __syncthreads();
    if (held) { /* and the first digit's counts: integers, so any order gives the same */
#pragma unroll 8
        for (int t = begin + tid; t < end; t += kEvThreads) {
            const uint32_t k = evict_key(__ldg(w + t), __ldg(pos + t), guard);
            keys[t - begin] = k;
            atomicAdd(&hist[0][k >> 24], 1);
        }
    }
    __syncthreads();

    /* the n-th largest key, a digit at a time */
    uint32_t prefix = 0;
    int need = n, eq_before = 0;
    if (L > n) {
        for (int p = 0; p < 4; ++p) {
            const int shift = 24 - 8 * p;
            const uint32_t high = p ? 0xFFFFFFFFu << (shift + 8) : 0u;
            if (p || !held) {
#pragma unroll 4
                for (int t = begin + tid; t < end; t += kEvThreads) {
                    const uint32_t k = key(t);
                    if ((k & high) == prefix)
                        atomicAdd(&hist[p & 1][(k >> shift) & 255u], 1);
                }
            }
            cluster_barrier();
            if (tid < 256) {
                int n[8], sum = 0;
#pragma unroll
                for (int r = 0; r < 8; ++r)
                    n[r] = r < ctas ? load_there(there(&hist[p & 1][tid], r)) : 0;
#pragma unroll
                for (int r = 0; r < 8; ++r)
                    sum += n[r];
                tot[tid] = sum;
                hist[(p + 1) & 1][tid] = 0; /* read by the others before the barrier above */
            }
            __syncthreads();
            if (warp == 0) { /* lane i: bins 255 - 8 i down to 248 - 8 i */
                const int4 hi = reinterpret_cast<const int4 *>(tot)[63 - 2 * lane], lo = reinterpret_cast<const int4 *>(tot)[62 - 2 * lane];
                const int in[8] = {hi.w, hi.z, hi.y, hi.x, lo.w, lo.z, lo.y, lo.x};
                int sum = 0;
#pragma unroll
                for (int q = 0; q < 8; ++q)
                    sum += in[q];
                int left = need - warp_before(sum); /* still wanted from this lane's bins on */
                if (left > 0 && left <= sum) {
#pragma unroll
                    for (int q = 0; q < 8; ++q) {
                        if (left > 0 && left <= in[q])
                            s_prefix = prefix | ((uint32_t)(255 - 8 * lane - q) << shift), s_need = left, s_same = in[q];
                        left -= in[q];
                    }
                }
            }
            __syncthreads();
            prefix = s_prefix, need = s_need;
        }
    }
    /* kept: above the n-th key, and of those equal to it the `need` lowest slots (or all,
     * where there are no more).  A warp has per_warp words of 32 slots. */
    const int w0 = warp * per_warp;
    const bool ties = L > n && s_same > need;
    if (ties) { /* the last histogram counts, for its digit, the keys equal to the n-th */
#pragma unroll
        for (int r = 0; r < 8; ++r)
            eq_before += r < rank ? load_there(there(&hist[1][prefix & 255u], r)) : 0;
        int eqs = 0;
        for (int q = 0; q < per_warp; ++q) {
            const int t = begin + (w0 + q) * 32 + lane;
            eqs += __popc(__ballot_sync(0xFFFFFFFFu, t < end && key(t) == prefix));
        }
        if (lane == 0)
            eq_of[warp] = eqs;
        __syncthreads();
        for (int k = 0; k < warp; ++k)
            eq_before += eq_of[k];
    }
    int frees = 0, fars = 0;
#pragma unroll 4
    for (int q = 0; q < per_warp; ++q) {
        const int t0 = begin + (w0 + q) * 32, t = t0 + lane;
        const uint32_t k = t < end ? key(t) : 0u;
        bool keep = t < end && (L <= n || k >= prefix);
        if (ties) {
            const uint32_t me = __ballot_sync(0xFFFFFFFFu, t < end && k == prefix);
            if (k == prefix && eq_before + __popc(me & ((1u << lane) - 1u)) >= need)
                keep = false;
            eq_before += __popc(me);
        }
        const uint32_t m = __ballot_sync(0xFFFFFFFFu, keep), below = __ballot_sync(0xFFFFFFFFu, t < n);
        if (lane == 0)
            bits[w0 + q] = m, free_at[w0 + q] = frees, far_at[w0 + q] = fars;
        frees += __popc(below & ~m), fars += __popc(m & ~below);
    }
    if (lane == 0)
        near_of[warp] = frees, far_of[warp] = fars;
    __syncthreads(); /* also: the keys are not needed any more */
    if (warp == 0) {
        const int f = lane < kEvWarps ? near_of[lane] : 0, g = lane < kEvWarps ? far_of[lane] : 0;
        const int fb = warp_before(f), gb = warp_before(g);
        if (lane < kEvWarps)
            near_of[lane] = fb, far_of[lane] = gb;
        if (lane == 31)
            s_free = fb + f, s_far = gb + g;
    }
    cluster_barrier(); /* counts and the keys' memory, of every CTA */
    int free_base = 0, far_base = 0, moved = 0;
#pragma unroll
    for (int r = 0; r < 8; ++r) {
        const int f = r < ctas ? load_there(there(&s_free, r)) : 0, g = r < ctas ? load_there(there(&s_far, r)) : 0;
        free_base += r < rank ? f : 0, far_base += r < rank ? g : 0, moved += f;
    }
    const int part = max(1, (moved + ctas - 1) / ctas); /* entries of the list a CTA holds */
    const uint32_t inv = 0xFFFFFFFFu / (uint32_t)part;
    auto entry = [&](int k) { /* entry k of the list, k < 2^19: at most one off before the step up */
        int r = (int)__umulhi((uint32_t)k, inv);
        r += k - r * part >= part;
        return there(&list[k - r * part], r);
    };
    int *kept = e.kept + (int64_t)bh * e.budget;
#pragma unroll 2
    for (int q = 0; q < per_warp; ++q) { /* the free slots of this CTA's into the list */
        const int t0 = begin + (w0 + q) * 32, t = t0 + lane;
        const uint32_t out = t0 >= n ? 0u : ~bits[w0 + q] & (n - t0 >= 32 ? 0xFFFFFFFFu : (1u << (n - t0)) - 1u);
        if ((out >> lane) & 1u) {
            const int k = free_base + near_of[warp] + free_at[w0 + q] + __popc(out & ((1u << lane) - 1u));
            store_there(entry(k), t);
        }
    }
    cluster_barrier(); /* lists, the last words that others write here */
    /* the kept ones below n, shared out evenly: most of them lie in the first CTAs */
#pragma unroll 4
    for (int t = rank * kEvThreads + tid; t < n; t += ctas * kEvThreads) {
        const int r = t / stretch, at = t - r * stretch;
        if ((load_there(there(&bits[at / 32], r)) >> (at % 32)) & 1)
            kept[t] = t, e.weight_out[row + t] = __ldg(w + t), e.pos_out[row + t] = __ldg(pos + t);
    }
    for (int i = n + rank * kEvThreads + tid; i < e.budget; i += ctas * kEvThreads)
        kept[i] = -1;
    /* the kept slots from n on: a lane each to find number j of this CTA's by two searches, then
     * the lanes together, 16 bytes each of K and of V */
    constexpr int kLanes = D / 16; /* a slot's */
    const int *table = e.table + (int64_t)b * e.max_pages;
    for (int j0 = warp * 32; j0 < s_far; j0 += kEvThreads) {
        const int j = j0 + lane;
        int64_t from = -1, to = -1; /* slots' rows in the cache */
        if (j < s_far) {
            int wp = 0;
#pragma unroll
            for (int step = kEvWarps / 2; step > 0; step /= 2)
                if (far_of[wp + step] <= j)
                    wp += step;
            const int in = j - far_of[wp];
            int lo = wp * per_warp, hi = lo + per_warp - 1; /* its last word with far_at <= in */
            while (lo < hi) {
                const int mid = (lo + hi + 1) / 2;
                if (far_at[mid] <= in)
                    lo = mid;
                else
                    hi = mid - 1;
            }
            uint32_t m = bits[lo];
            const int t0 = begin + lo * 32;
            if (t0 < n)
                m &= 0xFFFFFFFFu << (n - t0); /* n - t0 < 32: the word has a slot from n on */
            int skip = in - far_at[lo], at = 0; /* its bit after `skip` others, by halves */
#pragma unroll
            for (int half = 16; half > 0; half /= 2) {
                const int low = __popc(m >> at & ((1u << half) - 1u));
                if (skip >= low)
                    skip -= low, at += half;
            }
            const int src = t0 + at, k = far_base + j;
            const int dst = load_there(entry(k));
            const float weight = __ldg(w + src);
            const int position = __ldg(pos + src);
            const int pf = __ldg(table + (src >> a.page_log2)), pt = __ldg(table + (dst >> a.page_log2));
            kept[dst] = src, e.weight_out[row + dst] = weight, e.pos_out[row + dst] = position;
            if (pf >= 0 && pf < c.pages && pt >= 0 && pt < c.pages) {
                from = (((int64_t)pf * c.kv_heads + h) << a.page_log2) + (src & (c.page_size - 1));
                to = (((int64_t)pt * c.kv_heads + h) << a.page_log2) + (dst & (c.page_size - 1));
            }
        }
        const int part16 = lane % (kLanes / 2), block = part16 / 2; /* 16 bytes of a row */
        const bool is_v = lane % kLanes >= kLanes / 2;
        uint8_t *const code = is_v ? c.v_code : c.k_code;
        uint32_t *const meta = reinterpret_cast<uint32_t *>(is_v ? c.v_meta : c.k_meta);
        uint4 x[kLanes];
        uint32_t y[kLanes];
#pragma unroll
        for (int q = 0; q < kLanes; ++q) {
            const int64_t at = __shfl_sync(0xFFFFFFFFu, from, q * (32 / kLanes) + lane / kLanes);
            if (at >= 0) {
                const int r = (int)at & (c.page_size - 1);
                x[q] = *reinterpret_cast<const uint4 *>(code + at * (D / 2) + kv4_unit<D>(block, r) + (part16 % 2) * 16);
                y[q] = part16 < D / 64 ? meta[at * (D / 64) + part16] : 0u;
            }
        }
#pragma unroll
        for (int q = 0; q < kLanes; ++q) {
            const int64_t at = __shfl_sync(0xFFFFFFFFu, to, q * (32 / kLanes) + lane / kLanes);
            if (at >= 0) {
                const int r = (int)at & (c.page_size - 1);
                *reinterpret_cast<uint4 *>(code + at * (D / 2) + kv4_unit<D>(block, r) + (part16 % 2) * 16) = x[q];
                if (part16 < D / 64)
                    meta[at * (D / 64) + part16] = y[q];
            }
        }
    }
    /* no CTA leaves while another may read its bits or list; nothing is handed over */
    __syncwarp();
    asm volatile("barrier.cluster.arrive.relaxed.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}

int launched() { return cudaGetLastError() == cudaSuccess ? kOk : kLaunch; }

} // namespace
} // namespace glint

using namespace glint;

extern "C" {

int glint_kv4_append_stream(const GlintKv4Cache *c, const glint_bf16_t *k, const glint_bf16_t *v, int64_t k_tok,
                            int64_t k_head, int64_t v_tok, int64_t v_head, const int *slots, int tokens,
                            cudaStream_t stream)
{
    const int rc = kv4_check(c);
    if (rc != kOk)
        return rc;
    if (tokens < 0 || (tokens > 0 && (!k || !v || !slots)))
        return kBadArg;
    if (tokens == 0)
        return kOk;
    const bool al = aligned_to(k, 16) && aligned_to(v, 16) && (k_tok | k_head | v_tok | v_head) % 8 == 0;
    const auto kernel = c->head_dim == 128 ? (al ? kv4_append_kernel<128, true> : kv4_append_kernel<128, false>)
                                           : (al ? kv4_append_kernel<64, true> : kv4_append_kernel<64, false>);
    const int most = slice_tokens(*c);
    for (int t = 0; t < tokens; t += std::min(most, tokens - t)) {
        const uint32_t n = (uint32_t)std::min(most, tokens - t) * c->kv_heads * (c->head_dim / 16);
        const AppendArgs a{*c, k + t * k_tok, v + t * v_tok, k_tok, k_head, v_tok, v_head, slots + t, n, log2_of(c->page_size)};
        kernel<<<(n + kThreads - 1) / kThreads, kThreads, 0, stream>>>(a);
    }
    return launched();
}

int glint_kv4_read_stream(const GlintKv4Cache *c, const int *slots, int tokens, glint_bf16_t *k_out,
                          glint_bf16_t *v_out, cudaStream_t stream)
{
    const int rc = kv4_check(c);
    if (rc != kOk)
        return rc;
    if (tokens < 0 || (tokens > 0 && (!k_out || !v_out || !slots || !aligned_to(k_out, 16) || !aligned_to(v_out, 16))))
        return kBadArg;
    if (tokens == 0)
        return kOk;
    const auto kernel = c->head_dim == 128 ? kv4_read_kernel<128> : kv4_read_kernel<64>;
    const int most = slice_tokens(*c);
    uint4 *ko = reinterpret_cast<uint4 *>(k_out), *vo = reinterpret_cast<uint4 *>(v_out);
    for (int t = 0; t < tokens; t += std::min(most, tokens - t)) {
        const uint32_t n = (uint32_t)std::min(most, tokens - t) * c->kv_heads * (c->head_dim / 8);
        const int64_t at = (int64_t)t * c->kv_heads * (c->head_dim / 8);
        kernel<<<(n + kThreads - 1) / kThreads, kThreads, 0, stream>>>(*c, slots + t, n, log2_of(c->page_size), ko + at, vo + at);
    }
    return launched();
}

int glint_kv4_evict_stream(const GlintKv4Cache *c, const GlintKv4Evict *e, cudaStream_t stream)
{
    const int rc = kv4_check(c);
    if (rc != kOk)
        return rc;
    if (!e || e->seqs < 0 || e->max_pages < 1 || e->budget < 1 || e->recent < 0 || e->recent > e->budget ||
        (int64_t)e->max_pages * c->page_size > kEvMaxSlots || (int64_t)e->max_pages * c->page_size > e->stride)
        return kBadArg;
    if (e->seqs == 0)
        return kOk;
    if (!e->table || !e->lens || !e->weight || !e->pos || !e->seen || !e->kept || !e->new_lens || !e->weight_out ||
        !e->pos_out || e->weight == e->weight_out || e->pos == e->pos_out ||
        (int64_t)e->seqs * c->kv_heads > INT32_MAX)
        return kBadArg;
    /* new_lens is written while other heads' CTAs, and others of a cluster, still read lens and seen:
     * CTAs that disagree on a length disagree on which of them take part */
    auto apart = [&](const int *in) { return in + e->seqs <= e->new_lens || e->new_lens + e->seqs <= in; };
    if (!apart(e->lens) || !apart(e->seen))
        return kBadArg;
    EvictArgs a{*c, *e, 1, 0, log2_of(c->page_size)};
    /* up to eight CTAs (a portable cluster) while each thread has kEvSlots or more */
    const int cap = e->max_pages * c->page_size;
    while (a.cluster < 8 && cap > kEvSlots * kEvThreads * a.cluster)
        a.cluster *= 2;
    /* a CTA's memory: its share of the longest sequence, or what fewer CTAs have of a shorter one */
    a.stretch = std::max((cap + a.cluster * kEvThreads - 1) / (a.cluster * kEvThreads), kEvSlots) * kEvThreads;
    if ((int64_t)e->seqs * c->kv_heads * a.cluster > INT32_MAX)
        return kBadArg;
    /* keys, or at least this CTA's part of the list: at most half of the slots are free ones below n */
    const int smem = a.stretch / 32 * 12 + (a.stretch <= kEvKeys ? a.stretch * 4 : a.stretch / 2 * 4 + 16);
    const auto kernel = c->head_dim == 128 ? kv4_evict_kernel<128> : kv4_evict_kernel<64>;
    if (!ensure_smem((const void *)kernel, kEvKeys / 32 * 12 + kEvKeys * 4))
        return kLaunch;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)a.cluster, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3((unsigned)(e->seqs * c->kv_heads * a.cluster)), cfg.blockDim = dim3(kEvThreads);
    cfg.dynamicSmemBytes = smem, cfg.stream = stream, cfg.attrs = attr, cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, kernel, a) != cudaSuccess) {
        cudaGetLastError();
        return kLaunch;
    }
    return launched();
}

} /* extern "C" */
