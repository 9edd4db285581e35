/* The 4-bit key/value cache: append (quantise rows into their slots), read (slots back
 * to BF16) and eviction by accumulated attention weight.
 *
 * Append and read move each byte once: a thread takes 8 neighbouring values of a row
 * (16 bytes of BF16, 4 bytes of codes), the 8 threads of a 64-value block find its
 * minimum and maximum with three shuffles, and K and V go through one thread so that
 * two loads are in flight.  HBM-bound in principle: 2 * (2 D + D / 2 + D / 16) bytes a
 * token and head.
 */
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "kv4.cuh"

namespace glint {
namespace {

constexpr int kThreads = 256;

/* 8 values of a row, BF16 -> f32; ALIGNED: one 16-byte load */
template <bool ALIGNED>
__device__ __forceinline__ void load8(const __nv_bfloat16 *p, float (&x)[8])
{
    if constexpr (ALIGNED) {
        const uint4 w = __ldg(reinterpret_cast<const uint4 *>(p));
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
            x[2 * i] = __uint_as_float(u[i] << 16), x[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            x[i] = __bfloat162float(p[i]);
    }
}

/* One block's 8 values of this lane -> 8 nibbles; (step, lo) of the block the same in
 * all 8 lanes of the aligned group. */
__device__ __forceinline__ uint32_t quantise8(const float (&x)[8], uint32_t &meta)
{
    float lo = x[0], hi = x[0];
    /* any NaN or infinity: its exponent is all ones, and stays so in this difference */
    float odd = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        lo = fminf(lo, x[i]), hi = fmaxf(hi, x[i]);
        odd += x[i] - x[i];
    }
#pragma unroll
    for (int off = 4; off > 0; off >>= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xFFFFFFFFu, lo, off));
        hi = fmaxf(hi, __shfl_xor_sync(0xFFFFFFFFu, hi, off));
        odd += __shfl_xor_sync(0xFFFFFFFFu, odd, off);
    }
    const __nv_bfloat16 sb = __float2bfloat16_rn(__fdiv_rn(hi - lo, 15.f));
    const float step = __bfloat162float(sb);
    if (odd != 0.f || step - step != 0.f) { /* not finite: the block reads as NaN */
        meta = 0x7FC00000u;
        return 0u;
    }
    /* lo is one of the BF16 inputs, so its upper half is all of it */
    meta = (__float_as_uint(lo) & 0xFFFF0000u) | (uint32_t)__bfloat16_as_ushort(sb);
    uint32_t w = 0;
    if (step > 0.f) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float c = fminf(fmaxf(rintf(__fdiv_rn(x[i] - lo, step)), 0.f), 15.f);
            w |= (uint32_t)c << (4 * i);
        }
    }
    return w;
}

struct AppendArgs {
    GlintKv4Cache c;
    const __nv_bfloat16 *k, *v;
    int64_t k_tok, k_head, v_tok, v_head;
    const int *slots;
    int64_t chunks; /* tokens * kv_heads * D / 8 */
};

template <int D, bool ALIGNED>
__global__ void __launch_bounds__(kThreads) kv4_append_kernel(const AppendArgs a)
{
    constexpr int CH = D / 8; /* chunks a row: a power of two, so a block's 8 lanes stay in one row */
    const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    const bool live = i < a.chunks;
    const int ch = (int)(i % CH);
    const int64_t row = i / CH;
    const int h = live ? (int)(row % a.c.kv_heads) : 0;
    const int64_t t = live ? row / a.c.kv_heads : 0;
    float x[8] = {}, y[8] = {};
    const int slot = live ? a.slots[t] : -1;
    if (live) {
        load8<ALIGNED>(a.k + t * a.k_tok + h * a.k_head + ch * 8, x);
        load8<ALIGNED>(a.v + t * a.v_tok + h * a.v_head + ch * 8, y);
    }
    uint32_t km, vm;
    const uint32_t kw = quantise8(x, km), vw = quantise8(y, vm);
    if (slot < 0 || slot >= a.c.pages * a.c.page_size)
        return;
    const int page = slot / a.c.page_size, r = slot - page * a.c.page_size;
    const int64_t at = ((int64_t)page * a.c.kv_heads + h) * a.c.page_size + r;
    const int64_t byte = at * (D / 2) + kv4_unit<D>(ch / 8, r) + (ch % 8) * 4;
    *reinterpret_cast<uint32_t *>(a.c.k_code + byte) = kw;
    *reinterpret_cast<uint32_t *>(a.c.v_code + byte) = vw;
    if (ch % 8 == 0) {
        reinterpret_cast<uint32_t *>(a.c.k_meta)[at * (D / 64) + ch / 8] = km;
        reinterpret_cast<uint32_t *>(a.c.v_meta)[at * (D / 64) + ch / 8] = vm;
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
__global__ void __launch_bounds__(kThreads) kv4_read_kernel(const GlintKv4Cache c, const int *slots, int64_t chunks,
                                                            uint4 *ko, uint4 *vo)
{
    constexpr int CH = D / 8;
    const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (i >= chunks)
        return;
    const int ch = (int)(i % CH);
    const int64_t row = i / CH;
    const int h = (int)(row % c.kv_heads);
    const int slot = slots[row / c.kv_heads];
    uint4 k = make_uint4(0u, 0u, 0u, 0u), v = k;
    if (slot >= 0 && slot < c.pages * c.page_size) {
        const int page = slot / c.page_size, r = slot - page * c.page_size;
        const int64_t at = ((int64_t)page * c.kv_heads + h) * c.page_size + r;
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
 * One CTA per (sequence, kv head).  The n-th largest key is found by four passes over
 * 8-bit digits (a histogram each); a bit per slot and the running count of kept bits
 * then give, for the k-th free slot below n, the k-th kept slot from n on by a binary
 * search, so no list is built and the moves are independent of one another (sources
 * lie at n and above, destinations below). */
constexpr int kEvThreads = 1024;
constexpr int kEvMaxSlots = 524288;

struct EvictArgs {
    GlintKv4Cache c;
    GlintKv4Evict e;
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

__device__ __forceinline__ int block_scan(int v, int *warp_sums, int &total)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int s = v;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const int o = __shfl_up_sync(0xFFFFFFFFu, s, off);
        if (lane >= off)
            s += o;
    }
    if (lane == 31)
        warp_sums[warp] = s;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < kEvThreads / 32; ++w) {
        before += w < warp ? warp_sums[w] : 0;
        total += warp_sums[w];
    }
    __syncthreads();
    return before + s - v; /* exclusive */
}

template <int D>
__global__ void __launch_bounds__(kEvThreads) kv4_evict_kernel(const EvictArgs a)
{
    extern __shared__ uint32_t ev_smem[];
    __shared__ int hist[256];
    __shared__ int warp_sums[kEvThreads / 32];
    __shared__ uint32_t s_prefix;
    __shared__ int s_need;
    const GlintKv4Cache &c = a.c;
    const GlintKv4Evict &e = a.e;
    const int b = blockIdx.x / c.kv_heads, h = blockIdx.x - b * c.kv_heads;
    const int tid = threadIdx.x, lane = tid & 31;
    const int cap = e.max_pages * c.page_size;
    const int L = min(max(e.lens[b], 0), cap), n = min(L, e.budget);
    const int words = (cap + 31) / 32;
    uint32_t *bits = ev_smem;                             /* one bit per slot: kept */
    int *rank = reinterpret_cast<int *>(ev_smem + words); /* kept bits before each word */
    const int64_t row = ((int64_t)b * c.kv_heads + h) * e.stride;
    const float *w = e.weight + row;
    const int *pos = e.pos + row;
    const int64_t guard = (int64_t)e.seen[b] - e.recent;
    if (h == 0 && tid == 0)
        e.new_lens[b] = n;

    /* the n-th largest key, a digit at a time */
    uint32_t prefix = 0;
    int need = n;
    for (int shift = 24; shift >= 0 && L > n; shift -= 8) {
        if (tid < 256)
            hist[tid] = 0;
        __syncthreads();
        const uint32_t high = shift == 24 ? 0u : 0xFFFFFFFFu << (shift + 8);
        for (int t = tid; t < L; t += kEvThreads) {
            const uint32_t k = evict_key(w[t], pos[t], guard);
            if ((k & high) == prefix)
                atomicAdd(&hist[(k >> shift) & 255u], 1); /* integer counts: the order does not matter */
        }
        __syncthreads();
        if (tid == 0) {
            int d = 255, left = need;
            while (d > 0 && hist[d] < left)
                left -= hist[d--];
            s_prefix = prefix | ((uint32_t)d << shift);
            s_need = left;
        }
        __syncthreads();
        prefix = s_prefix, need = s_need;
        __syncthreads();
    }
    /* kept: above the n-th key, and of those equal to it the `need` lowest slots */
    int eq_before = 0, kept_before = 0;
    for (int t0 = 0; t0 < L; t0 += kEvThreads) {
        const int t = t0 + tid;
        const uint32_t k = t < L ? evict_key(w[t], pos[t], guard) : 0u;
        const bool eq = t < L && L > n && k == prefix;
        int total;
        const int r = block_scan(eq ? 1 : 0, warp_sums, total);
        const bool keep = t < L && (L <= n || k > prefix || (eq && eq_before + r < need));
        eq_before += total;
        const uint32_t m = __ballot_sync(0xFFFFFFFFu, keep);
        int all;
        const int kr = block_scan(keep ? 1 : 0, warp_sums, all);
        if (lane == 0 && t / 32 < words)
            bits[t / 32] = m, rank[t / 32] = kept_before + kr;
        kept_before += all;
    }
    __syncthreads();
    /* result slot i: itself where kept, else the matching kept slot from n on */
    int *kept = e.kept + ((int64_t)b * c.kv_heads + h) * e.budget;
    const int below = n > 0 ? rank[(n - 1) / 32] + __popc(bits[(n - 1) / 32] & (0xFFFFFFFFu >> (31 - (n - 1) % 32))) : 0;
    for (int i = tid; i < e.budget; i += kEvThreads) {
        if (i >= n) {
            kept[i] = -1;
            continue;
        }
        int src = i;
        if (!((bits[i / 32] >> (i % 32)) & 1u)) {
            /* i is free slot number i - (kept before i); its row is kept slot `want` of all */
            const int want = below + i - (rank[i / 32] + __popc(bits[i / 32] & ((1u << (i % 32)) - 1u)));
            int lo = 0, hi = (L - 1) / 32; /* last word with rank <= want */
            while (lo < hi) {
                const int mid = (lo + hi + 1) / 2;
                if (rank[mid] <= want)
                    lo = mid;
                else
                    hi = mid - 1;
            }
            src = lo * 32 + __fns(bits[lo], 0, want - rank[lo] + 1);
        }
        kept[i] = src;
        e.weight_out[row + i] = w[src];
        e.pos_out[row + i] = pos[src];
        if (src == i)
            continue;
        const int *table = e.table + (int64_t)b * e.max_pages;
        const int pf = table[src / c.page_size], pt = table[i / c.page_size];
        if (pf < 0 || pf >= c.pages || pt < 0 || pt >= c.pages)
            continue;
        const int rf = src % c.page_size, rt = i % c.page_size;
        const int64_t from = ((int64_t)pf * c.kv_heads + h) * c.page_size + rf;
        const int64_t to = ((int64_t)pt * c.kv_heads + h) * c.page_size + rt;
        uint4 kc[D / 32], vc[D / 32];
#pragma unroll
        for (int q = 0; q < D / 32; ++q) {
            kc[q] = *reinterpret_cast<const uint4 *>(c.k_code + from * (D / 2) + kv4_unit<D>(q / 2, rf) + (q % 2) * 16);
            vc[q] = *reinterpret_cast<const uint4 *>(c.v_code + from * (D / 2) + kv4_unit<D>(q / 2, rf) + (q % 2) * 16);
        }
        uint32_t km[D / 64], vm[D / 64];
#pragma unroll
        for (int q = 0; q < D / 64; ++q) {
            km[q] = reinterpret_cast<const uint32_t *>(c.k_meta)[from * (D / 64) + q];
            vm[q] = reinterpret_cast<const uint32_t *>(c.v_meta)[from * (D / 64) + q];
        }
#pragma unroll
        for (int q = 0; q < D / 32; ++q) {
            *reinterpret_cast<uint4 *>(c.k_code + to * (D / 2) + kv4_unit<D>(q / 2, rt) + (q % 2) * 16) = kc[q];
            *reinterpret_cast<uint4 *>(c.v_code + to * (D / 2) + kv4_unit<D>(q / 2, rt) + (q % 2) * 16) = vc[q];
        }
#pragma unroll
        for (int q = 0; q < D / 64; ++q) {
            reinterpret_cast<uint32_t *>(c.k_meta)[to * (D / 64) + q] = km[q];
            reinterpret_cast<uint32_t *>(c.v_meta)[to * (D / 64) + q] = vm[q];
        }
    }
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
    const AppendArgs a{*c, k, v, k_tok, k_head, v_tok, v_head, slots, (int64_t)tokens * c->kv_heads * (c->head_dim / 8)};
    const bool al = aligned_to(k, 16) && aligned_to(v, 16) && (k_tok | k_head | v_tok | v_head) % 8 == 0;
    const unsigned grid = (unsigned)((a.chunks + kThreads - 1) / kThreads);
    if (c->head_dim == 128)
        al ? kv4_append_kernel<128, true><<<grid, kThreads, 0, stream>>>(a)
           : kv4_append_kernel<128, false><<<grid, kThreads, 0, stream>>>(a);
    else
        al ? kv4_append_kernel<64, true><<<grid, kThreads, 0, stream>>>(a)
           : kv4_append_kernel<64, false><<<grid, kThreads, 0, stream>>>(a);
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
    const int64_t chunks = (int64_t)tokens * c->kv_heads * (c->head_dim / 8);
    const unsigned grid = (unsigned)((chunks + kThreads - 1) / kThreads);
    uint4 *ko = reinterpret_cast<uint4 *>(k_out), *vo = reinterpret_cast<uint4 *>(v_out);
    if (c->head_dim == 128)
        kv4_read_kernel<128><<<grid, kThreads, 0, stream>>>(*c, slots, chunks, ko, vo);
    else
        kv4_read_kernel<64><<<grid, kThreads, 0, stream>>>(*c, slots, chunks, ko, vo);
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
    const EvictArgs a{*c, *e};
    const int words = (e->max_pages * c->page_size + 31) / 32;
    const int smem = words * 8;
    const void *kern = c->head_dim == 128 ? (const void *)kv4_evict_kernel<128> : (const void *)kv4_evict_kernel<64>;
    if (smem > 40 * 1024 && !ensure_smem(kern, kEvMaxSlots / 32 * 8))
        return kLaunch;
    const unsigned grid = (unsigned)(e->seqs * c->kv_heads);
    if (c->head_dim == 128)
        kv4_evict_kernel<128><<<grid, kEvThreads, smem, stream>>>(a);
    else
        kv4_evict_kernel<64><<<grid, kEvThreads, smem, stream>>>(a);
    return launched();
}

} /* extern "C" */
