/* The gated feed-forward projection's entry point: which kernel takes a call, and the pass over x before it.
 *
 * In fast mode weights and activations meet the tensor cores in FP16: a weight's rounding to one BF16 value (2^-8
 * of it) would show in h as much as h's own rounding does (error against 64 bits 0.0027 of h's norm, where
 * BF16 outputs alone are 0.0017 off), to one FP16 value (2^-11) it does not (0.0017), at the same rate.
 * FP16's range is what that takes care of: each row of x is multiplied by the power of two that brings its
 * largest finite value into [2^14, 2^15), exactly: every BF16 value down to 2^-29 of the largest keeps all its bits,
 * and what lies below is off by 2^-39 of the largest at most.  Where weights carry their absmax into the
 * products (more than 32 rows), so is each row of W by the one that brings its largest absmax into [2^14, 2^15) (no cell
 * is above 1; products of 2^30 at most, whose sums stay far inside f32): every weight down to 2^-28 of its row's largest
 * absmax keeps its 11 bits, and what lies below is off by 2^-39 of that at most.
 * The epilogues divide by both, again exactly.  The pass is one small kernel (a row of x a CTA; 2.8 us for a token,
 * 25 for 8191 x 4096), beside which the next kernel's weights stream or are expanded.
 *
 * Three ways, at 4096 x 2 x 14336 (us; memory's floor 19.5, the tensor cores' 0.145 a row in a burst):
 *   1 to 32 rows    the decode kernels, lookups straight into mma.sync: 35.9 for a row, 63.3 for 32 (the second 67.5
 *                   for 33)
 *   from there      the tcgen05 product from planes: 68 for 64 rows, 81 for 256, 135 for 511
 *   from 769 rows, unless there are fewer tiles than CTA pairs, weights expanded first: 226 to 231 for 900 (the
 *                   second 262), 381 to 391 for 2048 (483), 1330 to 1515 for 8191, as the clock goes (2246)
 * Precise mode takes the first two ways with x as it is: 37.4 us for a row (the pass is not there), 78.5 for 32, 126
 * for 64, 421 for 511, 5745 for 8191.
 */
#include <cuda_fp16.h>

#include <algorithm>

#include "common.cuh"
#include "gated.cuh"
#include "glint_internal.h"
#include "ptx.cuh"

namespace glint {
namespace {

constexpr int kThreads = 256;
constexpr int kHeld = 4; /* 16 bytes a thread that stay in registers: K up to 8192 */
/* rows that the decode kernels take; 17 and 32 rows there, and through the tcgen05 product: 2560 x 2 x 6911 20.6 and
 * 21.5 us, 29.7; 4096 x 2 x 14336 60.9 and 63.1, 68; 8192 x 2 x 28672 196 and 199, 209; 1024 x 2 x 2000 10.7 and 10.4, 17 */
constexpr int kDecodeM = 32;

struct PrepArgs {
    const __nv_bfloat16 *x;
    __half *x16;
    float *x_scale;
    const float *absmax;
    float *row_scale;
    int *counts;
    int M, N, K;
    int x_ctas, row_ctas, n_counts;
    int expands; /* gated_expand_kernel follows */
};

/* largest finite |value| of two BF16, as its bits */
__device__ __forceinline__ uint32_t top2(uint32_t w, uint32_t top)
{
    const uint32_t lo = w & 0x7FFFu, hi = (w >> 16) & 0x7FFFu;
    top = lo < 0x7F80u ? max(top, lo) : top;
    return hi < 0x7F80u ? max(top, hi) : top;
}
/* 2^k, k in [-126, 127] */
__device__ __forceinline__ float power(int k) { return __uint_as_float((uint32_t)(k + 127) << 23); }

__device__ __forceinline__ uint32_t finite_bits(float v)
{
    const uint32_t b = __float_as_uint(v) & 0x7FFFFFFFu;
    return b < 0x7F800000u ? b : 0u;
}
/* the power of two that brings a row of W whose largest absmax has these bits into [2^14, 2^15); up to 2^126, so
 * that its inverse is a normal number too */
__device__ __forceinline__ float row_power(uint32_t top)
{
    return power(min(126, 14 - ((int)(top >> 23) - 127)));
}

__global__ void __launch_bounds__(kThreads) gated_prep_kernel(const PrepArgs a)
{
    /* The next kernel may start.  One that reads what is written here waits for this one, its weights stream
     * meanwhile; gated_expand_kernel writes what kernels before this one may still read. */
    if (!a.expands)
        asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (a.expands)
        asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int cta = blockIdx.x, warp = threadIdx.x / 32, lane = threadIdx.x & 31;
    if (cta < a.x_ctas) {
        __shared__ uint32_t tops[kThreads / 32];
        const uint4 *x = reinterpret_cast<const uint4 *>(a.x + (int64_t)cta * a.K);
        uint4 *out = reinterpret_cast<uint4 *>(a.x16 + (int64_t)cta * a.K);
        const int n = a.K / 8;
        uint4 held[kHeld];
        uint32_t top = 0;
#pragma unroll
        for (int j = 0; j < kHeld; ++j) {
            const int i = threadIdx.x + j * kThreads;
            held[j] = i < n ? x[i] : make_uint4(0u, 0u, 0u, 0u);
        }
#pragma unroll
        for (int j = 0; j < kHeld; ++j)
            top = top2(held[j].x, top2(held[j].y, top2(held[j].z, top2(held[j].w, top))));
        for (int i = threadIdx.x + kHeld * kThreads; i < n; i += kThreads) {
            const uint4 w = x[i];
            top = top2(w.x, top2(w.y, top2(w.z, top2(w.w, top))));
        }
        top = __reduce_max_sync(0xFFFFFFFFu, top);
        if (lane == 0)
            tops[warp] = top;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kThreads / 32; ++i)
            top = max(top, tops[i]);
        const int k = min(126, 14 - ((int)(top >> 7) - 127)); /* >= -113 */
        const float by = power(k);
        auto pair = [&](uint32_t w) {
            const __half2 h = __floats2half2_rn(__uint_as_float(w << 16) * by, __uint_as_float(w & 0xFFFF0000u) * by);
            return *reinterpret_cast<const uint32_t *>(&h);
        };
        auto put = [&](int i, uint4 w) { out[i] = make_uint4(pair(w.x), pair(w.y), pair(w.z), pair(w.w)); };
#pragma unroll
        for (int j = 0; j < kHeld; ++j) {
            const int i = threadIdx.x + j * kThreads;
            if (i < n)
                put(i, held[j]);
        }
        for (int i = threadIdx.x + kHeld * kThreads; i < n; i += kThreads)
            put(i, x[i]);
        if (threadIdx.x == 0)
            a.x_scale[cta] = power(-k);
    } else if (cta < a.x_ctas + a.row_ctas) {
        /* a warp a row of W: its largest finite absmax */
        const int n = (cta - a.x_ctas) * (kThreads / 32) + warp, blocks = a.K / 64;
        if (n >= a.N)
            return;
        uint32_t top = 0;
        for (int i = lane; i < blocks; i += 32)
            top = max(top, finite_bits(a.absmax[(int64_t)n * blocks + i]));
        top = __reduce_max_sync(0xFFFFFFFFu, top);
        if (lane == 0)
            a.row_scale[n] = row_power(top);
    } else {
        for (int i = threadIdx.x; i < a.n_counts; i += kThreads)
            a.counts[i] = 0;
    }
}

/* W in FP16, its rows multiplied by their powers of two, for calls of many rows: a warp a row of W, which first takes
 * the row's largest absmax; the codebook lies in shared memory once for each lane, so a lookup meets no conflict and
 * its address is one byte permute.  Memory bounds it: 2 x 14336 x 4096 64 us, 5.6 TB/s; two or eight loads of a plane
 * under way in place of four, or two CTAs of 768 threads, 63 to 67. */
constexpr int kExpandThreads = 512, kExpandCtas = 3 /* an SM */, kExpandAtOnce = 4, kLutBytes = 256 * 256;
__global__ void __launch_bounds__(kExpandThreads, kExpandCtas)
    gated_expand_kernel(const uint8_t *hole, const uint8_t *plug, const float *absmax, uint4 *out, float *row_scale, int N,
                        int K)
{
    extern __shared__ __align__(16) float lut[];
    for (int i = threadIdx.x; i < 256 * 32; i += kExpandThreads)
        lut[(i >> 5) * 64 + (i & 31)] = (&g_cells[0][0])[i >> 5];
    __syncthreads();
    const int warp = threadIdx.x / 32, lane = threadIdx.x & 31, blocks = K / 64, words = K / 8;
    const uint32_t base = saddr(lut), lane4 = (uint32_t)lane * 4u;
    for (int n = blockIdx.x * (kExpandThreads / 32) + warp; n < N; n += gridDim.x * (kExpandThreads / 32)) {
        const uint32_t *H = reinterpret_cast<const uint32_t *>(hole) + (int64_t)n * words;
        const uint32_t *P = reinterpret_cast<const uint32_t *>(plug) + (int64_t)n * words;
        const float *am = absmax + (int64_t)n * blocks;
        uint4 *o = out + (int64_t)n * words;
        uint32_t h[kExpandAtOnce], p[kExpandAtOnce];
        auto load = [&](int i0) {
#pragma unroll
            for (int j = 0; j < kExpandAtOnce; ++j) {
                const int i = min(i0 + j * 32, words - 1);
                h[j] = __ldcs(H + i), p[j] = __ldcs(P + i);
            }
        };
        load(lane);
        uint32_t top = 0;
        for (int i = lane; i < blocks; i += 32)
            top = max(top, finite_bits(__ldg(am + i)));
        const float scale = row_power(__reduce_max_sync(0xFFFFFFFFu, top));
        if (lane == 0)
            row_scale[n] = scale;
        for (int i0 = lane; i0 < words; i0 += kExpandAtOnce * 32) {
            if (i0 != lane)
                load(i0);
#pragma unroll
            for (int j = 0; j < kExpandAtOnce; ++j) {
                const int i = i0 + j * 32;
                if (i >= words)
                    break;
                const float s = __ldg(am + i / 8) * scale;
                const uint32_t E = ((h[j] << 4) & 0xF0F0F0F0u) | (p[j] & 0x0F0F0F0Fu);
                const uint32_t O = (h[j] & 0xF0F0F0F0u) | ((p[j] >> 4) & 0x0F0F0F0Fu);
                uint32_t w[4];
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    const float c0 = __uint_as_float(lds32(base + __byte_perm(E, lane4, 0x5504u | (b << 4))));
                    const float c1 = __uint_as_float(lds32(base + __byte_perm(O, lane4, 0x5504u | (b << 4))));
                    const __half2 v = __floats2half2_rn(c0 * s, c1 * s);
                    w[b] = *reinterpret_cast<const uint32_t *>(&v);
                }
                o[i] = make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
    }
    asm volatile("griddepcontrol.wait;" ::: "memory"); /* whoever follows this kernel follows gated_prep_kernel too */
}

/* kOk, or what glint_htile_gated_stream returns for these arguments before it looks at pointers */
int check(const GlintHtileGated *a)
{
    if (!a || a->M < 0 || a->F < 0 || a->K < 0 || a->F > INT32_MAX / 2 ||
        (a->mode != GLINT_HTILE_PRECISE && a->mode != GLINT_HTILE_FAST) ||
        (a->act != GLINT_ACT_SILU && a->act != GLINT_ACT_GELU_TANH))
        return kBadArg;
    if (a->blocksize <= 0)
        return kBadBlocksize;
    return kOk;
}
/* the shapes that the kernels on TMA take, at any M */
bool streams(const GlintHtileGated &a)
{
    return htile_decode_supported(a.hole, a.plug, a.absmax, a.x, std::min(a.M, 32), 2 * a.F, a.K, a.blocksize);
}

/* what lies where in the workspace */
struct Layout {
    bool half = false; /* x in FP16 */
    bool wide = false; /* W in FP16 */
    int64_t x16 = 0, w16 = 0, x_scale = 0, row_scale = 0, sums = 0, counts = 0, n_counts = 0, bytes = 0; /* -1: unknown */
    explicit Layout(const GlintHtileGated &a)
    {
        const int N = 2 * a.F;
        const bool decode = a.M <= kDecodeM;
        half = a.mode == GLINT_HTILE_FAST;
        wide = half && htile_gated_wide_takes(a.M, N);
        auto take = [&](int64_t n) {
            const int64_t at = bytes;
            bytes += (n + 255) / 256 * 256;
            return at;
        };
        if (half) {
            x16 = take((int64_t)a.M * a.K * 2);
            x_scale = take(((int64_t)a.M + 255) / 256 * 256 * 4); /* whole tiles of rows are read */
            if (!decode)
                row_scale = take((int64_t)N * 4);
            if (wide)
                w16 = take((int64_t)N * a.K * 2);
        }
        const int64_t s = decode ? htile_decode_gated_work(a.M, N, a.K, &n_counts)
                          : wide ? htile_gated_wide_work(a.M, N, a.K)
                          : half ? htile_gemm_gated_work(a.M, N, a.K, &n_counts)
                                 : 0;
        if (s < 0) {
            bytes = -1;
            return;
        }
        sums = take(s), counts = take(n_counts * (int64_t)sizeof(int));
    }
};

/* a kernel that may start while the one before it runs */
template <typename... P, typename... A>
bool launch_early(void (*kernel)(P...), int ctas, int threads, int smem, cudaStream_t stream, A... args)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas), cfg.blockDim = dim3(threads), cfg.dynamicSmemBytes = smem, cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr, cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, kernel, P(args)...) == cudaSuccess)
        return true;
    cudaGetLastError();
    return false;
}

} // namespace
} // namespace glint

using namespace glint;

int64_t glint_htile_gated_work_bytes(const GlintHtileGated *a)
{
    if (check(a) != kOk)
        return kBadArg;
    if (a->M == 0 || a->F == 0 || a->K == 0 || !streams(*a))
        return 0;
    return Layout(*a).bytes;
}

int glint_htile_gated_stream(const GlintHtileGated *a, cudaStream_t stream)
{
    const int rc = check(a);
    if (rc != kOk)
        return rc;
    if (a->M == 0 || a->F == 0)
        return kOk;
    if (!a->h || (a->K && (!a->hole || !a->plug || !a->absmax || !a->x)))
        return kBadArg;
    if (a->K == 0)
        return cudaMemsetAsync(a->h, 0, (size_t)a->M * a->F * 2, stream) == cudaSuccess ? kOk : kLaunch;
    const int N = 2 * a->F;
    if (!streams(*a))
        return htile_gemv_gated_launch(a->hole, a->plug, a->absmax, a->x, a->h, a->M, N, a->K, a->blocksize, a->act,
                                       stream);
    const Layout at(*a);
    if (at.bytes < 0)
        return kLaunch;
    if (at.bytes > 0 && (!a->work || !aligned_to(a->work, 16)))
        return kBadArg;
    char *work = static_cast<char *>(a->work);
    const bool decode = a->M <= kDecodeM;
    float *x_scale = reinterpret_cast<float *>(work + at.x_scale);
    float *row_scale = reinterpret_cast<float *>(work + at.row_scale);
    int *counts = reinterpret_cast<int *>(work + at.counts);
    if (at.half || at.n_counts) {
        PrepArgs p{a->x, reinterpret_cast<__half *>(work + at.x16), x_scale, a->absmax, row_scale, counts, a->M, N, a->K, 0, 0,
                   (int)at.n_counts, at.wide};
        if (at.half)
            p.x_ctas = a->M, p.row_ctas = decode || at.wide ? 0 : (N + kThreads / 32 - 1) / (kThreads / 32);
        if (!launch_early(gated_prep_kernel, p.x_ctas + p.row_ctas + (at.n_counts ? 1 : 0), kThreads, 0, stream, p))
            return kLaunch;
    }
    const HtileMode mode = at.half ? kFast : kPrecise;
    /* FP16 in BF16's place: the kernels know by the mode */
    const glint_bf16_t *x = at.half ? reinterpret_cast<const glint_bf16_t *>(work + at.x16) : a->x;
    const GatedEpilogue ep{a->act, at.half ? x_scale : nullptr, at.half && !decode ? row_scale : nullptr};
    float *sums = reinterpret_cast<float *>(work + at.sums);
    if (at.wide) {
        if (!ensure_smem((const void *)gated_expand_kernel, kLutBytes))
            return kLaunch;
        const int ctas = std::min(kExpandCtas * sm_count(), (N + kExpandThreads / 32 - 1) / (kExpandThreads / 32));
        if (!launch_early(gated_expand_kernel, ctas, kExpandThreads, kLutBytes, stream, a->hole, a->plug, a->absmax,
                          reinterpret_cast<uint4 *>(work + at.w16), row_scale, N, a->K))
            return kLaunch;
        return htile_gated_wide_launch(work + at.w16, x, a->h, sums, a->M, N, a->K, ep, stream);
    }
    const auto launch = decode ? htile_decode_gated_launch : htile_gemm_gated_launch;
    return launch(a->hole, a->plug, a->absmax, x, a->h, sums, counts, a->M, N, a->K, mode, ep, stream);
}
