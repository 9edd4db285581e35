/* Causal attention over packed prompts with grouped heads, on tcgen05.
 *
 * A CTA takes two tiles of up to 128 query rows of one sequence and one kv head: rows
 * are (token, query head of the group) pairs, group * (128 / group) of them, so the
 * group's heads share every K and V tile that is loaded.  Per tile of 128 keys
 *
 *   S = Q K^T          UMMA 128 x 128 x D, Q and K in shared memory (TMA, 128-byte swizzle)
 *   P = 2^(S c - m)    a thread per row: S from TMEM, running maximum m and sum l in f32,
 *                      P as BF16 back into S's columns (2^-8 of each weight at most, the
 *                      rounding that the tensor cores' operand asks for)
 *   O += P V           UMMA 128 x D x 128, P from TMEM, V as it lies (inner index = key rows)
 *
 * Where the weights are many, their roundings cancel; a row of few keys, or of a few that
 * carry most of it, would show them.  So a tile of keys in which some row has a weight
 * above 1/16 of its running sum also gets what the rounding dropped, as a second BF16
 * operand (a sequence's first tile nearly always, later ones as peaked as they are).
 *
 * The two tiles take turns: while one's softmax runs, the tensor cores work on the
 * other.  m may lag behind the true maximum by 2^8, so O is rescaled rarely.  Few blocks
 * with many keys are cut along the keys and joined by a second kernel.
 *
 * Masked scores are replaced, never added to, and a masked weight is 0; a NaN or an
 * infinity in V would still reach other rows as 0 * NaN, so tiles with masked places
 * are looked through and such values taken out of shared memory.  Rows that do see one
 * get it afterwards: o of a column is then known without a product.  So it is with an
 * infinity among other tiles' values, whose products make a NaN of it wherever a weight
 * or the half that BF16 drops is 0 or negative: rows that come out not finite are looked at.
 *
 * Floor: exponentials (16 a clock and SM) and the tensor cores take the same time at
 * D = 128, 2048 clocks for two tiles of queries by one of keys.  Bound: a tile's softmax
 * (about 2150 clocks) and its UMMA round trip (1870) follow on one another, and only two
 * tiles alternate (TMEM holds two S and two O); tensor pipe 55 %, exponentials 52 % busy.
 * 8192 tokens, 32 / 8 heads of 128: 502 us, 1095 TFLOP/s (a tile pair per CTA launch in
 * place of persistent CTAs: 578).  16384: 2116 us, 1039.  Twelve prompts of up to 2011: 112.
 * 512 after 7777, 16 / 4 heads of 64: 54.  17 tokens: 11, latency.
 * A value that is not finite, seen or not, costs the blocks that meet it a pass over their
 * V: 100 queries over 20000 keys 77 -> 330 to 360 us, 4096 tokens 83 -> 130 to 170.
 */
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "../../include/glint_attn.h"
#include "common.cuh"
#include "glint_internal.h"
#include "item_loop.h"
#include "ptx.cuh"

namespace glint {
static __device__ int g_attn_error = 0, g_attn_error_taken = 0;
int attn_error_word(bool clear) { return read_error_word(g_attn_error, g_attn_error_taken, clear); }

namespace {

constexpr int kWarps = 4; /* of the plain kernel */

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

/* one query row by one warp, in f32: right for any stride, alignment and scale; some 200 clocks
 * a key (2048 tokens, 32 / 8 heads of 128: 8.4 ms, where the tensor-core kernel takes 0.08) */
template <int D>
__device__ __forceinline__ void plain_row(const GlintAttnPrompt &a, const Span &s, int t, int hq, int lane)
{
    const int h = hq / (a.heads / a.kv_heads);
    const int seen = a.causal ? min(s.k1 - s.k0, t - s.q0 + 1 + (s.k1 - s.k0) - (s.q1 - s.q0)) : s.k1 - s.k0;
    float q[D / 32], o[D / 32] = {}, m = -INFINITY, l = 0.f;
    float odd[D / 32] = {}; /* infinities and NaN among the values seen, added up: a weight may be 0 in f32 */
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
        for (int i = 0; i < D / 32; ++i) {
            const float y = __bfloat162float(v[32 * i]);
            const bool finite = fabsf(y) < INFINITY;
            o[i] = fmaf(p, finite ? y : 0.f, o[i] * keep);
            odd[i] += finite ? 0.f : y;
        }
        m = top;
    }
    const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
        a.o[t * a.o_tok + hq * a.o_head + lane + 32 * i] = __float2bfloat16_rn(l > 0.f && !(odd[i] == 0.f) ? odd[i] : o[i] * inv);
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


/* ---- tensor-core kernel ------------------------------------------------------------ */
constexpr int kRows = 128, kKeys = 128;
constexpr float kLazy = 8.f;   /* the running maximum may lag by 2^8 */
constexpr float kHeavy = 15.f; /* a weight above 1 / (1 + kHeavy) of the running sum keeps its low half */
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

template <int D>
struct Cfg {
    static constexpr int kTileBytes = kKeys * D * 2;
    static constexpr int kStages = D == 128 ? 2 : 4; /* of V and the K after it */
    static constexpr int kSmem = 1024 + 2 * kTileBytes + 2 * kStages * kTileBytes + 256;
    /* TMEM columns: S of tile i at 128 i, O at 256 + D i.  In S's place, for 32 keys a
     * time, 16 columns of P and 16 of what P's rounding dropped. */
    static constexpr uint32_t kS = 0, kO = 256;
};
/* warps 0-3, 4-7: softmax of the two tiles; 8: loads; 9: UMMA, the two tiles in turn (one
 * thread each let them fall into step, both in softmax and then both in UMMA: 1.3 times
 * the time; two threads a row of softmax: as fast over 16384 keys, 4 % slower over fewer) */
constexpr int kLoadWarp = 8, kMmaWarp = 9, kThreads = 320;
constexpr int kSlotRows = 2 * kRows;

struct Args {
    GlintAttnPrompt a;
    int group, tok;    /* query heads a kv head; tokens a tile */
    int sms;
    bool vec;          /* o takes 16-byte stores */
    bool split;        /* there is a workspace for parts */
    float *part;       /* [slot][2 tiles][D / 4][128 rows] of 4, then m, l [slot][256] each, then bad [slot][2] */
};
struct Maps {
    CUtensorMap q, k, v;
};

__device__ __forceinline__ float ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void umma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool acc)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
                 "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)acc)
                 : "memory");
}
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool acc)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
                 "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)acc)
                 : "memory");
}
/* the same, added to D, but to none of the lanes whose bit in `off` is set */
__device__ __forceinline__ void umma_ts_lanes(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, const uint32_t (&off)[4])
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.eq.b32 p, 0, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%4, %5, %6, %7}, p;\n\t}\n" ::"r"(d),
                 "r"(a), "l"(b), "r"(idesc), "r"(off[0]), "r"(off[1]), "r"(off[2]), "r"(off[3])
                 : "memory");
}
__device__ __forceinline__ void umma_commit(uint64_t *bar)
{
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(saddr(bar))
                 : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t *r)
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
                 "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
                 "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]),
                   "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]),
                   "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]),
                   "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(taddr));
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t *r)
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
                 "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
                 "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
                 "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
                 : "memory");
}
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t *r)
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];\n\t"
                 "tcgen05.wait::ld.sync.aligned;"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr)
                 : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t *r)
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]),
                 "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}
/* the loads into r have arrived: its values are this statement's, so no use moves ahead of it */
__device__ __forceinline__ void tmem_ld_wait(uint32_t *r)
{
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]),
                   "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]),
                   "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]),
                   "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
                 :
                 : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

/* UMMA shared-memory descriptors, 128-byte swizzle, version 1.  Inner index contiguous
 * (Q, K): 8-row atoms of 1024 B.  Outer index contiguous (V: 64 of D by 8 keys an atom):
 * the next 64 of D lie a box of 128 keys further, the next 8 keys 1024 B further. */
__device__ __forceinline__ uint64_t desc_base(uint32_t sa)
{
    return (uint64_t)((sa >> 4) & 0x3FFF) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
__device__ __forceinline__ uint64_t desc_inner(uint32_t sa) { return desc_base(sa) | ((uint64_t)1 << 16); }
__device__ __forceinline__ uint64_t desc_outer(uint32_t sa)
{
    return desc_base(sa) | ((uint64_t)(kKeys * 128 >> 4) << 16);
}
/* f32 accumulate, BF16 A and B, M = 128; bit 16: B has its outer index contiguous */
constexpr uint32_t idesc_of(int n, bool outer_b)
{
    return (1u << 4) | (1u << 7) | (1u << 10) | (outer_b ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | (8u << 24);
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
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c)
{
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b)
{
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

/* The blocks (two tiles of one sequence) of all sequences in one row, each with every kv
 * head, those that see the most keys first, so that the CTAs, which take them in turn,
 * end together (12 prompts of 1 to 2011 tokens in their own order: 133 us).  A block's
 * cost is its level: its number in the sequence, plus the blocks of keys before it.
 * Where there are at most half as many items as SMs, the keys of each are cut into parts
 * of kCut tiles or more (a part costs its block's rows in f32, written and read: 130 KB
 * each way). */
constexpr int kCut = 4, kMostCuts = 32; /* a warp's lanes join them */
constexpr int kSeqsHeld = 1024; /* sequences whose blocks and levels a CTA keeps in shared memory */
struct Seq {
    int blocks, level; /* level of the first block; of every block where all keys are seen */
};
struct Item {
    Span s;
    int block, head, cut, cuts, slot;
    int t0, first, last0, last1; /* first token; query tile i goes through the tiles of keys [first, lasti) */
};
__device__ __forceinline__ Seq seq_of(const Args &g, int seq)
{
    const int n = max(0, bound(g.a.cu_q, seq + 1, g.a.q_tokens) - bound(g.a.cu_q, seq, g.a.q_tokens));
    const int keys = max(0, bound(g.a.cu_k, seq + 1, g.a.k_tokens) - bound(g.a.cu_k, seq, g.a.k_tokens));
    return Seq{(n + 2 * g.tok - 1) / (2 * g.tok), (g.a.causal ? max(0, keys - n) : keys) / (2 * g.tok)};
}
__device__ __forceinline__ int seen_of(const Args &g, const Span &s, int t);
/* tiles of keys that an item's two query tiles see */
__device__ __forceinline__ void tiles_of(const Args &g, const Item &it, int (&n)[2])
{
    const int t0 = it.s.q0 + it.block * 2 * g.tok;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int end = min(it.s.q1, t0 + (i + 1) * g.tok); /* one past the tile's last token */
        n[i] = end > t0 + i * g.tok ? (seen_of(g, it.s, end - 1) + kKeys - 1) / kKeys : 0;
    }
}
/* item `index` (or, with `whole`, the first part of the index-th item before its keys are
 * cut), by the whole warp; false past the last one.  held: the first kSeqsHeld sequences' seq_of */
__device__ __forceinline__ bool item_of(const Args &g, const Seq *held, int index, bool whole, Item &it)
{
    const int lane = threadIdx.x & 31;
    auto seq = [&](int b) { return b >= g.a.seqs ? Seq{0, 0} : b < kSeqsHeld ? held[b] : seq_of(g, b); };
    /* of a sequence's blocks, those of this level or above */
    auto above = [&](Seq q, int level) {
        return g.a.causal ? min(q.blocks, max(0, q.blocks + q.level - level)) : q.level >= level ? q.blocks : 0;
    };
    int blocks = 0, top = 0;
    for (int b = lane; b < g.a.seqs; b += 32) {
        const Seq q = seq(b);
        blocks += q.blocks, top = max(top, q.blocks + q.level);
    }
    blocks = __reduce_add_sync(0xFFFFFFFFu, blocks), top = __reduce_max_sync(0xFFFFFFFFu, top);
    const int64_t items = (int64_t)blocks * g.a.kv_heads;
    const int cuts = g.split && items > 0 ? (int)min((int64_t)kMostCuts, max((int64_t)1, g.sms / items)) : 1;
    if (whole ? index >= items : index >= items * cuts)
        return false;
    index *= whole ? cuts : 1;
    it.slot = index, it.cut = index % cuts, it.cuts = cuts;
    const int rest = index / cuts, want = rest / g.a.kv_heads;
    it.head = rest - want * g.a.kv_heads;
    /* the level it is in: the highest with more than `want` blocks at or above it */
    int lo = 0, hi = top;
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        int n = 0;
        for (int b = lane; b < g.a.seqs; b += 32)
            n += above(seq(b), mid);
        if (__reduce_add_sync(0xFFFFFFFFu, n) > want)
            lo = mid;
        else
            hi = mid - 1;
    }
    int n = 0;
    for (int b = lane; b < g.a.seqs; b += 32)
        n += above(seq(b), lo + 1);
    int left = want - __reduce_add_sync(0xFFFFFFFFu, n); /* its number among the blocks of this level */
    for (int b0 = 0; b0 < g.a.seqs; b0 += 32) {
        const Seq q = seq(b0 + lane);
        const int here = above(q, lo) - above(q, lo + 1);
        int sum = here;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int o = __shfl_up_sync(0xFFFFFFFFu, sum, off);
            if (lane >= off)
                sum += o;
        }
        const uint32_t past = __ballot_sync(0xFFFFFFFFu, sum > left);
        if (past) {
            const int l = __ffs(past) - 1, b = b0 + l;
            const int first = __shfl_sync(0xFFFFFFFFu, sum - here, l), level = __shfl_sync(0xFFFFFFFFu, q.level, l);
            it.block = g.a.causal ? lo - level : left - first;
            it.s.q0 = bound(g.a.cu_q, b, g.a.q_tokens), it.s.q1 = bound(g.a.cu_q, b + 1, g.a.q_tokens);
            it.s.k0 = bound(g.a.cu_k, b, g.a.k_tokens);
            it.s.k1 = max(it.s.k0, bound(g.a.cu_k, b + 1, g.a.k_tokens));
            int tiles[2];
            tiles_of(g, it, tiles);
            it.cuts = min(cuts, max(1, max(tiles[0], tiles[1]) / kCut));
            return true;
        }
        left -= __shfl_sync(0xFFFFFFFFu, sum, 31);
    }
    return false;
}
/* keys that query token t of the item's sequence sees */
__device__ __forceinline__ int seen_of(const Args &g, const Span &s, int t)
{
    const int keys = s.k1 - s.k0;
    return g.a.causal ? min(keys, max(0, t - s.q0 + 1 + keys - (s.q1 - s.q0))) : keys;
}
/* first tile of a cut, of n tiles */
__device__ __forceinline__ int cut_begin(int n, int cut, int cuts) { return (int)((int64_t)n * cut / cuts); }

/* any NaN or infinity among two BF16 */
__device__ __forceinline__ uint32_t odd2(uint32_t w) { return ((w & 0x7F807F80u) + 0x00800080u) & 0x80008000u; }
/* acc + 0 * w, BF16 pairs: NaN from the first of them on */
__device__ __forceinline__ uint32_t add_times0(uint32_t w, uint32_t acc)
{
    asm("fma.rn.bf16x2 %0, %1, %2, %0;" : "+r"(acc) : "r"(w), "r"(0u));
    return acc;
}
/* two BF16, 0 in place of such a one */
__device__ __forceinline__ uint32_t without_odd2(uint32_t w) { return w & ~((odd2(w) >> 15) * 0xFFFFu); }

/* V's first keys of a column with a NaN, +infinity and -infinity, of the first n keys of a
 * sequence: at[kind * D + column], n and more for none.  By `threads` threads, with `sync` their
 * barrier; V as the tensor-core kernel takes it (16-byte loads). */
template <int D, class Sync>
__device__ __noinline__ void first_odd(const GlintAttnPrompt &a, const Span &s, int head, int n, int *at, int tid,
                                       int threads, Sync sync)
{
    for (int e = tid; e < 3 * D; e += threads)
        at[e] = INT32_MAX;
    sync();
    constexpr int C = D / 8; /* 16 bytes of a row */
    const __nv_bfloat16 *v = a.v + (int64_t)s.k0 * a.v_tok + head * a.v_head + tid % C * 8;
    const int step = threads / C;
    constexpr int N = 8; /* loads under way */
    for (int j0 = tid / C; j0 < n; j0 += N * step) {
        uint4 w[N];
#pragma unroll
        for (int q = 0; q < N; ++q) /* of the last key again, past it */
            w[q] = __ldg(reinterpret_cast<const uint4 *>(v + min(j0 + q * step, n - 1) * a.v_tok));
#pragma unroll
        for (int q = 0; q < N; ++q) {
            if (odd2(w[q].x) | odd2(w[q].y) | odd2(w[q].z) | odd2(w[q].w)) {
                const uint32_t x[4] = {w[q].x, w[q].y, w[q].z, w[q].w};
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const uint32_t b = x[e / 2] >> (16 * (e % 2)) & 0xFFFFu;
                    if ((b & 0x7F80u) == 0x7F80u)
                        atomicMin(at + (b & 0x7Fu ? 0 : b & 0x8000u ? 2 * D : D) + tid % C * 8 + e, min(j0 + q * step, n - 1));
                }
            }
        }
    }
    sync();
}
/* what column d of a row that sees `seen` keys is by them: NaN, an infinity, or (0) its sum */
template <int D>
__device__ __forceinline__ float odd_value(const int *at, int d, int seen)
{
    const bool up = at[D + d] < seen, down = at[2 * D + d] < seen;
    return at[d] < seen || (up && down) ? __int_as_float(0x7FFFFFFF) : up ? INFINITY : down ? -INFINITY : 0.f;
}

__device__ __forceinline__ float max_nan(float a, float b)
{
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float max3_nan(float a, uint32_t b, uint32_t c)
{
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(__uint_as_float(b)), "f"(__uint_as_float(c)));
    return r;
}
/* whether any of a tile's 128 softmax threads has `p` */
__device__ __forceinline__ bool any_of_tile(int i, bool p)
{
    uint32_t r;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\t"
                 "barrier.cta.red.or.pred q, %2, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}\n"
                 : "=r"(r)
                 : "r"((uint32_t)p), "r"(1 + i)
                 : "memory");
    return r != 0;
}

/* One CTA an SM for all items: barriers and TMEM are set up once, and while a tile's
 * softmax warps write one item's rows, the next item's loads and first products run.
 * K of the tiles of keys, and V of them, stand in rings that run on from item to item. */
template <int D>
__global__ void __launch_bounds__(kThreads, 1) attn_kernel(const __grid_constant__ Args g, const __grid_constant__ Maps maps)
{
    using C = Cfg<D>;
    extern __shared__ uint8_t raw[];
    uint8_t *smem = raw + ((1024 - (saddr(raw) & 1023)) & 1023);
    uint8_t *sq = smem, *sk = sq + 2 * C::kTileBytes, *sv = sk + C::kStages * C::kTileBytes;
    uint64_t *bars = reinterpret_cast<uint64_t *>(sv + C::kStages * C::kTileBytes);
    /* q_full: an item's Q and first K; kv_full[p]: V of the tile at ring place p and K of the next one */
    uint64_t *q_full = bars, *q_empty = bars + 1, *item_full = bars + 2, *item_empty = bars + 4, *s_full = bars + 6,
             *p_full = bars + 8, *o_done = bars + 10, *kv_full = bars + 12, *k_empty = kv_full + C::kStages,
             *v_empty = k_empty + C::kStages, *drained = v_empty + C::kStages;
    __shared__ uint32_t tmem_slot;
    /* Of four items: item k is published once all warps have begun item k - 2, so a place is filled
     * again after both tiles are done with its item, however far one is ahead of the other; an
     * item's fields are read again where they are needed, not held in registers. */
    __shared__ Item s_item[4];
    __shared__ int s_more[4];
    __shared__ Seq s_seqs[kSeqsHeld];
    __shared__ __align__(4) uint8_t s_low[2][4]; /* per tile and softmax warp: P has a low half */
    __shared__ int s_odd[4][2]; /* and per tile: odd values that a row of it sees were taken out of V */
    __shared__ uint4 s_stage[8][32 * 4]; /* per softmax warp: 32 rows of 32 BF16 */
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (warp == kLoadWarp && lane == 0) {
        mbar_init(q_full, 1), mbar_init(q_empty, 1), mbar_init(drained, 1);
        for (int i = 0; i < C::kStages; ++i)
            mbar_init(kv_full + i, 1), mbar_init(k_empty + i, 1), mbar_init(v_empty + i, 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(item_full + i, 1), mbar_init(item_empty + i, 9); /* eight softmax warps and the UMMA one */
            mbar_init(s_full + i, 1), mbar_init(o_done + i, 1), mbar_init(p_full + i, 4);
        }
        mbar_init_fence();
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(saddr(&tmem_slot)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_before();
    __syncthreads();
    tc_after();
    const uint32_t tmem = tmem_slot;
    asm volatile("griddepcontrol.launch_dependents;");
    bool alive = true;
    auto wait = [&](uint64_t *bar, uint32_t parity) {
        if (alive)
            alive = mbar_wait_suspend_bounded(bar, parity, &g_attn_error);
        return alive;
    };
    auto warp_wait = [&](uint64_t *bar, uint32_t parity) { /* a warp goes on, or gives up, as one */
        alive = __all_sync(0xFFFFFFFFu, wait(bar, parity));
    };

    if (warp == kLoadWarp) {
        /* ---- items and loads */
        for (int b = lane; b < min(kSeqsHeld, g.a.seqs); b += 32)
            s_seqs[b] = seq_of(g, b);
        __syncwarp();
        int place = 0, items = 0, queries = 0; /* ring place; items published; of them with tiles */
        for (int round = 0;; ++round) {
            /* every other round in reverse: the items fall in cost, and the CTAs take turns at the dear end */
            Item it;
            const int index = round * (int)gridDim.x + (round & 1 ? (int)gridDim.x - 1 - (int)blockIdx.x : (int)blockIdx.x);
            const bool more = item_of(g, s_seqs, index, false, it);
            if (more && it.cut >= it.cuts)
                continue;
            if (lane == 0) {
                if (more) {
                    it.t0 = it.s.q0 + it.block * 2 * g.tok;
                    int n[2];
                    tiles_of(g, it, n);
                    const int most = max(n[0], n[1]), stop = cut_begin(most, it.cut + 1, it.cuts);
                    it.first = cut_begin(most, it.cut, it.cuts);
                    it.last0 = max(it.first, min(n[0], stop)), it.last1 = max(it.first, min(n[1], stop));
                }
                wait(item_empty + (items & 1), (items / 2 + 1) & 1); /* first uses return at once */
                s_more[items & 3] = more && alive, s_item[items & 3] = it;
                s_odd[items & 3][0] = s_odd[items & 3][1] = 0;
                mbar_arrive(item_full + (items & 1));
                const int total = more ? max(it.last0, it.last1) - it.first : 0;
                if (total > 0 && wait(q_empty, (queries + 1) & 1)) {
                    auto load = [&](uint8_t *to, const CUtensorMap *map, uint64_t *bar, int j) {
                        for (int d = 0; d < D / 64; ++d)
                            tma_load_3d(to + d * kKeys * 128, map, bar, d * 64, it.head, it.s.k0 + j * kKeys);
                    };
                    /* K at ring place p: free once K at p - kStages has been used */
                    auto k_free = [&](int p) { return wait(k_empty + p % C::kStages, (p / C::kStages + 1) & 1); };
                    if (k_free(place)) {
                        mbar_expect_tx(q_full, 2 * (D / 64) * g.group * g.tok * 128 + C::kTileBytes);
                        for (int i = 0; i < 2; ++i)
                            for (int d = 0; d < D / 64; ++d)
                                tma_load_3d(sq + i * C::kTileBytes + d * kRows * 128, &maps.q, q_full, d * 64,
                                            it.head * g.group, it.t0 + i * g.tok);
                        load(sk + place % C::kStages * C::kTileBytes, &maps.k, q_full, it.first);
                        ++queries;
                        for (int c = 0; c < total; ++c, ++place) {
                            const int st = place % C::kStages;
                            const bool next = c + 1 < total;
                            if (!wait(v_empty + st, (place / C::kStages + 1) & 1) || (next && !k_free(place + 1)))
                                break;
                            mbar_expect_tx(kv_full + st, (next ? 2 : 1) * C::kTileBytes);
                            load(sv + st * C::kTileBytes, &maps.v, kv_full + st, it.first + c);
                            if (next)
                                load(sk + (place + 1) % C::kStages * C::kTileBytes, &maps.k, kv_full + st, it.first + c + 1);
                        }
                    }
                }
            }
            ++items;
            alive = __shfl_sync(0xFFFFFFFFu, alive, 0);
            if (!more || !alive)
                break;
        }
        if (lane == 0 && !alive) { /* let the copies already started land before the CTA exits */
            if (queries)
                mbar_wait_bounded(q_full, (queries - 1) & 1, &g_attn_error);
            for (int p = max(0, place - C::kStages); p < place; ++p)
                mbar_wait_bounded(kv_full + p % C::kStages, (p / C::kStages) & 1, &g_attn_error);
        }
        __syncwarp();
    } else if (warp == kMmaWarp) {
        /* ---- UMMA */
        if (lane == 0) {
            constexpr uint32_t kQk = idesc_of(kKeys, false), kPv = idesc_of(D, true);
            /* descriptors of one operand differ in their addresses alone (in 16 bytes, with no
             * carry out of the field), so each is a base and a constant: the thread has about
             * 60 clocks to make the next product's */
            const uint64_t dq = desc_inner(saddr(sq)), dk = desc_inner(saddr(sk)), dv = desc_outer(saddr(sv));
            auto scores = [&](int i, int st) { /* S_i = Q_i K^T */
                const uint64_t a = dq + (uint32_t)(i * (C::kTileBytes >> 4)), b = dk + (uint32_t)(st * (C::kTileBytes >> 4));
                const uint32_t to = tmem + C::kS + 128 * i;
#pragma unroll
                for (int d = 0; d < D / 16; ++d) {
                    const uint32_t off = ((d / 4) * kKeys * 128 + (d % 4) * 32) >> 4;
                    umma_ss(to, a + off, b + off, kQk, d > 0);
                }
                umma_commit(s_full + i);
            };
            int place = 0, queries = 0;
            uint32_t done = 0; /* bit i: parity of the tiles of keys that query tile i is through */
            for (int items = 0; wait(item_full + (items & 1), (items / 2) & 1); ++items) {
                const bool more = s_more[items & 3];
                const int first = s_item[items & 3].first;
                const int n0 = s_item[items & 3].last0 - first, n1 = s_item[items & 3].last1 - first;
                mbar_arrive(item_empty + (items & 1));
                if (!more)
                    break;
                const int total = max(n0, n1);
                if (total == 0)
                    continue;
                if (!wait(q_full, queries & 1))
                    break;
                ++queries;
                tc_after();
                for (int i = 0; i < 2; ++i)
                    if ((i ? n1 : n0) > 0)
                        scores(i, place % C::kStages);
                umma_commit(k_empty + place % C::kStages);
                if (total == 1)
                    umma_commit(q_empty);
                for (int c = 0; c < total && alive; ++c, ++place) {
                    const int st = place % C::kStages, nst = (place + 1) % C::kStages;
                    wait(kv_full + st, (place / C::kStages) & 1);
                    for (int i = 0; i < 2 && alive; ++i) {
                        const int n = i ? n1 : n0;
                        if (c >= n || !wait(p_full + i, (done >> i) & 1u))
                            continue;
                        done ^= 1u << i;
                        tc_after();
                        /* 16 keys a product: P_i in TMEM, V in shared memory */
                        const uint32_t to = tmem + C::kO + D * i, from = tmem + C::kS + 128 * i;
                        const uint64_t v = dv + (uint32_t)(st * (C::kTileBytes >> 4));
#pragma unroll
                        for (int k = 0; k < 8; ++k)
                            umma_ts(to, from + (k / 2) * 32 + (k % 2) * 8, v + k * 128, kPv, c > 0 || k > 0);
                        if (const uint32_t low = *reinterpret_cast<const volatile uint32_t *>(s_low[i])) {
                            /* the warps without one have left scores in its place */
                            const uint32_t off[4] = {low & 0xFFu ? 0u : ~0u, low & 0xFF00u ? 0u : ~0u,
                                                     low & 0xFF0000u ? 0u : ~0u, low & 0xFF000000u ? 0u : ~0u};
#pragma unroll
                            for (int k = 0; k < 8; ++k)
                                umma_ts_lanes(to, from + (k / 2) * 32 + (k % 2) * 8 + 16, v + k * 128, kPv, off);
                        }
                        umma_commit(o_done + i);
                        if (c + 1 < n)
                            scores(i, nst);
                    }
                    if (!alive)
                        break;
                    if (c + 1 < total)
                        umma_commit(k_empty + nst);
                    if (c + 2 == total)
                        umma_commit(q_empty);
                    umma_commit(v_empty + st);
                }
            }
            /* every product is done before this CTA's memory can go, after a wait that ran out too */
            umma_commit(drained);
            mbar_wait_bounded(drained, 0, &g_attn_error);
        }
        __syncwarp();
    } else {
        /* ---- softmax of tile i, row r */
        const int i = warp >> 2, wl = warp & 3, r = wl * 32 + lane;
        const uint32_t lanes = (uint32_t)(wl * 32) << 16;
        const uint32_t ts = tmem + C::kS + 128 * i + lanes, to = tmem + C::kO + D * i + lanes;
        const float scale2 = g.a.scale * kLog2e;
        uint32_t turns = 0; /* tiles of keys gone through, of all items */
        int place0 = 0;     /* ring place of the item's first */
        auto next = [&](int items) {
            warp_wait(item_full + (items & 1), (items / 2) & 1);
            return alive && s_more[items & 3];
        };
        auto any = [&](bool p) { return any_of_tile(i, p); };
        item_loop(next, any, [&](int items) {
            const Item &it = s_item[items & 3];
            __syncwarp();
            if (lane == 0)
                mbar_arrive(item_empty + (items & 1));
            const Span &s = it.s;
            const int done = (i ? it.last1 : it.last0) - it.first;
            /* Few registers live through this loop: 128 hold scores, and a spilled one would come
             * back from L2 (the tiles leave next to no L1).  None is at D = 128, two at 64. */
            int seen; /* keys this row sees, from the item's first on; 0 or less where it is no query's */
            {
                const int t = it.t0 + i * g.tok + r / g.group;
                seen = (r < g.group * g.tok && t < s.q1 ? seen_of(g, s, t) : 0) - it.first * kKeys;
            }
            /* tiles of keys from `plain` on have a place that some row does not see */
            const int plain = it.t0 + i * g.tok < s.q1 ? seen_of(g, s, it.t0 + i * g.tok) / kKeys - it.first : 0;
            float m = -INFINITY, l = 0.f; /* of the row */
#pragma unroll 1
            for (int c = 0; c < done; ++c, ++turns) {
                const bool masked = c >= plain;
                /* V's odd values would reach rows that do not see them.  The first tile that multiplies
                 * by this V takes them out for both: its weights are waited for before either product
                 * (and tile 1 has masked places in no tile of keys where tile 0 has none). */
                if (masked && (i == 0 || c >= it.last0 - it.first)) {
                    const int p = place0 + c;
                    warp_wait(kv_full + p % C::kStages, (p / C::kStages) & 1);
                    uint4 *v = reinterpret_cast<uint4 *>(sv + p % C::kStages * C::kTileBytes);
                    uint32_t zero[4] = {}; /* 0 times every value, added up */
#pragma unroll 8
                    for (int e = r; e < C::kTileBytes / 16; e += kRows) {
                        const uint4 w = v[e];
                        zero[0] = add_times0(w.x, zero[0]), zero[1] = add_times0(w.y, zero[1]);
                        zero[2] = add_times0(w.z, zero[2]), zero[3] = add_times0(w.w, zero[3]);
                    }
                    if (odd2(zero[0]) | odd2(zero[1]) | odd2(zero[2]) | odd2(zero[3])) {
                        int key = kKeys; /* the first that has one */
#pragma unroll 1
                        for (int e = r; e < C::kTileBytes / 16; e += kRows) {
                            const uint4 w = v[e];
                            if (odd2(w.x) | odd2(w.y) | odd2(w.z) | odd2(w.w)) {
                                v[e] = make_uint4(without_odd2(w.x), without_odd2(w.y), without_odd2(w.z), without_odd2(w.w));
                                key = min(key, e / 8 % kKeys);
                            }
                        }
                        fence_proxy_async_smem(); /* the products read through the asynchronous proxy */
                        for (int j = i; j < 2; ++j) /* the tiles that have a row that sees it */
                            if (c < (j ? it.last1 : it.last0) - it.first &&
                                (it.first + c) * kKeys + key < seen_of(g, s, min(s.q1, it.t0 + (j + 1) * g.tok) - 1))
                                s_odd[items & 3][j] = 1;
                    }
                }
                warp_wait(s_full + i, turns & 1);
                tc_after();
                uint32_t x[kKeys];
#pragma unroll
                for (int q = 0; q < kKeys; q += 32)
                    tmem_ld32(ts + q, x + q);
#pragma unroll
                for (int q = 0; q < kKeys; q += 32)
                    tmem_ld_wait(x + q);
                if (masked) {
                    const int lim = seen - c * kKeys;
#pragma unroll
                    for (int e = 0; e < kKeys; ++e)
                        x[e] = e < lim ? x[e] : 0xFF800000u;
                }
                float top = max3_nan(__uint_as_float(x[0]), x[1], x[2]), other = max3_nan(__uint_as_float(x[3]), x[4], x[5]);
#pragma unroll
                for (int e = 6; e < kKeys - 2; e += 4) {
                    top = max3_nan(top, x[e], x[e + 1]);
                    other = max3_nan(other, x[e + 2], x[e + 3]);
                }
                top = max3_nan(top, x[kKeys - 2], x[kKeys - 1]);
                /* rows that are no query's (of whatever lies there) take no part in what the warps decide */
                top = seen > 0 ? max_nan(top, other) * scale2 : -INFINITY;
                if (__any_sync(0xFFFFFFFFu, !(top <= m + kLazy))) { /* NaN too */
                    /* a NaN or an infinite score: every weight of the row is NaN from here on */
                    const float nm = top < INFINITY ? fmaxf(m, top) : __int_as_float(0x7FFFFFFF);
                    const float f = m == -INFINITY && nm == nm ? 0.f : ex2(m - nm);
                    m = m == m ? nm : m, l *= f;
                    if (c > 0) { /* O of the tiles before, once they are in */
                        warp_wait(o_done + i, (turns + 1) & 1);
                        tc_after();
#pragma unroll 1
                        for (int q = 0; q < D; q += 8) {
                            uint32_t o[8];
                            tmem_ld8(to + q, o);
#pragma unroll
                            for (int e = 0; e < 8; ++e)
                                o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                            tmem_st8(to + q, o);
                        }
                        tmem_st_wait();
                    }
                }
                const float less = m == -INFINITY ? 0.f : -m;
                const bool low = __any_sync(0xFFFFFFFFu, ex2(top + less) * kHeavy > l);
                if (lane == 0)
                    s_low[i][wl] = low;
                const uint64_t sc = pack2f(scale2, scale2), ls = pack2f(less, less);
                uint64_t sum = 0;
#pragma unroll
                for (int q = 0; q < kKeys / 32; ++q) {
                    uint32_t p[16];
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        uint32_t *v = x + 32 * q + 2 * e;
                        float a, b;
                        unpack2f(fma2(pack2f(__uint_as_float(v[0]), __uint_as_float(v[1])), sc, ls), a, b);
                        a = ex2(a), b = ex2(b);
                        sum = add2(sum, pack2f(a, b));
                        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
                        p[e] = *reinterpret_cast<const uint32_t *>(&h);
                        v[0] = __float_as_uint(a), v[1] = __float_as_uint(b);
                    }
                    tmem_st16(ts + 32 * q, p);
                    if (low) { /* what the rounding dropped */
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const float a = __uint_as_float(x[32 * q + 2 * e]) - __uint_as_float(p[e] << 16);
                            const float b = __uint_as_float(x[32 * q + 2 * e + 1]) - __uint_as_float(p[e] & 0xFFFF0000u);
                            const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
                            p[e] = *reinterpret_cast<const uint32_t *>(&h);
                        }
                        tmem_st16(ts + 32 * q + 16, p);
                    }
                }
                tmem_st_wait();
                tc_before();
                __syncwarp();
                if (lane == 0)
                    mbar_arrive(p_full + i);
                float a, b;
                unpack2f(sum, a, b);
                l += a + b;
            }
            place0 += max(it.last0, it.last1) - it.first;
            const int tile0 = it.t0 + i * g.tok, t = tile0 + r / g.group, hq = it.head * g.group + r % g.group;
            const bool live = r < g.group * g.tok && t < s.q1;
            if (done > 0) {
                warp_wait(o_done + i, (turns + 1) & 1);
                tc_after();
            }
            const bool odd = done > 0 && s_odd[items & 3][i];
            if (it.cuts > 1) {
                uint4 *part = reinterpret_cast<uint4 *>(g.part) + ((int64_t)it.slot * 2 + i) * (D / 4) * kRows + r;
                float *ml = g.part + (int64_t)g.sms * kSlotRows * D + (int64_t)it.slot * kSlotRows + i * kRows + r;
#pragma unroll 1
                for (int q = 0; q < D / 32; ++q) {
                    uint32_t o[32] = {};
                    if (done > 0) {
                        tmem_ld32(to + 32 * q, o);
                        tmem_ld_wait(o);
                    }
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        part[(8 * q + e) * kRows] = make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
                }
                ml[0] = m, ml[(int64_t)g.sms * kSlotRows] = l;
                if (r == 0)
                    reinterpret_cast<int *>(g.part + (int64_t)g.sms * kSlotRows * (D + 2))[2 * it.slot + i] = odd;
            } else {
                const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
                /* 32 columns a time through shared memory: a thread's own row would be a line of its
                 * own in every store, four threads a row make whole sectors (12 prompts 114 -> 112 us) */
                uint4 *stage = s_stage[warp];
                uint32_t zero[4] = {}; /* 0 times the row's values, added up */
                int64_t at[4]; /* of rows lane / 4 + 8 k, 16 bytes at lane % 4 */
                uint32_t mine = 0;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int row = wl * 32 + lane / 4 + 8 * k, tk = tile0 + row / g.group;
                    mine |= row < g.group * g.tok && tk < s.q1 ? 1u << k : 0u;
                    at[k] = tk * g.a.o_tok + (it.head * g.group + row % g.group) * g.a.o_head + lane % 4 * 8;
                }
#pragma unroll 1
                for (int q = 0; q < D / 32; ++q) {
                    uint32_t o[32] = {}, w[16];
                    if (done > 0) {
                        tmem_ld32(to + 32 * q, o);
                        tmem_ld_wait(o);
                    }
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const __nv_bfloat162 h = __floats2bfloat162_rn(done > 0 ? __uint_as_float(o[2 * e]) * inv : 0.f,
                                                                       done > 0 ? __uint_as_float(o[2 * e + 1]) * inv : 0.f);
                        w[e] = *reinterpret_cast<const uint32_t *>(&h);
                        zero[e % 4] = add_times0(w[e], zero[e % 4]);
                    }
                    if (g.vec) {
                        __syncwarp();
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            stage[lane * 4 + (e ^ ((lane >> 1) & 3))] = make_uint4(w[4 * e], w[4 * e + 1], w[4 * e + 2], w[4 * e + 3]);
                        __syncwarp();
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const int row = lane / 4 + 8 * k;
                            const uint4 v = stage[row * 4 + (lane % 4 ^ ((row >> 1) & 3))];
                            if ((mine >> k) & 1u)
                                *reinterpret_cast<uint4 *>(g.a.o + at[k] + 32 * q) = v;
                        }
                    } else if (live) {
                        __nv_bfloat16 *out = g.a.o + t * g.a.o_tok + hq * g.a.o_head + 32 * q;
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            out[2 * e] = __ushort_as_bfloat16((unsigned short)(w[e] & 0xFFFFu));
                            out[2 * e + 1] = __ushort_as_bfloat16((unsigned short)(w[e] >> 16));
                        }
                    }
                }
                if (live && g.a.lse)
                    g.a.lse[(int64_t)hq * g.a.q_tokens + t] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
                const bool seen_odd = live && l > 0.f && l < INFINITY; /* a NaN score is the whole row's */
                if (any(odd || (seen_odd && (odd2(zero[0]) | odd2(zero[1]) | odd2(zero[2]) | odd2(zero[3]))))) {
                    int *at_key = reinterpret_cast<int *>(s_stage[4 * i]); /* of the tile's four warps; 3 D ints */
                    first_odd<D>(g.a, s, it.head, seen_of(g, s, min(s.q1, tile0 + g.tok) - 1), at_key, r, kRows,
                                 [&] { any(false); });
                    if (seen_odd)
                        for (int d = 0; d < D; ++d) {
                            const float x = odd_value<D>(at_key, d, seen_of(g, s, t));
                            if (x != 0.f)
                                g.a.o[t * g.a.o_tok + hq * g.a.o_head + d] = __float2bfloat16_rn(x);
                        }
                }
            }
            tc_before(); /* O is read: the next item's products may write it once this warp's weights are in */
        });
    }
    __syncthreads();
    if (warp == kMmaWarp) {
        tc_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

constexpr int kJoinRows = 32; /* divides a tile's 128 */
/* Joins the parts of blocks whose keys were cut: 32 rows a block, a row a lane, an eighth of
 * its columns a warp (the parts lie by row within four columns, so loads are whole lines). */
template <int D>
__global__ void __launch_bounds__(256, 4) attn_join_kernel(const __grid_constant__ Args g)
{
    __shared__ Seq s_seqs[kSeqsHeld];
    __shared__ Item s_item;
    __shared__ int s_ok, s_first[3 * D];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int b = threadIdx.x; b < min(kSeqsHeld, g.a.seqs); b += 256)
        s_seqs[b] = seq_of(g, b);
    __syncthreads();
    /* blockIdx.x: an item; blockIdx.y: kJoinRows of its rows */
    if (warp == 0) {
        Item first;
        const bool ok = item_of(g, s_seqs, blockIdx.x, true, first);
        first.t0 = first.s.q0 + first.block * 2 * g.tok;
        if (lane == 0)
            s_item = first, s_ok = ok && first.cuts > 1;
    }
    __syncthreads();
    asm volatile("griddepcontrol.wait;" ::: "memory"); /* the parts are the kernel's before */
    if (!s_ok)
        return;
    const Item it = s_item;
    constexpr int C4 = D / 32; /* fours of columns a thread */
    const int row0 = blockIdx.y * kJoinRows, i = row0 / kRows, r = row0 % kRows + lane;
    const float *ml = g.part + (int64_t)g.sms * kSlotRows * D + (int64_t)it.slot * kSlotRows + row0 + lane;
    const int *odds = reinterpret_cast<const int *>(g.part + (int64_t)g.sms * kSlotRows * (D + 2)) + 2 * it.slot + i;
    const float4 *part = reinterpret_cast<const float4 *>(g.part) + (((int64_t)it.slot * 2 + i) * (D / 4) + warp * C4) * kRows + r;
    const bool odd = __any_sync(0xFFFFFFFFu, lane < it.cuts && odds[2 * lane]);
    float m = -INFINITY, l = 0.f;
#pragma unroll 8
    for (int c = 0; c < it.cuts; ++c)
        m = max_nan(m, ml[(int64_t)c * kSlotRows]);
    float4 o[C4];
#pragma unroll
    for (int e = 0; e < C4; ++e)
        o[e] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int c = 0; c < it.cuts; ++c) {
        const float mc = ml[(int64_t)c * kSlotRows], f = mc == -INFINITY ? 0.f : ex2(mc - m);
        l = fmaf(f, ml[((int64_t)g.sms + c) * kSlotRows], l);
#pragma unroll
        for (int e = 0; e < C4; ++e) {
            const float4 v = part[((int64_t)c * 2 * (D / 4) + e) * kRows];
            o[e].x = fmaf(f, v.x, o[e].x), o[e].y = fmaf(f, v.y, o[e].y);
            o[e].z = fmaf(f, v.z, o[e].z), o[e].w = fmaf(f, v.w, o[e].w);
        }
    }
    const int t = it.t0 + i * g.tok + r / g.group, hq = it.head * g.group + r % g.group;
    const bool live = r < g.group * g.tok && t < it.s.q1, seen_odd = live && l > 0.f && l < INFINITY;
    float zero = 0.f; /* 0 times the thread's values, added up */
#pragma unroll
    for (int e = 0; e < C4; ++e)
        zero = fmaf(0.f, o[e].x, fmaf(0.f, o[e].y, fmaf(0.f, o[e].z, fmaf(0.f, o[e].w, zero))));
    if (__syncthreads_or(odd || (seen_odd && zero != zero))) {
        first_odd<D>(g.a, it.s, it.head, seen_of(g, it.s, min(it.s.q1, it.t0 + (i + 1) * g.tok) - 1), s_first, threadIdx.x,
                     256, [] { __syncthreads(); });
        if (seen_odd) {
            const int seen = seen_of(g, it.s, t), d = warp * C4 * 4;
#pragma unroll
            for (int e = 0; e < C4; ++e) {
                auto set = [&](float &x, int at) {
                    const float z = odd_value<D>(s_first, d + at, seen);
                    x = z != 0.f ? z : x;
                };
                set(o[e].x, 4 * e), set(o[e].y, 4 * e + 1), set(o[e].z, 4 * e + 2), set(o[e].w, 4 * e + 3);
            }
        }
    }
    if (!live)
        return;
    const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
    __nv_bfloat16 *out = g.a.o + t * g.a.o_tok + hq * g.a.o_head + warp * C4 * 4;
#pragma unroll
    for (int e = 0; e < C4; ++e) {
        const __nv_bfloat162 a = __floats2bfloat162_rn(o[e].x * inv, o[e].y * inv);
        const __nv_bfloat162 b = __floats2bfloat162_rn(o[e].z * inv, o[e].w * inv);
        if (g.vec) {
            *reinterpret_cast<uint2 *>(out + 4 * e) =
                make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
        } else {
            out[4 * e] = a.x, out[4 * e + 1] = a.y, out[4 * e + 2] = b.x, out[4 * e + 3] = b.y;
        }
    }
    if (warp == 0 && g.a.lse)
        g.a.lse[(int64_t)hq * g.a.q_tokens + t] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
}

/* [tokens][heads][D] as (D, heads, tokens); boxes of 64 x heads x tokens */
bool encode(CUtensorMap *m, const void *p, int D, int heads, int tokens, int64_t head_stride, int64_t tok_stride,
            int box_heads, int box_tokens)
{
    auto enc = tensor_map_encoder();
    if (!enc)
        return false;
    /* the stride of a dimension of one is never used */
    const cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)heads, (cuuint64_t)tokens};
    const cuuint64_t strides[2] = {(cuuint64_t)(heads > 1 ? head_stride : D) * 2, (cuuint64_t)(tokens > 1 ? tok_stride : D) * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)box_heads, (cuuint32_t)box_tokens}, one[3] = {1, 1, 1};
    return enc(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void *>(p), dims, strides, box, one,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
bool strides_ok(const void *p, int heads, int tokens, int64_t head, int64_t tok)
{
    auto ok = [](int64_t s) { return s > 0 && s % 8 == 0 && s < ((int64_t)1 << 38); };
    return aligned_to(p, 16) && (heads == 1 || ok(head)) && (tokens == 1 || ok(tok));
}
/* the tensor-core kernel's calls: what TMA can address, rows that fit a tile, a scale
 * whose order the running maximum keeps */
bool tc_supported(const GlintAttnPrompt &a)
{
    const int group = a.heads / a.kv_heads;
    return group <= kRows && a.scale > 0.f && a.k_tokens > 0 && strides_ok(a.q, a.heads, a.q_tokens, a.q_head, a.q_tok) &&
           strides_ok(a.k, a.kv_heads, a.k_tokens, a.k_head, a.k_tok) &&
           strides_ok(a.v, a.kv_heads, a.k_tokens, a.v_head, a.v_tok);
}
int64_t part_bytes(const GlintAttnPrompt &a)
{
    return (int64_t)sm_count() * (kSlotRows * (a.head_dim + 2) + 2) * 4;
}
/* whether some lengths of the sequences could make cuts worth while */
bool may_split(const GlintAttnPrompt &a)
{
    const int tok = kRows / (a.heads / a.kv_heads);
    const int64_t least = ((int64_t)a.q_tokens + 2 * tok - 1) / (2 * tok) * a.kv_heads;
    return a.k_tokens > kKeys && 2 * least <= sm_count();
}

template <int D>
int tc_launch(const GlintAttnPrompt &a, cudaStream_t st)
{
    Args g{};
    g.a = a;
    g.group = a.heads / a.kv_heads, g.tok = kRows / g.group, g.sms = sm_count();
    g.vec = aligned_to(a.o, 16) && a.o_tok % 8 == 0 && a.o_head % 8 == 0;
    g.split = a.work && may_split(a);
    g.part = static_cast<float *>(a.work);
    Maps maps;
    if (!encode(&maps.q, a.q, D, a.heads, a.q_tokens, a.q_head, a.q_tok, g.group, g.tok) ||
        !encode(&maps.k, a.k, D, a.kv_heads, a.k_tokens, a.k_head, a.k_tok, 1, kKeys) ||
        !encode(&maps.v, a.v, D, a.kv_heads, a.k_tokens, a.v_head, a.v_tok, 1, kKeys))
        return kUnsupported;
    if (!ensure_smem((const void *)attn_kernel<D>, Cfg<D>::kSmem))
        return kLaunch;
    /* every sequence may end in a block of its own */
    const int64_t items = ((int64_t)a.q_tokens / (2 * g.tok) + a.seqs) * a.kv_heads;
    if (items > INT32_MAX / 2)
        return kUnsupported;
    const int64_t grid = g.split ? g.sms : std::min(items, (int64_t)g.sms);
    attn_kernel<D><<<(unsigned)grid, kThreads, Cfg<D>::kSmem, st>>>(g, maps);
    if (cudaGetLastError() != cudaSuccess)
        return kLaunch;
    if (g.split) {
        /* launched beside the other; it waits for that one's end itself */
        cudaLaunchConfig_t cfg = {};
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.gridDim = dim3((unsigned)std::min(items, (int64_t)g.sms / 2), kSlotRows / kJoinRows);
        cfg.blockDim = dim3(256), cfg.stream = st, cfg.attrs = attr, cfg.numAttrs = 1;
        if (cudaLaunchKernelEx(&cfg, attn_join_kernel<D>, g) != cudaSuccess) {
            cudaGetLastError();
            return kLaunch;
        }
    }
    return kOk;
}

} // namespace
} // namespace glint

using namespace glint;

namespace {
int check(const GlintAttnPrompt *a)
{
    if (!a || a->seqs < 0 || a->q_tokens < 0 || a->k_tokens < 0 || a->heads < 1 || a->kv_heads < 1 ||
        a->heads % a->kv_heads)
        return kBadArg;
    return a->head_dim == 64 || a->head_dim == 128 ? kOk : kUnsupported;
}
} // namespace

extern "C" {

int64_t glint_attn_prompt_work_bytes(const GlintAttnPrompt *a)
{
    const int rc = check(a);
    if (rc != kOk)
        return rc;
    return may_split(*a) && a->q_tokens > 0 ? part_bytes(*a) : 0;
}

int glint_attn_prompt_stream(const GlintAttnPrompt *a, cudaStream_t stream)
{
    const int rc = check(a);
    if (rc != kOk)
        return rc;
    if (a->seqs == 0 || a->q_tokens == 0)
        return kOk;
    if (!a->q || !a->o || !a->cu_q || !a->cu_k || (a->k_tokens > 0 && (!a->k || !a->v)) || !aligned_to(a->work, 16))
        return kBadArg;
    if (tc_supported(*a)) {
        const int r = a->head_dim == 128 ? tc_launch<128>(*a, stream) : tc_launch<64>(*a, stream);
        if (r != kUnsupported)
            return r;
    }
    return plain_launch(*a, stream);
}

} /* extern "C" */
