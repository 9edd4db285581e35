/* Attention of a sequence's newest tokens over its 4-bit cache.
 *
 * The rows of one kv head (its query heads times the new tokens, 8 or 16 at a time: the
 * columns of a tensor-core tile) share every byte of the cache that is read.  With
 * x = lo + step * code for K and V, per 64-value block b of a slot t:
 *
 *   s[t, n] = sum_b step (sum_d (code + 16) q[n, d]) + (lo - 16 step) (sum_d q[n, d])
 *   o[d, n] = sum_t (code - 8) (p[t, n] step)       + sum_t p[t, n] (lo + 8 step)
 *
 * so the products are mma.sync tiles whose A operand is the codes themselves: (w &
 * 0x00780078) | 0x41804180 is the BF16 pair 16 + code, as K takes it; (w & 0x000F000F) |
 * 0x43004300 is 128 + code, less 136 it is code - 8, as V does; all exact.
 * The tile's inner index may be any order that both operands share, so a 32-bit word's
 * nibbles j and j + 4 make a pair as they lie.  For K (rows = slots, inner = d) q is
 * permuted to match once; for V (rows = d, inner = slots) a pair is the same nibble of
 * two slots, two byte permutes for eight pairs.  p * step is rounded to BF16 (2^-8 of
 * each weight, the rounding any BF16 tensor-core attention makes); scores, maximum,
 * sums and the lo terms stay in f32.
 *
 * Floor: HBM, D + D / 8 bytes a slot and head at 4.5 bits a value.  Bound: instructions,
 * about 790 of a warp for 32 slots of K and V at D = 128 (ALU 63 %, issue 64 % busy): 320
 * unpack codes, the rest fetch, look up pages, find maxima, exponentiate and multiply.
 * 16 sequences of 16384 slots, 64 / 8 heads: 81 us (loads alone 57, arithmetic alone 71);
 * 64 of 32768: 536 us, 4.51 TB/s.  32 ragged ones of up to 8191, 32 / 8 heads: 30 us, 38
 * with weights.  One of 1021: 11 us, latency.
 */
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "kv4.cuh"
#include "ptx.cuh"

namespace glint {
namespace {

constexpr int kTile = 32;        /* slots a warp takes at a time */
/* What a segment costs beside its tiles, in tiles: with 2, 4, 6, 8, 12 thirty-two sequences
 * of 3 to 8191 slots (8 heads of 128) took 49, 37, 32, 30, 30 us. */
constexpr int kJoin = 8;
constexpr int kWorker = 4;       /* a worker's range, at least */
constexpr float kLazy = 8.f;     /* the running maximum may lag by 2^8 */
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

/* Workers of four warps.  An SM quarter shares 512 registers a lane among its warps:
 * four of 128 for 8 columns; for 16 (twice the accumulators) three of 168 at head_dim 64,
 * two of 255 at 128. */
constexpr int kGroup = 4;
template <int D, int NT>
struct Cfg {
    static constexpr int kWarps = NT == 1 ? 16 : D == 64 ? 12 : 8;
    static constexpr int kThreads = kWarps * 32;
    static constexpr int kStages = NT == 1 && D == 128 ? 2 : 4;
    static constexpr int kCols = 8 * NT;
    static constexpr int kNb = D / 64;
    static constexpr int kJoinThreads = kCols * (D / 4) < 256 ? kCols * (D / 4) : 256;
    static constexpr int kCode = kTile * D / 2, kMeta = kTile * kNb * 4;
    static constexpr int kStage = 2 * (kCode + kMeta);
    static constexpr int kState = kCols * D + 2 * kCols; /* floats: O, m, l */
    static constexpr int kRing = kWarps * kStages * kStage;
    static constexpr int kSmem = kRing + kWarps * kState * 4 + kWarps * 4;
};

struct Args {
    GlintKv4Cache c;
    GlintKv4Attn a;
    int group, cols;      /* query heads a kv head; group * rows */
    int chunks, segs;     /* column chunks a kv head; segments a sequence = kv_heads * chunks */
    int parts;            /* workers at most: workers of a CTA times CTAs */
    int page_log2;
    bool vec;             /* q takes 16-byte loads */
    float *part;          /* [parts][2][kState] unfinished segments */
    float *score;         /* [seqs][kv_heads][max slots][cols] log2-scaled scores, or NULL */
    float *lse2;          /* [seqs][kv_heads][cols] log2 sums, with score */
};

__device__ __forceinline__ float ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ int length_of(const Args &g, int b)
{
    return min(max(g.a.lens[b], 0), g.a.max_pages * g.c.page_size);
}
/* a length may be 2^31 - 16: no signed sum goes past it, here and below */
__device__ __forceinline__ int tiles_of(const Args &g, int b) { return (int)(((uint32_t)length_of(g, b) + kTile - 1) / kTile); }

/* All segments in one row (sequence after sequence), each as long as kJoin plus its
 * tiles, cut into equal ranges over the workers (kGroup warps each): sequences of any mix
 * of lengths keep every SM busy, and a range of many short segments, each with a query
 * to load and a result to write, is not taken for as little work as one long one. */
struct Plan {
    int units;    /* the host has seen to it that they fit */
    int parts;    /* workers with a range */
    int each, more; /* units of a range; ranges with one more */
    __device__ __forceinline__ int begin(int i) const { return each * i + min(i, more); }
    __device__ __forceinline__ int owner(int u) const
    {
        const int big = more * (each + 1);
        return u < big ? u / (each + 1) : more + (u - big) / each;
    }
};
__device__ __forceinline__ int cost_of(int tiles) { return tiles ? tiles + kJoin : 0; }
__device__ __forceinline__ Plan plan_of(const Args &g)
{
    int n = 0;
    for (int b = threadIdx.x & 31; b < g.a.seqs; b += 32)
        n += cost_of(tiles_of(g, b));
#pragma unroll
    for (int off = 16; off > 0; off >>= 1)
        n += __shfl_xor_sync(0xFFFFFFFFu, n, off);
    Plan p;
    p.units = n * g.segs;
    p.parts = max(1, min(g.parts, p.units / kWorker));
    p.each = p.units / p.parts, p.more = p.units - p.each * p.parts;
    return p;
}
/* A segment on a walk along a range: `first` is its first tile's place, counted from
 * the range's begin (negative where the range begins inside the segment). */
struct Walk {
    int b, seg, tiles, first;
    __device__ __forceinline__ int lo() const { return max(0, -first); }
    __device__ __forceinline__ int hi(int range) const { return min(tiles, range - first); }
    __device__ __forceinline__ bool next(const Args &g, int range) /* false at the range's end */
    {
        first += tiles + kJoin;
        if (first >= range)
            return false;
        if (++seg == g.segs) {
            seg = 0;
            do
                tiles = ++b < g.a.seqs ? tiles_of(g, b) : 0;
            while (tiles == 0 && b < g.a.seqs);
        }
        return b < g.a.seqs;
    }
};
__device__ __forceinline__ Walk locate(const Args &g, int u) /* u < units; whole warp */
{
    const int lane = threadIdx.x & 31;
    int before = 0;
    for (int b0 = 0;; b0 += 32) {
        const int t = b0 + lane < g.a.seqs ? tiles_of(g, b0 + lane) : 0;
        int s = cost_of(t);
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int o = __shfl_up_sync(0xFFFFFFFFu, s, off);
            if (lane >= off)
                s += o;
        }
        const uint32_t past = __ballot_sync(0xFFFFFFFFu, (before + s) * g.segs > u);
        if (past || b0 + 32 >= g.a.seqs) {
            const int l = past ? __ffs(past) - 1 : 31;
            Walk w;
            w.b = b0 + l;
            w.tiles = __shfl_sync(0xFFFFFFFFu, t, l);
            const int cost = max(1, cost_of(w.tiles));
            const int off = u - (before + __shfl_sync(0xFFFFFFFFu, s, l) - cost) * g.segs;
            w.seg = off / cost;
            w.first = w.seg * cost - off + kJoin;
            return w;
        }
        before += __shfl_sync(0xFFFFFFFFu, s, 31);
    }
}

__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                 "{%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
/* the same onto zero */
__device__ __forceinline__ void mma0(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                 "{%10,%10,%10,%10};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
/* (step, lo) of a row's blocks */
template <int NB>
__device__ __forceinline__ void load_meta(uint32_t at, uint32_t (&m)[NB])
{
    if constexpr (NB == 2) {
        const uint2 v = lds64(at);
        m[0] = v.x, m[1] = v.y;
    } else {
        m[0] = lds32(at);
    }
}
/* nibbles j and j + 4 of w as the BF16 pair (16 + code, 16 + code), for the products whose
 * excess is taken back in f32: 128 + code needs a shift less, but its eight times larger sums
 * cancel to eight times the error (lse of few slots: 2e-6 of its value) */
__device__ __forceinline__ uint32_t codes16(uint32_t w, int j)
{
    uint32_t r;
    asm("lop3.b32 %0, %1, 0x00780078, %2, 0xEA;" : "=r"(r) : "r"(j ? w >> (4 * j - 3) : w << 3), "r"(0x41804180u));
    return r;
}
/* the same as (128 + code, 128 + code) */
__device__ __forceinline__ uint32_t codes128(uint32_t w, int j)
{
    uint32_t r;
    asm("lop3.b32 %0, %1, 0x000F000F, %2, 0xEA;" : "=r"(r) : "r"(w >> (4 * j)), "r"(0x43004300u));
    return r;
}
/* the same as (code - 8, code - 8), exact */
__device__ __forceinline__ uint32_t codes(uint32_t w, int j)
{
    const uint32_t r = codes128(w, j);
    const __nv_bfloat162 v = __hsub2(*reinterpret_cast<const __nv_bfloat162 *>(&r), __floats2bfloat162_rn(136.f, 136.f));
    return *reinterpret_cast<const uint32_t *>(&v);
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v)
{
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi)
{
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&v);
}
/* slot (of 8) that row r of a tile stands for: with the swapped halves, the four slots
 * of any fragment load (rows 0-3, rows 4-7, even rows, odd rows) differ mod 4 */
__device__ __forceinline__ int slot_of(int r) { return (r & 4) | (((r ^ (r >> 2)) & 1) << 1) | ((r >> 1) & 1); }

/* A warp's running softmax over the slots it has seen, as tile fragments: lane (g, c) =
 * (lane / 4, lane % 4) holds columns 2c, 2c + 1 of m, l and, per 64-block b and j < 4,
 * o at d = 64 b + 8 g + j (values 0, 1) and + 4 (values 2, 3). */
template <int D, int NT>
struct State {
    float o[NT][D / 64][4][4];
    float m[NT][2], l[NT][2], lo[NT][D / 64][2];
    __device__ __forceinline__ void clear()
    {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int b = 0; b < D / 64; ++b) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        o[n][b][j][i] = 0.f;
                lo[n][b][0] = lo[n][b][1] = 0.f;
            }
            m[n][0] = m[n][1] = -INFINITY;
            l[n][0] = l[n][1] = 0.f;
        }
    }
};

/* q of one segment's columns as B fragments, and its sums per block */
template <int D, int NT>
struct Query {
    uint32_t b[NT][D / 64][4][2];
    float sum[NT][D / 64][2];
    int see[NT][2]; /* slots that columns 2c, 2c + 1 see */
};

template <int D, int NT>
__device__ __forceinline__ void load_query(const Args &g, int b, int seg, Query<D, NT> &q, int lane)
{
    const int h = seg / g.chunks, ch = seg - h * g.chunks;
    const int gr = lane >> 2, c = lane & 3;
    const uint32_t sign = g.a.scale < 0.f ? 0x8000u : 0u; /* the kernel scales by |scale| */
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int col = ch * 8 * NT + n * 8 + gr;
        const bool live = col < g.cols;
        const int r = live ? col / g.group : 0, hq = h * g.group + (live ? col - r * g.group : 0);
        const __nv_bfloat16 *p = g.a.q + b * g.a.q_seq + r * g.a.q_row + hq * g.a.q_head + 16 * c;
#pragma unroll
        for (int k = 0; k < D / 64; ++k) {
            uint32_t v[16];
            float s = 0.f;
            if (g.vec) {
                const uint4 z = make_uint4(0u, 0u, 0u, 0u);
                const uint4 a = live ? *reinterpret_cast<const uint4 *>(p + 64 * k) : z;
                const uint4 c = live ? *reinterpret_cast<const uint4 *>(p + 64 * k + 8) : z;
                const uint32_t w[8] = {a.x, a.y, a.z, a.w, c.x, c.y, c.z, c.w};
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    v[2 * i] = w[i] & 0xFFFFu, v[2 * i + 1] = w[i] >> 16;
            } else {
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    v[i] = live ? (uint32_t)__bfloat16_as_ushort(p[64 * k + i]) : 0u;
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                v[i] ^= live ? sign : 0u;
                s += __uint_as_float(v[i] << 16);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                q.b[n][k][j][0] = v[j] | (v[j + 4] << 16);
                q.b[n][k][j][1] = v[j + 8] | (v[j + 12] << 16);
            }
            s += __shfl_xor_sync(0xFFFFFFFFu, s, 1);
            s += __shfl_xor_sync(0xFFFFFFFFu, s, 2);
            q.sum[n][k][0] = __shfl_sync(0xFFFFFFFFu, s, 8 * c);
            q.sum[n][k][1] = __shfl_sync(0xFFFFFFFFu, s, 8 * c + 4);
        }
        const int len = length_of(g, b);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int cc = ch * 8 * NT + n * 8 + 2 * c + i;
            q.see[n][i] = cc < g.cols ? len - g.a.rows + cc / g.group + 1 : len;
        }
    }
}

/* One tile of 32 slots (from slot t0) in shared memory. */
template <int D, int NT, bool SCORE, bool WHOLE>
__device__ __forceinline__ void tile_step(const Args &g, const Query<D, NT> &q, State<D, NT> &st, uint32_t stage,
                                          int t0, uint32_t valid, float scale2, float *score, int chunk,
                                          int lane)
{
    using C = Cfg<D, NT>;
    constexpr int NB = D / 64, RB = D / 2;
    const int gr = lane >> 2, c = lane & 3;
    const int tg = slot_of(gr);
    const uint32_t kcode = stage, kmeta = stage + C::kCode, vcode = kmeta + C::kMeta, vmeta = vcode + C::kCode;
    float s[2][NT][4];
#pragma unroll
    for (int sl = 0; sl < 2; ++sl) {
        const int ta = sl * 16 + tg, tb = ta + 8; /* slots of fragment rows g and g + 8 */
        float acc[NB][NT][4];
#pragma unroll
        for (int k = 0; k < NB; ++k) {
            const uint2 wa = lds64(kcode + ta * RB + kv4_unit<D>(k, ta) + 8 * c);
            const uint2 wb = lds64(kcode + tb * RB + kv4_unit<D>(k, tb) + 8 * c);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t a[4] = {codes16(wa.x, j), codes16(wb.x, j), codes16(wa.y, j), codes16(wb.y, j)};
#pragma unroll
                for (int n = 0; n < NT; ++n)
                    j ? mma(acc[k][n], a, q.b[n][k][j][0], q.b[n][k][j][1])
                      : mma0(acc[k][n], a, q.b[n][k][j][0], q.b[n][k][j][1]);
            }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                s[sl][n][i] = 0.f;
        uint32_t mas[NB], mbs[NB];
        load_meta(kmeta + ta * NB * 4, mas);
        load_meta(kmeta + tb * NB * 4, mbs);
#pragma unroll
        for (int k = 0; k < NB; ++k) {
            const uint32_t ma = mas[k], mb = mbs[k];
            const float sa = __uint_as_float(ma << 16), sb = __uint_as_float(mb << 16);
            const float la = fmaf(-16.f, sa, __uint_as_float(ma & 0xFFFF0000u));
            const float lb = fmaf(-16.f, sb, __uint_as_float(mb & 0xFFFF0000u));
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                s[sl][n][0] = fmaf(sa, acc[k][n][0], fmaf(la, q.sum[n][k][0], s[sl][n][0]));
                s[sl][n][1] = fmaf(sa, acc[k][n][1], fmaf(la, q.sum[n][k][1], s[sl][n][1]));
                s[sl][n][2] = fmaf(sb, acc[k][n][2], fmaf(lb, q.sum[n][k][0], s[sl][n][2]));
                s[sl][n][3] = fmaf(sb, acc[k][n][3], fmaf(lb, q.sum[n][k][1], s[sl][n][3]));
            }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int t = i < 2 ? ta : tb;
                if (!WHOLE && (!((valid >> t) & 1u) || t0 + t >= q.see[n][i & 1]))
                    s[sl][n][i] = -INFINITY;
            }
        if constexpr (SCORE) {
            auto scaled = [&](float v) { return !WHOLE && v == -INFINITY ? v : v * scale2; };
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const int col = chunk * 8 * NT + n * 8 + 2 * c;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    float *p = score + (int64_t)(t0 + (i ? tb : ta)) * g.cols + col;
                    if (WHOLE || ((valid >> (i ? tb : ta)) & 1u)) {
                        if (col < g.cols)
                            p[0] = scaled(s[sl][n][2 * i]);
                        if (col + 1 < g.cols)
                            p[1] = scaled(s[sl][n][2 * i + 1]);
                    }
                }
            }
        }
    }
    /* running maximum per column, over the 8 lanes that share it */
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        float top[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            top[i] = fmaxf(fmaxf(s[0][n][i], s[0][n][i + 2]), fmaxf(s[1][n][i], s[1][n][i + 2]));
#pragma unroll
            for (int off = 4; off < 32; off <<= 1)
                top[i] = fmaxf(top[i], __shfl_xor_sync(0xFFFFFFFFu, top[i], off));
            top[i] *= scale2;
        }
        const bool grow = top[0] > st.m[n][0] + kLazy || top[1] > st.m[n][1] + kLazy ||
                          (st.m[n][0] == -INFINITY && top[0] != -INFINITY) ||
                          (st.m[n][1] == -INFINITY && top[1] != -INFINITY);
        if (__any_sync(0xFFFFFFFFu, grow)) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float m = fmaxf(st.m[n][i], top[i]);
                const float f = st.m[n][i] == -INFINITY ? 0.f : ex2(st.m[n][i] - m);
                st.m[n][i] = m;
                st.l[n][i] *= f;
#pragma unroll
                for (int k = 0; k < NB; ++k) {
                    st.lo[n][k][i] *= f;
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        st.o[n][k][j][i] *= f, st.o[n][k][j][i + 2] *= f;
                }
            }
        }
    }
    float less[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i)
            less[n][i] = st.m[n][i] == -INFINITY ? 0.f : -st.m[n][i];
#pragma unroll
    for (int sl = 0; sl < 2; ++sl) {
        const int ta = sl * 16 + tg, tb = ta + 8;
        uint32_t pb[NT][NB][2];
        float steps[NB][2], mids[NB][2];
        uint32_t mas[NB], mbs[NB];
        load_meta(vmeta + ta * NB * 4, mas);
        load_meta(vmeta + tb * NB * 4, mbs);
#pragma unroll
        for (int k = 0; k < NB; ++k) {
            const uint32_t ma = mas[k], mb = mbs[k];
            steps[k][0] = __uint_as_float(ma << 16), steps[k][1] = __uint_as_float(mb << 16);
            mids[k][0] = fmaf(8.f, steps[k][0], __uint_as_float(ma & 0xFFFF0000u));
            mids[k][1] = fmaf(8.f, steps[k][1], __uint_as_float(mb & 0xFFFF0000u));
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            float p[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                p[i] = !WHOLE && s[sl][n][i] == -INFINITY ? 0.f : ex2(fmaf(s[sl][n][i], scale2, less[n][i & 1]));
                st.l[n][i & 1] += p[i];
            }
#pragma unroll
            for (int k = 0; k < NB; ++k) {
                float w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    /* a masked slot's step and lo may be anything, NaN too */
                    const bool out = !WHOLE && s[sl][n][i] == -INFINITY;
                    w[i] = out ? 0.f : p[i] * steps[k][i >> 1];
                    st.lo[n][k][i & 1] = out ? st.lo[n][k][i & 1] : fmaf(p[i], mids[k][i >> 1], st.lo[n][k][i & 1]);
                }
                pb[n][k][0] = transpose8x8(pack2(w[0], w[1]));
                pb[n][k][1] = transpose8x8(pack2(w[2], w[3]));
            }
        }
        const int te = sl * 16 + slot_of(2 * c), to = sl * 16 + slot_of(2 * c + 1); /* inner 2c, 2c + 1; + 8 */
#pragma unroll
        for (int k = 0; k < NB; ++k) {
            const uint32_t w0 = lds32(vcode + te * RB + kv4_unit<D>(k, te) + 4 * gr);
            const uint32_t w1 = lds32(vcode + to * RB + kv4_unit<D>(k, to) + 4 * gr);
            const uint32_t w2 = lds32(vcode + (te + 8) * RB + kv4_unit<D>(k, te + 8) + 4 * gr);
            const uint32_t w3 = lds32(vcode + (to + 8) * RB + kv4_unit<D>(k, to + 8) + 4 * gr);
            const uint32_t x0 = __byte_perm(w0, w1, 0x5410), y0 = __byte_perm(w0, w1, 0x7632);
            const uint32_t x1 = __byte_perm(w2, w3, 0x5410), y1 = __byte_perm(w2, w3, 0x7632);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t a[4] = {codes(x0, j), codes(y0, j), codes(x1, j), codes(y1, j)};
#pragma unroll
                for (int n = 0; n < NT; ++n)
                    mma(st.o[n][k][j], a, pb[n][k][0], pb[n][k][1]);
            }
        }
    }
}

/* A warp's walk over the tiles it fetches. */
struct Fetch {
    Walk w;
    int tile; /* the next one, -1: none left */
    int len;  /* its sequence's length */
    int page; /* lanes 0 and 1: the page of its slots 0-15 and 16-31, -1 for none */
};
__device__ __forceinline__ void fetch_seek(const Args &g, Fetch &f, int range, int lane)
{
    while (f.tile >= f.w.hi(range)) {
        f.tile -= max(f.w.hi(range), f.w.lo());
        const int b = f.w.b;
        if (!f.w.next(g, range)) {
            f.tile = -1;
            return;
        }
        if (f.w.b != b)
            f.len = length_of(g, f.w.b);
    }
    const int t = f.tile * kTile + 16 * lane;
    f.page = -1;
    if (lane < 2 && t < f.len)
        f.page = g.a.table[(int64_t)f.w.b * g.a.max_pages + (t >> g.page_log2)];
}
__device__ __forceinline__ void copy16(uint32_t dst, const uint8_t *src)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
/* start copying the tile into a stage (16 bytes a lane and copy); returns its valid slots */
template <int D, int NT>
__device__ __forceinline__ uint32_t fetch_issue(const Args &g, const Fetch &f, uint32_t stage, int lane)
{
    using C = Cfg<D, NT>;
    constexpr int N = C::kCode / 512, M = C::kMeta / 16;
    const int t0 = f.tile * kTile, h = f.w.seg / g.chunks;
    const uint32_t half = __ballot_sync(0xFFFFFFFFu, f.page >= 0 && f.page < g.c.pages);
    const int p0 = __shfl_sync(0xFFFFFFFFu, f.page, 0), p1 = __shfl_sync(0xFFFFFFFFu, f.page, 1);
    /* rows of slots 0 and 16: the halves are in two pages or 16 rows apart in one */
    const int in = t0 & (g.c.page_size - 1);
    const int64_t r0 = (((int64_t)p0 * g.c.kv_heads + h) << g.page_log2) + in;
    const int64_t r1 = g.page_log2 == 4 ? ((int64_t)p1 * g.c.kv_heads + h) << 4 : r0 + 16;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int u = i >= N / 2;
        if ((half >> u) & 1u) {
            const int at = (lane + 32 * i) * 16;
            const int64_t src = (u ? r1 : r0) * (D / 2) + at - u * (C::kCode / 2);
            copy16(stage + at, g.c.k_code + src);
            copy16(stage + C::kCode + C::kMeta + at, g.c.v_code + src);
        }
    }
    const int m = lane & (M - 1), u = m >= M / 2;
    if (lane < 2 * M && ((half >> u) & 1u)) {
        const bool key = lane < M;
        const uint16_t *meta = key ? g.c.k_meta : g.c.v_meta;
        copy16(stage + (key ? 0 : C::kCode + C::kMeta) + C::kCode + m * 16,
               reinterpret_cast<const uint8_t *>(meta) + (u ? r1 : r0) * (D / 16) + m * 16 - u * (C::kMeta / 2));
    }
    uint32_t v = ((half & 1u) ? 0xFFFFu : 0u) | ((half & 2u) ? 0xFFFF0000u : 0u);
    if ((uint32_t)t0 + kTile > (uint32_t)f.len)
        v &= (1u << (f.len - t0)) - 1u; /* len > t0 */
    return v;
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() /* all but the newest N groups have landed */
{
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

/* columns [0, cols) of one segment from its joined state: thread i of n */
template <int D>
__device__ __forceinline__ void write_column4(const Args &g, int b, int seg, int kcols, int n, int d, float4 o, float m,
                                              float l)
{
    const int h = seg / g.chunks, col = (seg - h * g.chunks) * kcols + n;
    if (col >= g.cols)
        return;
    const int r = col / g.group, hq = h * g.group + col - r * g.group;
    const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l); /* no slot seen: 0; NaN stays */
    uint2 w;
    w.x = pack2(o.x * inv, o.y * inv), w.y = pack2(o.z * inv, o.w * inv);
    __nv_bfloat16 *out = g.a.o + (((int64_t)b * g.a.rows + r) * g.a.heads + hq) * D + d;
    *reinterpret_cast<uint2 *>(out) = w;
    if (d == 0) {
        const float z = l == 0.f ? -INFINITY : m + log2f(l);
        if (g.a.lse)
            g.a.lse[((int64_t)b * g.a.heads + hq) * g.a.rows + r] = z == -INFINITY ? z : z * kLn2;
        if (g.lse2)
            g.lse2[((int64_t)b * g.c.kv_heads + h) * g.cols + col] = z;
    }
}

/* barrier of one worker's warps */
template <int WARPS>
__device__ __forceinline__ void worker_sync(int i)
{
    asm volatile("bar.sync %0, %1;" ::"r"(i + 1), "n"(WARPS * 32) : "memory");
}

/* a warp's state to shared memory (O by column, m, l), the lo terms added in */
template <int D, int NT>
__device__ __forceinline__ void store_state(const State<D, NT> &st, float *mem, int lane)
{
    using C = Cfg<D, NT>;
    const int gr = lane >> 2, c = lane & 3;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float l = st.l[n][i], lo[D / 64];
#pragma unroll
            for (int k = 0; k < D / 64; ++k)
                lo[k] = st.lo[n][k][i];
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) {
                l += __shfl_xor_sync(0xFFFFFFFFu, l, off);
#pragma unroll
                for (int k = 0; k < D / 64; ++k)
                    lo[k] += __shfl_xor_sync(0xFFFFFFFFu, lo[k], off);
            }
            const int col = n * 8 + 2 * c + i;
            if (gr == 0)
                mem[C::kCols * D + col] = st.m[n][i], mem[C::kCols * D + C::kCols + col] = l;
#pragma unroll
            for (int k = 0; k < D / 64; ++k)
#pragma unroll
                for (int up = 0; up < 2; ++up)
                    *reinterpret_cast<float4 *>(mem + col * D + 64 * k + 8 * gr + 4 * up) =
                        make_float4(st.o[n][k][0][2 * up + i] + lo[k], st.o[n][k][1][2 * up + i] + lo[k],
                                    st.o[n][k][2][2 * up + i] + lo[k], st.o[n][k][3][2 * up + i] + lo[k]);
        }
}

template <int D, int NT, bool SCORE>
__global__ void __launch_bounds__(Cfg<D, NT>::kThreads, 1) kv4_attn_kernel(const Args g)
{
    using C = Cfg<D, NT>;
    extern __shared__ __align__(128) uint8_t smem[];
    float *state = reinterpret_cast<float *>(smem + C::kRing);
    int *used = reinterpret_cast<int *>(state + C::kWarps * C::kState);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const Plan plan = plan_of(g);
    asm volatile("griddepcontrol.launch_dependents;");

    /* sequences without a slot: no tile reaches them */
    for (int b = blockIdx.x; b < g.a.seqs; b += gridDim.x)
        if (length_of(g, b) == 0)
            for (int i = threadIdx.x; i < g.segs * C::kCols * (D / 4); i += C::kThreads) {
                const int seg = i / (C::kCols * (D / 4)), e = i % (C::kCols * (D / 4));
                write_column4<D>(g, b, seg, C::kCols, e / (D / 4), e % (D / 4) * 4, make_float4(0.f, 0.f, 0.f, 0.f),
                                 -INFINITY, 0.f);
            }
    /* workers go round the SMs first, so a few of them spread out */
    const int worker = (warp / kGroup) * gridDim.x + blockIdx.x, w = warp % kGroup;
    if (worker >= plan.parts || plan.units == 0)
        return;
    const int begin = plan.begin(worker), range = plan.begin(worker + 1) - begin;
    Walk at = locate(g, begin);

    const uint32_t ring = saddr(smem + warp * C::kStages * C::kStage);
    const float scale2 = fabsf(g.a.scale) * kLog2e;
    uint32_t valid[C::kStages]; /* of the tiles on their way, in order */
    Fetch f{at, at.lo() + w, length_of(g, at.b), -1};
    fetch_seek(g, f, range, lane);
    auto fetch = [&](int stage) {
        uint32_t v = 0;
        if (f.tile >= 0) {
            v = fetch_issue<D, NT>(g, f, ring + stage * C::kStage, lane);
            f.tile += kGroup;
            fetch_seek(g, f, range, lane);
        }
        copies_commit();
        return v;
    };
#pragma unroll
    for (int i = 0; i < C::kStages; ++i)
        valid[i] = fetch(i);
    int slot = 0; /* the stage to read next */

    Query<D, NT> q;
    State<D, NT> st;
    float *mem = state + warp * C::kState;
    int turn = w; /* how far the worker's next tile is from this warp's */
    do {
        const int lo = at.lo(), hi = at.hi(range);
        if (lo >= hi)
            continue;
        const int h = at.seg / g.chunks, chunk = at.seg - h * g.chunks, len = length_of(g, at.b);
        int tile = lo + turn;
        const bool mine = tile < hi;
        if (mine) {
            load_query<D, NT>(g, at.b, at.seg, q, lane);
            st.clear();
        }
        float *score = SCORE ? g.score + ((int64_t)at.b * g.c.kv_heads + h) * g.a.max_pages * g.c.page_size * g.cols
                             : nullptr;
        for (; tile < hi; tile += kGroup) {
            copies_wait<C::kStages - 1>();
            __syncwarp();
            const uint32_t v = valid[0], stage = ring + slot * C::kStage;
            if (v == 0xFFFFFFFFu && (uint32_t)tile * kTile + kTile <= (uint32_t)max(len - g.a.rows + 1, 0))
                tile_step<D, NT, SCORE, true>(g, q, st, stage, tile * kTile, v, scale2, score, chunk, lane);
            else
                tile_step<D, NT, SCORE, false>(g, q, st, stage, tile * kTile, v, scale2, score, chunk, lane);
            __syncwarp();
#pragma unroll
            for (int i = 1; i < C::kStages; ++i)
                valid[i - 1] = valid[i];
            valid[C::kStages - 1] = fetch(slot);
            slot = slot + 1 == C::kStages ? 0 : slot + 1;
        }
        turn = tile - hi;
        if (mine)
            store_state<D, NT>(st, mem, lane);
        if (lane == 0)
            used[warp] = mine ? 1 : 0;
        worker_sync<kGroup>(warp / kGroup);
        /* joined over the warps in their order; the whole segment, or a part of it for the join kernel */
        const bool first = at.first >= 0, whole = first && at.first + at.tiles <= range;
        float *part = g.part + ((int64_t)worker * 2 + (first ? 1 : 0)) * C::kState;
        const float *states = state + (warp - w) * C::kState;
        const int *mask = used + (warp - w);
        for (int i = w * 32 + lane; i < C::kCols * (D / 4); i += kGroup * 32) {
            const int n = i / (D / 4), d = i % (D / 4) * 4;
            float m = -INFINITY, l = 0.f;
#pragma unroll
            for (int k = 0; k < kGroup; ++k)
                if (mask[k])
                    m = fmaxf(m, states[k * C::kState + C::kCols * D + n]);
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int k = 0; k < kGroup; ++k) {
                if (!mask[k])
                    continue;
                const float *s = states + k * C::kState;
                const float mk = s[C::kCols * D + n], fk = mk == -INFINITY ? 0.f : ex2(mk - m);
                const float4 v = *reinterpret_cast<const float4 *>(s + n * D + d);
                l = fmaf(fk, s[C::kCols * D + C::kCols + n], l);
                o.x = fmaf(fk, v.x, o.x), o.y = fmaf(fk, v.y, o.y), o.z = fmaf(fk, v.z, o.z), o.w = fmaf(fk, v.w, o.w);
            }
            if (whole) {
                write_column4<D>(g, at.b, at.seg, C::kCols, n, d, o, m, l);
            } else {
                *reinterpret_cast<float4 *>(part + n * D + d) = o;
                if (d == 0)
                    part[C::kCols * D + n] = m, part[C::kCols * D + C::kCols + n] = l;
            }
        }
        worker_sync<kGroup>(warp / kGroup);
    } while (at.next(g, range));
}

constexpr int kJoinParts = 32;
/* Joins the parts of the segment that begins in worker blockIdx.x's range and runs on
 * past it. */
template <int D, int NT>
__global__ void __launch_bounds__(Cfg<D, NT>::kJoinThreads) kv4_join_kernel(const Args g)
{
    using C = Cfg<D, NT>;
    __shared__ float ms[C::kCols][kJoinParts + 1], ls[C::kCols][kJoinParts + 1];
    const Plan plan = plan_of(g);
    const int i = blockIdx.x;
    Walk at{};
    int last = i;
    if (i + 1 < plan.parts && plan.units > 0) {
        const int begin = plan.begin(i), end = plan.begin(i + 1);
        at = locate(g, end - 1);
        const int first = end - 1 + at.first; /* the segment's first tile in the row */
        if (first >= begin && first < end && first + at.tiles > end)
            last = plan.owner(first + at.tiles - 1);
    }
    asm volatile("griddepcontrol.wait;" ::: "memory"); /* in every CTA: this kernel ends after the one before */
    if (last == i)
        return;
    /* kJoinParts parts a time: their maxima and sums side by side, then their rows */
    constexpr int T = C::kJoinThreads, N = C::kCols * (D / 4) / T;
    float m[N], l[N];
    float4 o[N];
#pragma unroll
    for (int k = 0; k < N; ++k)
        m[k] = -INFINITY, l[k] = 0.f, o[k] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int p0 = i; p0 <= last; p0 += kJoinParts) {
        const int np = min(kJoinParts, last + 1 - p0);
        for (int e = threadIdx.x; e < np * C::kCols; e += T) {
            const int p = p0 + e / C::kCols, n = e % C::kCols;
            const float *s = g.part + ((int64_t)p * 2 + (p == i)) * C::kState + C::kCols * D;
            ms[n][p - p0] = s[n], ls[n][p - p0] = s[C::kCols + n];
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const int e = threadIdx.x + T * k, n = e / (D / 4), d = e % (D / 4) * 4;
            float top = m[k];
            for (int p = 0; p < np; ++p)
                top = fmaxf(top, ms[n][p]);
            const float f0 = m[k] == -INFINITY ? 0.f : ex2(m[k] - top);
            l[k] *= f0;
            o[k].x *= f0, o[k].y *= f0, o[k].z *= f0, o[k].w *= f0;
            m[k] = top;
#pragma unroll 8
            for (int p = 0; p < np; ++p) {
                const float4 v = *reinterpret_cast<const float4 *>(
                    g.part + ((int64_t)(p0 + p) * 2 + (p0 + p == i)) * C::kState + n * D + d);
                const float f = ms[n][p] == -INFINITY ? 0.f : ex2(ms[n][p] - top);
                l[k] = fmaf(f, ls[n][p], l[k]);
                o[k].x = fmaf(f, v.x, o[k].x), o[k].y = fmaf(f, v.y, o[k].y);
                o[k].z = fmaf(f, v.z, o[k].z), o[k].w = fmaf(f, v.w, o[k].w);
            }
        }
        __syncthreads();
    }
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const int e = threadIdx.x + T * k, n = e / (D / 4), d = e % (D / 4) * 4;
        write_column4<D>(g, at.b, at.seg, C::kCols, n, d, o[k], m[k], l[k]);
    }
}

/* weight_out from the scores: the columns of a slot in order, by one thread (four a load
 * where they are a multiple of four). */
/* Slots a thread, 256 apart, loaded together.  1, 2, 4: one sequence of 1021 slots, 32 / 8
 * heads, 13.0, 13.6, 14.4 us; 32 ragged of up to 8191 38.4, 37.3, 36.8; 16 of 16384, 64 / 8
 * heads, 102.6, 101.1, 100.1. */
constexpr int kWeightSlots = 2;
__global__ void __launch_bounds__(256) kv4_weight_kernel(const Args g)
{
    const int bh = blockIdx.y, b = bh / g.c.kv_heads;
    const int len = length_of(g, b), first = blockIdx.x * 256 * kWeightSlots;
    if (first >= len && (blockIdx.x | blockIdx.y)) /* one CTA waits in any case: this kernel ends after the one before */
        return;
    /* the caller's, older than the scores' kernel */
    float sum[kWeightSlots], old[kWeightSlots];
    bool in[kWeightSlots];
    const int64_t row = (int64_t)bh * g.a.weight_stride;
#pragma unroll
    for (int j = 0; j < kWeightSlots; ++j) {
        const int t = first + j * 256 + threadIdx.x;
        old[j] = g.a.weight && t < len - g.a.rows ? g.a.weight[row + t] : 0.f;
        const int page = t < len ? g.a.table[(int64_t)b * g.a.max_pages + (t >> g.page_log2)] : -1;
        in[j] = page >= 0 && page < g.c.pages;
        sum[j] = 0.f;
    }
    asm volatile("griddepcontrol.wait;" ::: "memory"); /* scores and sums are the kernels' before */
    const float *z = g.lse2 + (int64_t)bh * g.cols;
    const float *s = g.score + ((int64_t)bh * (g.a.max_pages << g.page_log2) + first + threadIdx.x) * g.cols;
    auto add = [&](int j, int n, int count) {
        if (!in[j])
            return;
        const float *p = s + (int64_t)j * 256 * g.cols + n;
        auto one = [&](float v, float zn) { sum[j] += v == -INFINITY ? 0.f : ex2(v - zn); };
        if (count == 4) {
            const float4 v = *reinterpret_cast<const float4 *>(p), y = *reinterpret_cast<const float4 *>(z + n);
            one(v.x, y.x), one(v.y, y.y), one(v.z, y.z), one(v.w, y.w);
        } else {
            one(*p, z[n]);
        }
    };
    if (g.cols == 4) { /* one load a slot: all slots' at once */
#pragma unroll
        for (int j = 0; j < kWeightSlots; ++j)
            add(j, 0, 4);
    } else { /* a slot's columns lie apart from the next thread's: slot by slot, while its sectors are at hand */
#pragma unroll
        for (int j = 0; j < kWeightSlots; ++j) {
            int n = 0;
            if (g.cols % 4 == 0)
                for (; n < g.cols; n += 4)
                    add(j, n, 4);
            for (; n < g.cols; ++n)
                add(j, n, 1);
        }
    }
#pragma unroll
    for (int j = 0; j < kWeightSlots; ++j) {
        const int t = first + j * 256 + threadIdx.x;
        if (t < len)
            g.a.weight_out[row + t] = old[j] + sum[j];
    }
}

int check(const GlintKv4Cache *c, const GlintKv4Attn *a)
{
    const int rc = kv4_check(c);
    if (rc != kOk)
        return rc;
    if (!a || a->seqs < 0 || a->rows < 1 || a->heads < 1 || a->heads % c->kv_heads || a->max_pages < 1 ||
        (int64_t)a->heads / c->kv_heads * a->rows > 256 || (int64_t)a->max_pages * c->page_size > INT32_MAX ||
        (int64_t)a->seqs * c->kv_heads > 65535)
        return kBadArg;
    /* the row of segments is counted in 32 bits */
    const int64_t cols = (int64_t)a->heads / c->kv_heads * a->rows, chunks = cols <= 8 ? 1 : (cols + 15) / 16;
    if ((((int64_t)a->max_pages * c->page_size + kTile - 1) / kTile + kJoin) * a->seqs * c->kv_heads * chunks > INT32_MAX)
        return kBadArg;
    return kOk;
}

/* bytes of the parts; of the log2 sums, rounded up; of the scores */
struct Work {
    int64_t part, lse2, score;
};
Work work_of(const GlintKv4Cache &c, const GlintKv4Attn &a)
{
    const int64_t cols = (int64_t)a.heads / c.kv_heads * a.rows, kcols = cols <= 8 ? 8 : 16;
    Work w;
    w.part = 2 * (int64_t)sm_count() * (kcols == 8 ? Cfg<64, 1>::kWarps : Cfg<64, 2>::kWarps) / kGroup * (kcols * c.head_dim + 2 * kcols) * 4; /* workers an SM, at most */
    w.lse2 = a.weight_out ? ((int64_t)a.seqs * c.kv_heads * cols * 4 + 15) / 16 * 16 : 0;
    w.score = a.weight_out ? (int64_t)a.seqs * c.kv_heads * a.max_pages * c.page_size * cols * 4 : 0;
    return w;
}

/* the next kernel's launch may overlap the end of the one before; it waits itself
 * (griddepcontrol.wait) before it touches that one's results */
template <class... P>
cudaError_t launch_after(void (*kernel)(P...), dim3 grid, int threads, cudaStream_t st, const Args &g)
{
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = grid, cfg.blockDim = dim3(threads), cfg.stream = st, cfg.attrs = attr, cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, g);
}

template <int D, int NT>
int launch(Args &g, cudaStream_t st)
{
    using C = Cfg<D, NT>;
    const void *kernel = g.score ? (const void *)kv4_attn_kernel<D, NT, true> : (const void *)kv4_attn_kernel<D, NT, false>;
    if (!ensure_smem(kernel, C::kSmem))
        return kLaunch;
    g.chunks = (g.cols + C::kCols - 1) / C::kCols;
    g.segs = g.c.kv_heads * g.chunks;
    const int grid = sm_count();
    g.parts = grid * (C::kWarps / kGroup);
    if (g.score)
        kv4_attn_kernel<D, NT, true><<<grid, C::kThreads, C::kSmem, st>>>(g);
    else
        kv4_attn_kernel<D, NT, false><<<grid, C::kThreads, C::kSmem, st>>>(g);
    if (cudaGetLastError() != cudaSuccess)
        return kLaunch;
    if (launch_after(kv4_join_kernel<D, NT>, dim3(g.parts), C::kJoinThreads, st, g) != cudaSuccess) {
        cudaGetLastError();
        return kLaunch;
    }
    if (g.score) {
        const dim3 grid((g.a.max_pages * g.c.page_size - 1) / (256 * kWeightSlots) + 1, g.a.seqs * g.c.kv_heads);
        if (launch_after(kv4_weight_kernel, grid, 256, st, g) != cudaSuccess) {
            cudaGetLastError();
            return kLaunch;
        }
    }
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
    const Work w = work_of(*c, *a);
    return w.part + w.lse2 + w.score;
}

int glint_kv4_attn_stream(const GlintKv4Cache *c, const GlintKv4Attn *a, cudaStream_t stream)
{
    const int rc = check(c, a);
    if (rc != kOk)
        return rc;
    if (a->seqs == 0)
        return kOk;
    if (!a->q || !a->o || !a->table || !a->lens || !a->work || !aligned_to(a->work, 16) || !aligned_to(a->o, 16) ||
        (a->weight_out && a->weight_stride < (int64_t)a->max_pages * c->page_size))
        return kBadArg;
    Args g{};
    g.c = *c, g.a = *a;
    g.group = a->heads / c->kv_heads, g.cols = g.group * a->rows;
    while ((1 << g.page_log2) < c->page_size)
        ++g.page_log2;
    g.vec = aligned_to(a->q, 16) && (a->q_seq | a->q_row | a->q_head) % 8 == 0;
    const Work w = work_of(*c, *a);
    uint8_t *work = static_cast<uint8_t *>(a->work);
    g.part = reinterpret_cast<float *>(work);
    if (a->weight_out) {
        g.lse2 = reinterpret_cast<float *>(work + w.part);
        g.score = reinterpret_cast<float *>(work + w.part + w.lse2);
    }
    if (c->head_dim == 128)
        return g.cols <= 8 ? launch<128, 1>(g, stream) : launch<128, 2>(g, stream);
    return g.cols <= 8 ? launch<64, 1>(g, stream) : launch<64, 2>(g, stream);
}

} /* extern "C" */
