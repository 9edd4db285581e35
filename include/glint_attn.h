/* Attention between a decoder's q|k|v and o linears (libglint_encode.so; additive, no
 * counterpart in the reference's C ABI): causal attention over packed prompts, and a
 * paged key/value cache held in 4 bits with what fills, reads and shrinks it.
 *
 *   glint_attn_prompt_stream  o = softmax(scale q k^T) v over packed sequences
 *   glint_kv4_append_stream   new key/value rows, quantised into their slots
 *   glint_kv4_read_stream     slots back to BF16 rows
 *   glint_kv4_attn_stream     the newest tokens attend to their sequence's slots
 *   glint_kv4_evict_stream    a sequence's slots cut down to a budget, by weight
 *
 * q, k, v and o are BF16; head_dim is 64 or 128; heads is a multiple of kv_heads and
 * query head h reads key/value head h / (heads / kv_heads).  Strides are in elements,
 * a head's head_dim values are contiguous.  A row whose mask leaves no key gives o = 0
 * and lse = -inf.  Values in masked places (NaN and infinities included) never reach
 * a result; an infinity in v that a row sees is that column of its o, NaN where it sees
 * a NaN or infinities of both signs.  lse is the natural log of the sum of exponentials of the scaled scores.
 *
 * Return codes: 0 ok, -1 bad argument, -3 launch failure, -6 (GLINT_ERR_UNSUPPORTED)
 * a head_dim or page_size outside the lists here.  All calls are asynchronous on
 * `stream` and results are the same bits from run to run. */
#ifndef GLINT_ATTN_H_
#define GLINT_ATTN_H_
#include <cuda_runtime.h>
#include <stdint.h>

#include "glint_htile.h"
#ifdef __cplusplus
extern "C" {
#endif

/* Packed prompts.  Sequence s has the query tokens [cu_q[s], cu_q[s + 1]) and the
 * keys [cu_k[s], cu_k[s + 1]) (device int32, seqs + 1 entries, non-decreasing; values
 * are clamped to [0, q_tokens] and [0, k_tokens]).  Query i of Lq sees the keys
 * j <= i + Lk - Lq when causal, all Lk keys otherwise; where Lk < Lq the first
 * Lq - Lk rows see none.  o [q_tokens, heads, head_dim] with strides o_tok, o_head;
 * lse [heads, q_tokens] f32 or NULL.  Tokens outside every sequence are not written.
 * o may not overlap q, k or v.  work: glint_attn_prompt_work_bytes() of 16-byte
 * aligned device memory, the call's own until it completes, of any content; it lets few
 * queries with many keys share the GPU, and may be NULL.  16-byte aligned q, k and v
 * with positive strides that are multiples of 8, and scale > 0, take the tensor-core
 * kernel, anything else a plain one, which takes a hundred times as long (2048 tokens,
 * 32 / 8 heads of 128: 8.4 ms). */
typedef struct GlintAttnPrompt {
    const glint_bf16_t *q, *k, *v;
    glint_bf16_t *o;
    float *lse;
    const int *cu_q, *cu_k;
    void *work;
    int64_t q_tok, q_head, k_tok, k_head, v_tok, v_head, o_tok, o_head;
    int seqs, q_tokens, k_tokens, heads, kv_heads, head_dim, causal;
    float scale;
} GlintAttnPrompt;
int64_t glint_attn_prompt_work_bytes(const GlintAttnPrompt *a);
int glint_attn_prompt_stream(const GlintAttnPrompt *a, cudaStream_t stream);

/* The 4-bit cache.  Slots lie in pages of page_size (16, 32, 64 or 128) per head:
 *   code [pages, kv_heads, page_size, head_dim / 2] bytes, 16-byte aligned: element 2i of a
 *        row in the low nibble of byte i, element 2i + 1 in the high one; at head_dim 128
 *        the two 32-byte halves of a row are swapped in slots with slot & 2
 *   meta [pages, kv_heads, page_size, head_dim / 64, 2] BF16, 16-byte aligned: (step, lo) of
 *        each 64 values
 * Quantisation of 64 values x: lo = min x, step = BF16((max x - min x) / 15), code =
 * rint((x - lo) / step) clamped to 0..15 (0 where step is 0), all in f32 with IEEE
 * rounding; value = lo + step * code.  A block that holds a NaN or an infinity, or
 * whose range overflows, is stored as step 0, lo NaN: it reads as NaN.
 * A slot number is page * page_size + place in the page. */
typedef struct GlintKv4Cache {
    uint8_t *k_code;
    uint16_t *k_meta;
    uint8_t *v_code;
    uint16_t *v_meta;
    int pages, kv_heads, page_size, head_dim;
} GlintKv4Cache;

/* k, v [tokens, kv_heads, head_dim] into slots[t] (device int32; entries outside the
 * cache are skipped; no slot twice in one call). */
int glint_kv4_append_stream(const GlintKv4Cache *c, const glint_bf16_t *k, const glint_bf16_t *v, int64_t k_tok,
                            int64_t k_head, int64_t v_tok, int64_t v_head, const int *slots, int tokens,
                            cudaStream_t stream);
/* k_out, v_out [tokens, kv_heads, head_dim] BF16, contiguous and 16-byte aligned: the
 * values of slots[t], rounded to BF16; zeros for entries outside the cache. */
int glint_kv4_read_stream(const GlintKv4Cache *c, const int *slots, int tokens, glint_bf16_t *k_out,
                          glint_bf16_t *v_out, cudaStream_t stream);

/* Attention over the cache.  Sequence b has lens[b] slots (clamped to [0, max_pages *
 * page_size]), slot t in page table[b * max_pages + t / page_size] (a page outside the
 * cache masks its slots).  Its last `rows` slots are the query tokens' own: row i
 * sees the slots t < lens[b] - rows + i + 1.  q [seqs, rows, heads, head_dim] with
 * strides q_seq, q_row, q_head; o contiguous; lse [seqs, heads, rows] f32 or NULL.
 * weight_out (NULL: none) [seqs, kv_heads, weight_stride] f32: weight + the slot's
 * softmax weights summed over the head's query heads and rows; weight counts as zero
 * when NULL and in the newest `rows` slots; slots >= lens[b] are not written; weight
 * may be weight_out.  work: glint_kv4_attn_work_bytes() of 16-byte aligned device
 * memory, the call's own until it completes, of any content.
 * Limits: rows >= 1, heads / kv_heads * rows <= 256, seqs * kv_heads <= 65535, and
 * max_pages * page_size / 32 tiles times seqs * kv_heads (times a 16th of heads /
 * kv_heads * rows where that is above 16) in 31 bits. */
typedef struct GlintKv4Attn {
    const glint_bf16_t *q;
    glint_bf16_t *o;
    float *lse;
    const int *table, *lens;
    const float *weight;
    float *weight_out;
    void *work;
    int64_t q_seq, q_row, q_head, weight_stride;
    int seqs, rows, heads, max_pages;
    float scale;
} GlintKv4Attn;
int64_t glint_kv4_attn_work_bytes(const GlintKv4Cache *c, const GlintKv4Attn *a);
int glint_kv4_attn_stream(const GlintKv4Cache *c, const GlintKv4Attn *a, cudaStream_t stream);

/* Eviction, per sequence and key/value head: of L = lens[b] slots n = min(L, budget)
 * are kept, first those with pos >= seen[b] - recent, then those with the largest
 * weight (NaN the smallest), ties to the lowest slot.  The kept slots below n stay
 * where they are; the k-th kept slot from n on moves into the k-th free slot below n.
 * table and lens as above; weight, pos, weight_out, pos_out [seqs, kv_heads, stride].
 * kept [seqs, kv_heads, budget] int32: the slot each of the n now comes from (-1 from
 * n on); new_lens [seqs], which may not overlap lens or seen; weight_out and pos_out
 * get the kept slots' entries below n and may not overlap weight and pos.  Sequences do
 * not share the pages they move rows in.  Limits: 0 <= recent <= budget, budget >= 1, max_pages * page_size <=
 * 524288 and <= stride. */
typedef struct GlintKv4Evict {
    const int *table, *lens;
    const float *weight;
    const int *pos, *seen;
    int *kept, *new_lens;
    float *weight_out;
    int *pos_out;
    int64_t stride;
    int seqs, max_pages, budget, recent;
} GlintKv4Evict;
int glint_kv4_evict_stream(const GlintKv4Cache *c, const GlintKv4Evict *e, cudaStream_t stream);

#ifdef __cplusplus
}
#endif
#endif
