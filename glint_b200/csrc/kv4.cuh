/* The 4-bit key/value cache's layout, shared by the kernels that fill, read and
 * shrink it (kv4_cache.cu) and the attention over it (kv4_attn.cu).
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

} // namespace glint

#endif
