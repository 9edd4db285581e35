/* The activation of a gated feed-forward projection, shared by the H-TILE kernels whose
 * epilogue applies it (htile_gemv.cu, htile_decode.cu, htile_gemm.cu). */
#ifndef GLINT_B200_GATED_CUH_
#define GLINT_B200_GATED_CUH_

#include "../../include/glint_htile.h"

namespace glint {

/* What the H-TILE kernels' gated epilogues take.  Against activations in FP16 (see htile_gated.cu) a product's sums
 * are of x[m] / x_scale[m] and, where weights carry their absmax into the tensor cores, of W[n] * row_scale[n].  Both
 * are written by the kernel before, beside which the products may already run: behind griddepcontrol.wait they are read by
 * plain loads, never as data that stays the same for the kernel's whole life (__ldg, a const __restrict__ pointer). */
struct GatedEpilogue {
    int act;
    const float *x_scale;   /* [M] powers of two */
    const float *row_scale; /* [N] powers of two */
};

/* act(g) u, act(g) = g / (1 + exp(-z)): z = g (silu), or 2 sqrt(2 / pi) (g + 0.044715 g^3), which
 * makes it g (1 + tanh(z / 2)) / 2.  With e = exp(-|z|), at most 1, that is g / (1 + e), or g / (1 + e) e below 0: nothing
 * overflows, and the tail comes out down to f32's least value.  The fast exponential is within (2 + 1.18 |z|) 2^-23 of
 * its value (2^-16 at z = -87), the division, by 1 to 2, within 2^-22: far inside the result's rounding. */
__device__ __forceinline__ float gated_value(float g, float u, int act)
{
    const float z = act == GLINT_ACT_GELU_TANH ? g * fmaf(0.0713548162726f * g, g, 1.59576912160573f) : g;
    const float e = __expf(-fabsf(z)), h = __fdividef(g, 1.f + e);
    return (z < 0.f ? h * e : h) * u;
}

} // namespace glint

#endif
