// Shared by the 8-bit kernels: blocks of 128 values and the rule that quantises one.
#pragma once
#include <cuda_fp8.h>

#include "fp8_cut.h"
#include "hb_common.cuh"

namespace hb {

// ---- quantisation -------------------------------------------------------------------------------------------------------------------
// The largest magnitude of a block as the bits of a float: they order like the magnitudes, infinities and NaN last.  From it the scale that
// is stored (amax / 448) and the code of each value: e4m3(v · 448 / amax).  v · 448 is an fp32 product (of a bf16 value exact); the quotient is worked out
// from the reciprocal with one residual step, which gives the correctly rounded one (Markstein, "Computation of elementary functions on the
// IBM RISC System/6000 processor", 1990), and exactly the quotient where fp32 holds it, so a tie between two codes is seen as one.
// Blocks of very small or very large values are brought to the middle of the range by a power of two first: nothing over- or underflows
// that could be more than a zero code.
struct F8Block {
  float f448, f, d, r; bool live;                      // f: the power of two; d = amax·f, r = 1 / d
  __device__ __forceinline__ float init(uint32_t bits) {   // returns the scale
    const float amax = __uint_as_float(bits);
    live = bits > 0u && bits < 0x7f800000u;
    f = amax < 0x1p-60f ? 0x1p64f : amax > 0x1p60f ? 0x1p-64f : 1.f;
    f448 = f * 448.f;
    d = __fmul_rn(amax, f); r = live ? __fdiv_rn(1.f, d) : 0.f;                // (__frcp_rn, the same number, is a call: gate/up of 128-row tiles 10 % slower)
    if (bits >= 0x7f800000u) return __int_as_float(0x7fc00000);
    const float q = __fmul_rn(amax, 1.f / 448.f);
    return amax > 0x1p-90f ? __fmaf_rn(__fmaf_rn(-q, 448.f, amax), 1.f / 448.f, q) : __fdiv_rn(amax, 448.f);
  }
  __device__ __forceinline__ float quotient(float v) const {   // (a zero comes out as +0)
    const float t = __fmul_rn(v, f448), q = __fmul_rn(t, r);
    return __fmaf_rn(__fmaf_rn(-q, d, t), r, q);
  }
  __device__ __forceinline__ uint32_t pair(float a, float b) const {   // codes of two values, the first in the low byte
    uint16_t o;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(o) : "f"(quotient(b)), "f"(quotient(a)));
    return live ? (uint32_t)o : 0u;
  }
};
__device__ __forceinline__ uint32_t f8_mag(float v) { return __float_as_uint(v) & 0x7fffffffu; }

}  // namespace hb
