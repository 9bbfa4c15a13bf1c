// The activations of the gated feed-forward block and the words that a training
// forward keeps of them, shared by the kernels for many and for few tokens.
#pragma once

#include <math_constants.h>

#include "tc_pair.cuh"

namespace dsalt {
namespace ffn {

// ½·erfc(z) for z ≥ 0 given e = exp(−z²): e·t·P(t), t = 1 / (1 + z/2), with P a
// polynomial fitted to ½·erfcx(z) / t on t in (0, 1] (least squares in relative error at
// Chebyshev points, own coefficients; largest relative error 4.5e-7, in fp32 arithmetic 6.9e-7).
__device__ __forceinline__ float half_erfc(float z, float e) {
  const float t = sm100::fast_rcp(fmaf(0.5f, z, 1.f));
  float p = -0.0219386164f;
  p = fmaf(p, t, 0.110518053f);
  p = fmaf(p, t, -0.188654438f);
  p = fmaf(p, t, 0.0882052481f);
  p = fmaf(p, t, 0.0138631025f);
  p = fmaf(p, t, 0.0928735211f);
  p = fmaf(p, t, 0.123026401f);
  p = fmaf(p, t, 0.141059607f);
  p = fmaf(p, t, 0.141047329f);
  return e * (t * p);
}

// act(g) and act'(g).  exp and the reciprocal are the fast ones.  Relative error of act
// below 2^-19 for |g| <= 4 (silu 3e-7, gelu 1.1e-6, gelu_tanh 1.5e-6); towards −∞ it grows
// with the exponent's argument, whose rounding in fp32 alone is 2^-24 of its size: 3.5e-6
// for silu at −87, 7e-6 for gelu at −12 and 5e-6 for gelu_tanh at −9, the ends of bf16's
// range.  The results are rounded to 16 or cut to 24 bits next (2^-8, 2^-15).
template <int ACT>
__device__ __forceinline__ void act_pair(float g, float& a, float& da) {
  constexpr float kLog2e = 1.4426950409f;
  if constexpr (ACT == DSALT_ACT_SILU) {
    const float sig = sm100::fast_rcp(1.f + sm100::fast_exp2(-kLog2e * g));
    a = g * sig;
    da = fmaf(a, 1.f - sig, sig);
  } else if constexpr (ACT == DSALT_ACT_GELU) {
    // Φ(g) = ½·erfc(−g/√2); its density is e / √(2π) with the same e = exp(−g²/2).  From
    // |g| = 20 on e is 0 in fp32 (and g² must not overflow)
    const float z = fminf(fabsf(g), 20.f);
    const float e = sm100::fast_exp2(-0.5f * kLog2e * z * z);
    const float tail = half_erfc(0.7071067812f * z, e);
    const float cdf = g < 0.f ? tail : 1.f - tail;
    a = g * cdf;
    da = fmaf(g * 0.3989422804f, e, cdf);
  } else {
    // ½(1 + tanh z) = σ(2z), ½(1 − tanh² z) = 2σ(1 − σ), z = √(2/π)(g + 0.044715 g³)
    const float g2 = g * g;
    const float z2 = 1.5957691216f * g * fmaf(0.044715f, g2, 1.f);
    const float sig = sm100::fast_rcp(1.f + sm100::fast_exp2(-kLog2e * z2));
    const float w = sig * (1.f - sig);
    a = g * sig;
    da = sig + (w > 0.f ? g * w * 1.5957691216f * fmaf(0.134145f, g2, 1.f) : 0.f);
  }
}

__device__ __forceinline__ float2 unpack2(uint32_t w, bool bf16) {
  if (bf16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
// What v's rounding to the 16-bit value `high` leaves.  0 beside an infinity or NaN, which
// v − high would meet with an infinity of the other sign.
__device__ __forceinline__ float rounding_rest(float v, float high) {
  return fabsf(high) < CUDART_INF_F ? v - high : 0.f;
}
// Upper 16 bits of fp32 x (low half) and y: the words of a and b.
__device__ __forceinline__ uint32_t upper16(float x, float y) {
  return __byte_perm(__float_as_uint(x), __float_as_uint(y), 0x7632);
}
// Byte 1 of a0, b0, a1, b1: the words of ab.
__device__ __forceinline__ uint32_t next8(float a0, float b0, float a1, float b1) {
  return __byte_perm(__byte_perm(__float_as_uint(a0), __float_as_uint(b0), 0x0051),
                     __byte_perm(__float_as_uint(a1), __float_as_uint(b1), 0x0051), 0x5410);
}

}  // namespace ffn
}  // namespace dsalt
