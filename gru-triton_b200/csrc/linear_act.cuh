// Product with bias, activation and residual: element types and activations.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "approx.cuh"
#include "common.cuh"

namespace b200gru {
namespace lin {

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

// The slope act'(pre) that the backward multiplies with is kept in fp32 for fp32 and in fp16 for the 16-bit types: it lies
// in [-0.13, 1.13] for every activation, so fp16 holds it to 11 bits (below 6e-5 to 3e-8 absolute) where bf16 would add an
// error as large as that of the output's own rounding.
template <typename T> struct SlopeOf { typedef __half type; };
template <> struct SlopeOf<float> { typedef float type; };

struct Activated { float y, slope; };

// sigmoid: e = exp(-v), s = 1 / (1 + e), 1 - s = e s; above e = 2^127 s and e s are zero.
// silu: v s, slope s (1 + v (1 - s)); v held inside [-100, 100] where an infinite one would meet a zero.
// tanh: f = exp(-2|v|): (1 - f) / (1 + f) with v's sign, slope 4 f / (1 + f)^2; below |v| = 1/8, where 1 - f cancels, the series
//   v - v^3/3 + 2 v^5/15 (next term 2e-7 of v at most).
// gelu: v Phi(v), slope Phi(v) + v phi(v), with Phi by formula 7.1.26 of Abramowitz and Stegun's handbook:
//   erfc(x) = (a1 t + .. + a5 t^5) exp(-x^2), t = 1 / (1 + 0.3275911 x), |error| <= 1.5e-7: half of that in Phi, a unit in the
//   last place of 1; exp(-v^2 / 2) serves phi as well.
template <int ACT>
__device__ __forceinline__ Activated activate(float v) {
  constexpr float LOG2E = 1.44269504f;
  Activated r;
  if (ACT == B200GRU_ACT_RELU) {
    r.y = max_nan(v, 0.f);
    r.slope = v > 0.f ? 1.f : 0.f;
  } else if (ACT == B200GRU_ACT_SILU || ACT == B200GRU_ACT_SIGMOID) {
    const float e = exp2_approx(min_nan(v * -LOG2E, 127.5f));
    const float s = rcp_approx(1.f + e), o = e * s;
    if (ACT == B200GRU_ACT_SIGMOID) {
      r.y = s;
      r.slope = s * o;
    } else {
      const float w = max_nan(v, -100.f);
      r.y = w * s;
      r.slope = s * fmaf(min_nan(w, 100.f), o, 1.f);
    }
  } else if (ACT == B200GRU_ACT_TANH) {
    const float f = exp2_approx(fabsf(v) * (-2.f * LOG2E)), q = rcp_approx(1.f + f);
    const float v2 = v * v, near0 = fmaf(fmaf(v2, 2.f / 15.f, -1.f / 3.f) * v2, v, v);
    r.y = fabsf(v) < 0.125f ? near0 : copysignf((1.f - f) * q, v);
    r.slope = 4.f * f * q * q;
  } else if (ACT == B200GRU_ACT_GELU) {
    const float w = max_nan(v, -100.f), c = min_nan(w, 100.f);
    const float E = exp2_approx(c * c * (-0.5f * LOG2E));
    const float t = rcp_approx(fmaf(fabsf(c), 0.3275911f * 0.70710678f, 1.f));
    float poly = fmaf(t, 1.061405429f, -1.453152027f);
    poly = fmaf(poly, t, 1.421413741f);
    poly = fmaf(poly, t, -0.284496736f);
    poly = fmaf(poly, t, 0.254829592f);
    const float tail = poly * t * (0.5f * E);                // 1 - Phi(|v|)
    const float cdf = c >= 0.f ? 1.f - tail : tail;
    r.y = w * cdf;
    r.slope = fmaf(c, 0.39894228f * E, cdf);
  } else {
    r.y = v;
    r.slope = 1.f;
  }
  return r;
}

__device__ __forceinline__ Activated activate_as(int act, float v) {
  switch (act) {
    case B200GRU_ACT_RELU: return activate<B200GRU_ACT_RELU>(v);
    case B200GRU_ACT_SILU: return activate<B200GRU_ACT_SILU>(v);
    case B200GRU_ACT_GELU: return activate<B200GRU_ACT_GELU>(v);
    case B200GRU_ACT_SIGMOID: return activate<B200GRU_ACT_SIGMOID>(v);
    case B200GRU_ACT_TANH: return activate<B200GRU_ACT_TANH>(v);
  }
  return activate<B200GRU_ACT_NONE>(v);
}

}  // namespace lin
}  // namespace b200gru
