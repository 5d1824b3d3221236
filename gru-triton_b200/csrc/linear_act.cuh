// Product with bias, activation and residual: element types and activations.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

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

// exp(-|v|) never overflows; s is the smaller of sigmoid(v) and 1 - sigmoid(v).
template <int ACT>
__device__ __forceinline__ Activated activate(float v) {
  Activated r;
  if (ACT == B200GRU_ACT_RELU) {
    r.y = v > 0.f ? v : (v != v ? v : 0.f);
    r.slope = v > 0.f ? 1.f : 0.f;
  } else if (ACT == B200GRU_ACT_SILU || ACT == B200GRU_ACT_SIGMOID) {
    const float e = expf(-fabsf(v)), q = __frcp_rn(1.f + e), lo = e * q;
    const float s = v >= 0.f ? q : lo, o = v >= 0.f ? lo : q;          // sigmoid(v), 1 - sigmoid(v)
    if (ACT == B200GRU_ACT_SIGMOID) {
      r.y = s;
      r.slope = s * o;
    } else {
      // an infinite v: v s = +inf or 0, slope 1 or 0
      const float w = fabsf(v) <= 3.0e38f ? v : (v != v ? v : (v > 0.f ? v : 0.f));
      r.y = w * s;
      r.slope = fabsf(v) < 100.f || v != v ? s * fmaf(v, o, 1.f) : (v > 0.f ? 1.f : 0.f);
    }
  } else if (ACT == B200GRU_ACT_TANH) {
    const float y = tanhf(v);
    const float f = expf(-2.f * fabsf(v)), q = __frcp_rn(1.f + f);
    r.y = y;
    r.slope = 4.f * f * q * q;
  } else if (ACT == B200GRU_ACT_GELU) {
    // v Phi(v); Phi through erfc keeps its relative precision on the negative side
    const float cdf = 0.5f * erfcf(v * -0.70710678f);
    const float pdf = 0.39894228f * expf(-0.5f * v * v);
    const float w = v > -20.f ? v : (v != v ? v : 0.f);                // Phi(-20) = 3e-89
    r.y = w * cdf;
    r.slope = fabsf(v) < 20.f || v != v ? fmaf(v, pdf, cdf) : (v > 0.f ? 1.f : 0.f);
  } else {
    r.y = v;
    r.slope = 1.f;
  }
  return r;
}

}  // namespace lin
}  // namespace b200gru
