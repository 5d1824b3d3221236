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

// The slope act'(pre) that the backward multiplies with is kept in fp32 for fp32.  For the 16-bit types it is a fixed-point number:
// it lies in [-0.13, 1.13] for every activation, so 16 bits hold it to 2^-16, and zero and one exactly.  (As fp16 it was off by
// up to 2^-12 at one, which doubled the error of an fp16 gradient.)  0xffff: NaN.
struct Slope16 { unsigned short u; };
__device__ __forceinline__ float to_float(Slope16 s) {
  const float v = fmaf(__uint_as_float(0x4b000000u | s.u), 1.f / 32768.f, -256.5f);      // (2^23 + u) 2^-15 - 256.5 = u 2^-15 - 0.5
  return s.u == 0xffffu ? __uint_as_float(0x7fffffffu) : v;
}
template <> __device__ __forceinline__ Slope16 from_float<Slope16>(float v) {            // the low bits of 2^23 + 2^14 + v 2^15
  return Slope16{(unsigned short)(__float_as_uint(fmaf(v, 32768.f, 8404992.f)) & 0xffffu)};
}
template <typename T> struct SlopeOf { typedef Slope16 type; };
template <> struct SlopeOf<float> { typedef float type; };

// Two values behind the activation, and its slopes there.
struct Activated2 {
  P2 y, slope;
};

// sigmoid: e = exp(-v), s = 1 / (1 + e), 1 - s = e s.  silu: v s, slope s (1 + v (1 - s)).
// tanh: f = exp(-2|v|): (1 - f) / (1 + f) with v's sign, slope 4 f / (1 + f)^2; below |v| = 1/8, where 1 - f cancels, the series
//   v - v^3/3 + 2 v^5/15 (next term 2e-7 of v at most).
// gelu: v Phi(v), slope Phi(v) + v phi(v), with Phi by formula 7.1.26 of Abramowitz and Stegun's handbook:
//   erfc(x) = (a1 t + .. + a5 t^5) exp(-x^2), t = 1 / (1 + 0.3275911 x), |error| <= 1.5e-7: half of that in Phi, a unit in the
//   last place of 1; exp(-v^2 / 2) serves phi as well.
// Values far out reach the limits without an infinity times zero (e above 2^126 counts as 2^126 in e s).
template <int ACT>
__device__ __forceinline__ Activated2 activate(P2 v) {
  constexpr float LOG2E = 1.44269504f;
  Activated2 r;
  const float2 at = split(v);
  const P2 one = both(1.f);
  if (ACT == B200GRU_ACT_RELU) {
    r.y = pair(max_nan(at.x, 0.f), max_nan(at.y, 0.f));
    r.slope = pair(at.x > 0.f ? 1.f : 0.f, at.y > 0.f ? 1.f : 0.f);
  } else if (ACT == B200GRU_ACT_SILU || ACT == B200GRU_ACT_SIGMOID) {
    const float2 e = make_float2(exp2_approx(at.x * -LOG2E), exp2_approx(at.y * -LOG2E));
    const P2 s = pair(rcp_approx(1.f + e.x), rcp_approx(1.f + e.y));
    const P2 o = mul2(pair(min_nan(e.x, 8.507059e37f), min_nan(e.y, 8.507059e37f)), s);
    if (ACT == B200GRU_ACT_SIGMOID) {
      r.y = s;
      r.slope = mul2(s, o);
    } else {
      r.y = mul2(v, s);
      r.slope = mul2(s, fma2(v, o, one));
    }
  } else if (ACT == B200GRU_ACT_TANH) {
    const P2 f = pair(exp2_approx(fabsf(at.x) * (-2.f * LOG2E)), exp2_approx(fabsf(at.y) * (-2.f * LOG2E)));
    const float2 d = split(add2(one, f));
    const P2 q = pair(rcp_approx(d.x), rcp_approx(d.y));
    const P2 v2 = mul2(v, v);
    const float2 near0 = split(fma2(mul2(fma2(v2, both(2.f / 15.f), both(-1.f / 3.f)), v2), v, v));
    const float2 far = split(mul2(sub2(one, f), q));
    r.y = pair(fabsf(at.x) < 0.125f ? near0.x : copysignf(far.x, at.x), fabsf(at.y) < 0.125f ? near0.y : copysignf(far.y, at.y));
    r.slope = mul2(mul2(mul2(f, q), q), both(4.f));
  } else if (ACT == B200GRU_ACT_GELU) {
    const float2 h = split(mul2(mul2(v, v), both(-0.5f * LOG2E)));
    const P2 E = pair(exp2_approx(h.x), exp2_approx(h.y));
    const P2 t = pair(rcp_approx(fmaf(fabsf(at.x), 0.3275911f * 0.70710678f, 1.f)),
                      rcp_approx(fmaf(fabsf(at.y), 0.3275911f * 0.70710678f, 1.f)));
    P2 poly = fma2(t, both(0.5f * 1.061405429f), both(0.5f * -1.453152027f));
    poly = fma2(poly, t, both(0.5f * 1.421413741f));
    poly = fma2(poly, t, both(0.5f * -0.284496736f));
    poly = fma2(poly, t, both(0.5f * 0.254829592f));
    const P2 tail = mul2(mul2(poly, t), E);                  // 1 - Phi(|v|)
    const float2 lo = split(tail), hi = split(sub2(one, tail));
    const P2 cdf = pair(at.x >= 0.f ? hi.x : lo.x, at.y >= 0.f ? hi.y : lo.y);
    r.y = mul2(v, cdf);
    r.slope = fma2(v, mul2(E, both(0.39894228f)), cdf);
  } else {
    r.y = v;
    r.slope = one;
  }
  return r;
}

__device__ __forceinline__ Activated2 activate_as(int act, P2 v) {
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
