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
template <typename T> __device__ __forceinline__ T from_float(float v) { return T::encode(v); }
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

// The slope act'(pre) that the backward multiplies with is kept in fp32 for fp32, in 16 bits for the 16-bit types.  It lies in
// [-0.13, 1.13] for every activation, and a saturated unit's is tiny, so its numbers are even steps of 2^-15 down to
// 2^(BITS - 15) and from there floating point with BITS bits behind the leading one, to 2^-LEAST, below which steps are even again.
// Half a step is 2^-16 at most, and 2^-(BITS + 1) of the value: below the rounding of bf16 (BITS 8, down to 2^-55), one of
// fp16 (BITS 9, down to 2^-30, where its gradients end).  Zero and one are exact.  (fp16 itself is off by up to 2^-12 at one, which doubled the
// error of an fp16 gradient; steps of 2^-15 throughout lost units behind sigmoid(8) and tanh(5).)
// Codes: 0 .. FIRST - 1 floating, from FIRST on even, 0xc000 added where negative; 0xffff: NaN.
template <int BITS, int LEAST>
struct Slope16 {
  static constexpr int SHIFT = 23 - BITS, FIRST = (LEAST + BITS - 15) << BITS;
  static constexpr uint32_t BASE = (uint32_t)(127 - LEAST) << 23;                        // 2^-LEAST
  static constexpr float EVEN = 1.f / (float)(1 << (15 - BITS));                         // the smallest of the even steps
  static_assert(FIRST - (1 << BITS) + 36995 < 0xc000 && FIRST - (1 << BITS) + 4227 < 0x3fff, "slopes in [-0.129, 1.129]");
  unsigned short u;

  static __device__ __forceinline__ Slope16 encode(float v) {
    const float t = fabsf(v);
    // the low bits of 2^23 + FIRST - 2^BITS + t 2^15
    const uint32_t even = __float_as_uint(fmaf(t, 32768.f, 8388608.f + (float)(FIRST - (1 << BITS))));
    const uint32_t floating = (__float_as_uint(t + __uint_as_float(BASE)) - BASE + (1u << (SHIFT - 1))) >> SHIFT;
    uint32_t c = t >= EVEN ? even : floating;
    c |= (uint32_t)(__float_as_int(v) >> 31) & 0xc000u;
    return Slope16{(unsigned short)(v == v ? c & 0xffffu : 0xffffu)};
  }
  __device__ __forceinline__ float value() const {
    const bool below = u >= 0xc000u;
    const uint32_t c = below ? u - 0xc000u : u;
    const float even = fmaf(__uint_as_float(0x4b000000u | c), 1.f / 32768.f, (float)(-256.0 - (FIRST - (1 << BITS)) / 32768.0));
    const float floating = __uint_as_float((c << SHIFT) + BASE) - __uint_as_float(BASE);
    const float t = c >= (uint32_t)FIRST ? even : floating;
    return u == 0xffffu ? __uint_as_float(0x7fffffffu) : (below ? -t : t);
  }
};
template <int BITS, int LEAST>
__device__ __forceinline__ float to_float(Slope16<BITS, LEAST> s) { return s.value(); }
template <typename T> struct SlopeOf;
template <> struct SlopeOf<float> { typedef float type; };
template <> struct SlopeOf<__nv_bfloat16> { typedef Slope16<8, 55> type; };
template <> struct SlopeOf<__half> { typedef Slope16<9, 30> type; };

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
