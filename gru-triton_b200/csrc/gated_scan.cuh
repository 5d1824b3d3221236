// Gated linear recurrence: arguments, gate arithmetic, element types.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "approx.cuh"
#include "common.cuh"

namespace b200gru {
namespace gated {

// Strides in elements; the units of a row are contiguous.  h0, dout, dh_T: NULL = zeros.
struct Args {
  int T, B, H;
  bool tanh;                   // n = tanh(c), else n = c
  const void* gi; long long gi_t, gi_b;
  const float* h0; long long h0_b;
  const void* lengths; int length_bytes;       // per row, 4 or 8 bytes each; NULL = T
  void* out; long long out_t, out_b;
  float* h_T;                  // [B][H]
  float* states;               // [tiles][B][H]: state before each tile (see tile_steps); NULL = not kept
  const void* dout; long long dout_t, dout_b;
  const float* dh_T; long long dh_b;
  void* dgi; long long dgi_t, dgi_b;
  float* dh0;                  // [B][H] or NULL
  // in bytes, ready to be added to an address (scaled in the loop, for want of registers, they cost ten instructions of 70)
  long long out_step, dgi_step, half;          // a step of out, of dgi; from x's to c's half of a row
};

struct StepArgs {
  int B, H;
  bool tanh;
  const void* gi; long long gi_b;
  const float* h; long long h_b;
  void* out;                   // [B][H]
  float* h_new; long long hn_b;
};

// Steps of row b: its length, held inside [0, T].
__device__ __forceinline__ int row_length(const Args& a, int b) {
  if (a.lengths == nullptr) return a.T;
  const long long n = a.length_bytes == 8 ? static_cast<const long long*>(a.lengths)[b] : static_cast<const int*>(a.lengths)[b];
  return (int)(n < 0 ? 0 : (n > a.T ? a.T : n));
}

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

// The constants of the packed instructions, which take registers alone.  Behind a volatile move they stay in theirs; the
// compiler would otherwise build each pair anew at each use, seven moves beside the 24 instructions of an element.
struct Constants {
  P2 one, cubic, fifth;
};
__device__ __forceinline__ P2 pinned(float v) {
  P2 p;
  asm volatile("mov.b64 %0, {%1, %1};" : "=l"(p.v) : "f"(v));
  return p;
}
__device__ __forceinline__ Constants constants() { return {pinned(1.f), pinned(-1.f / 3.f), pinned(2.f / 15.f)}; }

// 2^(|v| * scale), scale < 0: in [0, 1].
__device__ __forceinline__ P2 falling2(P2 v, float scale) {
  const float2 t = split(v);
  return pair(exp2_approx(fabsf(t.x) * scale), exp2_approx(fabsf(t.y) * scale));
}
__device__ __forceinline__ P2 reciprocal2(P2 v) {
  const float2 f = split(v);
  return pair(rcp_approx(f.x), rcp_approx(f.y));
}

// Gates of two units: z, keep = 1 - z, n and its slope.
struct Gates {
  P2 z, keep, n, slope;
};

// With e = exp(-|x|) and f = exp(-2|c|): the smaller of z and 1 - z is e / (1 + e), the larger one minus that.  So both have full
// relative precision, a closed gate (z of 1e-10) as well as an open one, and the two add to one to a rounding, so that a state
// which holds for hundreds of steps does not drift.  tanh |c| = (1 - f) / (1 + f), dn/dc = 4 f / (1 + f)^2.
// Both quotients come from one reciprocal, of (1 + e)(1 + f) <= 4: three special-function values instead of four, of which an SM
// has 16 a cycle.  APART: a NaN of c stays out of x's gate (in the forward both make the state NaN from there on; in the
// backward the gate alone carries the gradient to earlier steps).  Below |c| = 1/8, where 1 - f cancels, the series
// c - c^3/3 + 2 c^5/15 (next term 17/315 c^7: 2e-7 of c at most).
template <bool TANH, bool APART>
__device__ __forceinline__ Gates gates(P2 x, P2 c, const Constants& k) {
  constexpr float LOG2E = 1.44269504f;
  Gates g;
  const P2 e = falling2(x, -LOG2E);
  const P2 d = add2(k.one, e);
  P2 s;
  if (TANH) {
    const P2 f = falling2(c, -2.f * LOG2E);
    P2 q = add2(k.one, f);
    if (APART) {
      const float2 t = split(q);
      q = pair(fminf(t.x, 2.f), fminf(t.y, 2.f));
    }
    const P2 r = reciprocal2(mul2(d, q));
    s = mul2(r, q);
    q = mul2(r, d);
    const P2 c2 = mul2(c, c);
    const float2 far = split(mul2(sub2(k.one, f), q)), near0 = split(fma2(mul2(fma2(c2, k.fifth, k.cubic), c2), c, c)), at = split(c);
    g.n = pair(fabsf(at.x) < 0.125f ? near0.x : copysignf(far.x, at.x), fabsf(at.y) < 0.125f ? near0.y : copysignf(far.y, at.y));
    const P2 fq = mul2(mul2(f, q), q), twice = add2(fq, fq);
    g.slope = add2(twice, twice);
  } else {
    s = reciprocal2(d);
    g.n = c;
    g.slope = k.one;
  }
  const P2 small = mul2(e, s);
  const float2 lo = split(small), hi = split(sub2(k.one, small)), at = split(x);
  g.z = pair(at.x < 0.f ? lo.x : hi.x, at.y < 0.f ? lo.y : hi.y);
  g.keep = pair(at.x < 0.f ? hi.x : lo.x, at.y < 0.f ? hi.y : lo.y);
  return g;
}

// Steps of a tile for these sizes.
int tile_steps(int T, int B, int H);
int launch_forward(const Args& a, int dtype, cudaStream_t st);
int launch_backward(const Args& a, int dtype, cudaStream_t st);
int launch_step(const StepArgs& a, int dtype, cudaStream_t st);

}  // namespace gated
}  // namespace b200gru
