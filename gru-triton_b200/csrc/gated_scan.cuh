// Gated linear recurrence: arguments, gate arithmetic, element types.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace b200gru {
namespace gated {

constexpr int TILE = 64;       // steps between two kept states

// Strides in elements; the units of a row are contiguous.  h0, dout, dh_T: NULL = zeros.
struct Args {
  int T, B, H;
  bool tanh;                   // n = tanh(c), else n = c
  const void* gi; long long gi_t, gi_b;
  const float* h0; long long h0_b;
  const void* lengths; int length_bytes;       // per row, 4 or 8 bytes each; NULL = T
  void* out; long long out_t, out_b;
  float* h_T;                  // [B][H]
  float* states;               // [ceil(T / TILE)][B][H]: state before step k * TILE; NULL = not kept
  const void* dout; long long dout_t, dout_b;
  const float* dh_T; long long dh_b;
  void* dgi; long long dgi_t, dgi_b;
  float* dh0;                  // [B][H] or NULL
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

struct Gate {
  float z, keep, n, slope;     // sigmoid(x), 1 - z, candidate, dn / dc
};

// With e = exp(-|x|) and f = exp(-2|c|) in [0, 1]:
//   the smaller of z and 1 - z is e / (1 + e), to full relative precision; the larger is 1 minus it, so that the two add to
//   one to a rounding of the larger and a state that holds for hundreds of steps does not drift;
//   tanh|c| = (1 - f) / (1 + f), dn/dc = 4 f / (1 + f)^2; below |c| = 1/8, where 1 - f cancels, the series
//   c - c^3/3 + 2 c^5/15 (next term 17/315 c^7: 2e-7 of c at most).
// Both quotients come from one reciprocal, of (1 + e)(1 + f) in [1, 4].  A NaN in one argument stays out of the other's gate.
template <bool TANH>
__device__ __forceinline__ Gate gate(float x, float c) {
  Gate g;
  const float e = expf(-fabsf(x));
  const float d = 1.f + e;
  if (TANH) {
    const float f = expf(-2.f * fabsf(c));
    const float de = fminf(d, 2.f), df = fminf(1.f + f, 2.f);
    const float r = __frcp_rn(de * df);
    const float s = e * (r * df);
    const float q = r * de;
    const float c2 = c * c;
    const float near0 = fmaf(fmaf(c2, 2.f / 15.f, -1.f / 3.f) * c2, c, c);
    const float far = copysignf((1.f - f) * q, c);
    g.n = fabsf(c) < 0.125f ? near0 : far;
    g.slope = 4.f * f * q * q;
    g.z = x >= 0.f ? 1.f - s : s;
    g.keep = x >= 0.f ? s : 1.f - s;
  } else {
    const float s = e * __frcp_rn(d);
    g.n = c;
    g.slope = 1.f;
    g.z = x >= 0.f ? 1.f - s : s;
    g.keep = x >= 0.f ? s : 1.f - s;
  }
  return g;
}

int launch_forward(const Args& a, int dtype, cudaStream_t st);
int launch_backward(const Args& a, int dtype, cudaStream_t st);
int launch_step(const StepArgs& a, int dtype, cudaStream_t st);

}  // namespace gated
}  // namespace b200gru
