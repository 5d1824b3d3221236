// Gated linear recurrence: the GRU update with gates from the input alone.
//
//   z = sigmoid(x)   n = tanh(c) or c   h_t = z h_{t-1} + (1 - z) n        gi[t,b,:] = (x[H], c[H])
//
// Each (row, unit) is a chain of its own, and its steps are affine maps h -> z h + u.

#include "gated_scan.cuh"

namespace b200gru {
namespace gated {

namespace {

constexpr int THREADS = 128;

template <typename T>
__global__ void __launch_bounds__(THREADS) gated_fwd_kernel(const Args a) {
  const long long chain = (long long)blockIdx.x * THREADS + threadIdx.x;
  if (chain >= (long long)a.B * a.H) return;
  const int b = (int)(chain / a.H), i = (int)(chain % a.H);
  const int len = row_length(a, b);
  const T* gp = static_cast<const T*>(a.gi) + (long long)b * a.gi_b + i;
  T* op = static_cast<T*>(a.out) + (long long)b * a.out_b + i;
  float h = a.h0 != nullptr ? a.h0[(long long)b * a.h0_b + i] : 0.f;
  for (int t = 0; t < a.T; ++t) {
    float o = 0.f;
    if (t < len) {
      if (a.states != nullptr && t % TILE == 0) a.states[((long long)(t / TILE) * a.B + b) * a.H + i] = h;
      const Gate g = gate(to_float(gp[(long long)t * a.gi_t]), to_float(gp[(long long)t * a.gi_t + a.H]), a.tanh);
      h = fmaf(g.z, h, g.keep * g.n);
      o = h;
    }
    op[(long long)t * a.out_t] = from_float<T>(o);
  }
  a.h_T[(long long)b * a.H + i] = h;
}

template <typename T>
__global__ void __launch_bounds__(THREADS) gated_bwd_kernel(const Args a) {
  const long long chain = (long long)blockIdx.x * THREADS + threadIdx.x;
  if (chain >= (long long)a.B * a.H) return;
  const int b = (int)(chain / a.H), i = (int)(chain % a.H);
  const int len = row_length(a, b);
  const T* gp = static_cast<const T*>(a.gi) + (long long)b * a.gi_b + i;
  const T* dp = a.dout != nullptr ? static_cast<const T*>(a.dout) + (long long)b * a.dout_b + i : nullptr;
  T* dg = static_cast<T*>(a.dgi) + (long long)b * a.dgi_b + i;
  for (int t = a.T - 1; t >= len; --t) {
    dg[(long long)t * a.dgi_t] = from_float<T>(0.f);
    dg[(long long)t * a.dgi_t + a.H] = from_float<T>(0.f);
  }
  float G = a.dh_T != nullptr ? a.dh_T[(long long)b * a.dh_b + i] : 0.f;
  float before[TILE];
  for (int t0 = (len - 1) / TILE * TILE; t0 >= 0 && len > 0; t0 -= TILE) {
    const int n = min(TILE, len - t0);
    float h = a.states[((long long)(t0 / TILE) * a.B + b) * a.H + i];
    for (int k = 0; k < n; ++k) {
      const long long at = (long long)(t0 + k) * a.gi_t;
      const Gate g = gate(to_float(gp[at]), to_float(gp[at + a.H]), a.tanh);
      before[k] = h;
      h = fmaf(g.z, h, g.keep * g.n);
    }
    for (int k = n - 1; k >= 0; --k) {
      const long long t = t0 + k;
      const Gate g = gate(to_float(gp[t * a.gi_t]), to_float(gp[t * a.gi_t + a.H]), a.tanh);
      const float gr = G + (dp != nullptr ? to_float(dp[t * a.dout_t]) : 0.f);
      dg[t * a.dgi_t] = from_float<T>(gr * (before[k] - g.n) * (g.z * g.keep));
      dg[t * a.dgi_t + a.H] = from_float<T>(gr * (g.keep * g.slope));
      G = g.z * gr;
    }
  }
  if (a.dh0 != nullptr) a.dh0[(long long)b * a.H + i] = G;
}

template <typename T>
__global__ void __launch_bounds__(THREADS) gated_step_kernel(const StepArgs a) {
  const long long chain = (long long)blockIdx.x * THREADS + threadIdx.x;
  if (chain >= (long long)a.B * a.H) return;
  const int b = (int)(chain / a.H), i = (int)(chain % a.H);
  const T* gp = static_cast<const T*>(a.gi) + (long long)b * a.gi_b + i;
  const Gate g = gate(to_float(gp[0]), to_float(gp[a.H]), a.tanh);
  const float h = fmaf(g.z, a.h[(long long)b * a.h_b + i], g.keep * g.n);
  a.h_new[(long long)b * a.hn_b + i] = h;
  static_cast<T*>(a.out)[(long long)b * a.H + i] = from_float<T>(h);
}

unsigned blocks_of(long long chains) { return (unsigned)((chains + THREADS - 1) / THREADS); }

}  // namespace

int launch_forward(const Args& a, int dtype, cudaStream_t st) {
  const unsigned n = blocks_of((long long)a.B * a.H);
  if (dtype == B200GRU_F32) gated_fwd_kernel<float><<<n, THREADS, 0, st>>>(a);
  else if (dtype == B200GRU_BF16) gated_fwd_kernel<__nv_bfloat16><<<n, THREADS, 0, st>>>(a);
  else gated_fwd_kernel<__half><<<n, THREADS, 0, st>>>(a);
  note_launch();
  return check_launch("gated_fwd_kernel");
}

int launch_backward(const Args& a, int dtype, cudaStream_t st) {
  const unsigned n = blocks_of((long long)a.B * a.H);
  if (dtype == B200GRU_F32) gated_bwd_kernel<float><<<n, THREADS, 0, st>>>(a);
  else if (dtype == B200GRU_BF16) gated_bwd_kernel<__nv_bfloat16><<<n, THREADS, 0, st>>>(a);
  else gated_bwd_kernel<__half><<<n, THREADS, 0, st>>>(a);
  note_launch();
  return check_launch("gated_bwd_kernel");
}

int launch_step(const StepArgs& a, int dtype, cudaStream_t st) {
  const unsigned n = blocks_of((long long)a.B * a.H);
  if (dtype == B200GRU_F32) gated_step_kernel<float><<<n, THREADS, 0, st>>>(a);
  else if (dtype == B200GRU_BF16) gated_step_kernel<__nv_bfloat16><<<n, THREADS, 0, st>>>(a);
  else gated_step_kernel<__half><<<n, THREADS, 0, st>>>(a);
  note_launch();
  return check_launch("gated_step_kernel");
}

}  // namespace gated
}  // namespace b200gru

using namespace b200gru;

namespace {

// Sizes and pointers that both directions need; every stride is non-negative.
int check_scan(const b200gru_gated_args* p) {
  if (p == nullptr || p->T <= 0 || p->B <= 0 || p->H <= 0 || p->gi == nullptr) return B200GRU_INVALID_ARGUMENT;
  if (p->dtype < B200GRU_F32 || p->dtype > B200GRU_F16) return B200GRU_INVALID_ARGUMENT;
  if (p->lengths != nullptr && p->length_bytes != 4 && p->length_bytes != 8) return B200GRU_INVALID_ARGUMENT;
  if ((long long)p->B * p->H > 0x7fffffffll || p->T > 0x40000000) return B200GRU_UNSUPPORTED;
  if (p->gi_t < 0 || p->gi_b < 0 || p->h0_b < 0) return B200GRU_INVALID_ARGUMENT;
  return B200GRU_OK;
}

gated::Args to_args(const b200gru_gated_args* p) {
  gated::Args a;
  a.T = p->T; a.B = p->B; a.H = p->H; a.tanh = p->candidate_tanh != 0;
  a.gi = p->gi; a.gi_t = p->gi_t; a.gi_b = p->gi_b;
  a.h0 = p->h0; a.h0_b = p->h0_b;
  a.lengths = p->lengths; a.length_bytes = p->length_bytes;
  a.out = p->out; a.out_t = p->out_t; a.out_b = p->out_b; a.h_T = p->h_T; a.states = p->states;
  a.dout = p->dout; a.dout_t = p->dout_t; a.dout_b = p->dout_b; a.dh_T = p->dh_T; a.dh_b = p->dh_b;
  a.dgi = p->dgi; a.dgi_t = p->dgi_t; a.dgi_b = p->dgi_b; a.dh0 = p->dh0;
  return a;
}

}  // namespace

extern "C" {

size_t b200gru_gated_states_bytes(int T, int B, int H) {
  if (T <= 0 || B <= 0 || H <= 0) return 0;
  return (size_t)cdiv(T, gated::TILE) * B * H * sizeof(float);
}

int b200gru_gated_scan_forward(const b200gru_gated_args* p, void* stream) {
  const int rc = check_scan(p);
  if (rc) return rc;
  if (p->out == nullptr || p->h_T == nullptr || p->out_t <= 0 || p->out_b <= 0) return B200GRU_INVALID_ARGUMENT;
  return gated::launch_forward(to_args(p), p->dtype, static_cast<cudaStream_t>(stream));
}

int b200gru_gated_scan_backward(const b200gru_gated_args* p, void* stream) {
  const int rc = check_scan(p);
  if (rc) return rc;
  if (p->states == nullptr || p->dgi == nullptr || p->dgi_t <= 0 || p->dgi_b <= 0) return B200GRU_INVALID_ARGUMENT;
  if (p->dout != nullptr && (p->dout_t < 0 || p->dout_b < 0)) return B200GRU_INVALID_ARGUMENT;
  return gated::launch_backward(to_args(p), p->dtype, static_cast<cudaStream_t>(stream));
}

int b200gru_gated_step(int dtype, int candidate_tanh, int B, int H, const void* gi, long long gi_b, const float* h,
                       long long h_b, void* out, float* h_new, long long hn_b, void* stream) {
  if (dtype < B200GRU_F32 || dtype > B200GRU_F16 || B <= 0 || H <= 0) return B200GRU_INVALID_ARGUMENT;
  if (gi == nullptr || h == nullptr || out == nullptr || h_new == nullptr) return B200GRU_INVALID_ARGUMENT;
  if (gi_b < 0 || h_b < 0 || hn_b < H) return B200GRU_INVALID_ARGUMENT;
  if ((long long)B * H > 0x7fffffffll) return B200GRU_UNSUPPORTED;
  gated::StepArgs a;
  a.B = B; a.H = H; a.tanh = candidate_tanh != 0;
  a.gi = gi; a.gi_b = gi_b; a.h = h; a.h_b = h_b; a.out = out; a.h_new = h_new; a.hn_b = hn_b;
  return gated::launch_step(a, dtype, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
