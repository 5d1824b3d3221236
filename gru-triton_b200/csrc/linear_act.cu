// y = act(x W^T + bias) + residual and its gradients.
//
//   d = dy * act'(pre)   dx = d W   dW = d^T x   db = sum over rows of d   (the residual's gradient is dy)

#include "linear_act.cuh"

namespace b200gru {
namespace lin {

namespace {

constexpr int TILE = 64, DEPTH = 16, PAD = 4;

// C(m, n) = sum_k a(m, k) b(n, k) for operands given as functions; a 64 x 64 tile by 256 threads, 4 x 4 results each.
template <typename LoadA, typename LoadB, typename Store>
__device__ __forceinline__ void tile_product(int M, int N, int K, LoadA a, LoadB b, Store store) {
  __shared__ float sa[DEPTH][TILE + PAD], sb[DEPTH][TILE + PAD];
  const int m0 = blockIdx.y * TILE, n0 = blockIdx.x * TILE;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  float acc[4][4] = {};
  for (int k0 = 0; k0 < K; k0 += DEPTH) {
    for (int e = threadIdx.x; e < TILE * DEPTH; e += 256) {
      const int r = e / DEPTH, k = e % DEPTH;
      sa[k][r] = (m0 + r < M && k0 + k < K) ? a(m0 + r, k0 + k) : 0.f;
      sb[k][r] = (n0 + r < N && k0 + k < K) ? b(n0 + r, k0 + k) : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < DEPTH; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(sa[k][ty * 4 + i], sb[k][tx * 4 + j], acc[i][j]);
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (m0 + ty * 4 + i < M && n0 + tx * 4 + j < N) store(m0 + ty * 4 + i, n0 + tx * 4 + j, acc[i][j]);
}

template <typename T, int ACT>
__global__ void __launch_bounds__(256) linear_fwd_kernel(const b200gru_linear_args p) {
  const T* x = static_cast<const T*>(p.x);
  const T* W = static_cast<const T*>(p.W);
  tile_product(p.M, p.N, p.K, [&](int m, int k) { return to_float(x[(long long)m * p.ldx + k]); },
               [&](int n, int k) { return to_float(W[(long long)n * p.ldw + k]); },
               [&](int m, int n, float v) {
                 if (p.bias != nullptr) v += to_float(static_cast<const T*>(p.bias)[n]);
                 const Activated r = activate<ACT>(v);
                 if (p.slope != nullptr)
                   static_cast<typename SlopeOf<T>::type*>(p.slope)[(long long)m * p.lds + n] = from_float<typename SlopeOf<T>::type>(r.slope);
                 float y = r.y;
                 if (p.residual != nullptr) y += to_float(static_cast<const T*>(p.residual)[(long long)m * p.ldr + n]);
                 static_cast<T*>(p.y)[(long long)m * p.ldy + n] = from_float<T>(y);
               });
}

template <typename T>
__device__ __forceinline__ float grad_at(const b200gru_linear_args& p, int m, int n) {
  float d = to_float(static_cast<const T*>(p.dy)[(long long)m * p.lddy + n]);
  if (p.slope != nullptr) d *= to_float(static_cast<const typename SlopeOf<T>::type*>(p.slope)[(long long)m * p.lds + n]);
  return d;
}

template <typename T>
__global__ void __launch_bounds__(256) linear_dx_kernel(const b200gru_linear_args p) {
  const T* W = static_cast<const T*>(p.W);
  tile_product(p.M, p.K, p.N, [&](int m, int n) { return grad_at<T>(p, m, n); },
               [&](int k, int n) { return to_float(W[(long long)n * p.ldw + k]); },
               [&](int m, int k, float v) { static_cast<T*>(p.dx)[(long long)m * p.K + k] = from_float<T>(v); });
}

template <typename T>
__global__ void __launch_bounds__(256) linear_dw_kernel(const b200gru_linear_args p) {
  const T* x = static_cast<const T*>(p.x);
  tile_product(p.N, p.K, p.M, [&](int n, int m) { return grad_at<T>(p, m, n); },
               [&](int k, int m) { return to_float(x[(long long)m * p.ldx + k]); },
               [&](int n, int k, float v) { static_cast<T*>(p.dW)[(long long)n * p.K + k] = from_float<T>(v); });
}

template <typename T>
__global__ void __launch_bounds__(256) linear_db_kernel(const b200gru_linear_args p) {
  const int n = blockIdx.x * 256 + threadIdx.x;
  if (n >= p.N) return;
  float s = 0.f;
  for (int m = 0; m < p.M; ++m) s += grad_at<T>(p, m, n);
  static_cast<T*>(p.db)[n] = from_float<T>(s);
}

template <typename T>
int forward(const b200gru_linear_args& p, cudaStream_t st) {
  const dim3 grid(cdiv(p.N, TILE), cdiv(p.M, TILE));
  switch (p.activation) {
    case B200GRU_ACT_NONE: linear_fwd_kernel<T, B200GRU_ACT_NONE><<<grid, 256, 0, st>>>(p); break;
    case B200GRU_ACT_RELU: linear_fwd_kernel<T, B200GRU_ACT_RELU><<<grid, 256, 0, st>>>(p); break;
    case B200GRU_ACT_SILU: linear_fwd_kernel<T, B200GRU_ACT_SILU><<<grid, 256, 0, st>>>(p); break;
    case B200GRU_ACT_GELU: linear_fwd_kernel<T, B200GRU_ACT_GELU><<<grid, 256, 0, st>>>(p); break;
    case B200GRU_ACT_SIGMOID: linear_fwd_kernel<T, B200GRU_ACT_SIGMOID><<<grid, 256, 0, st>>>(p); break;
    case B200GRU_ACT_TANH: linear_fwd_kernel<T, B200GRU_ACT_TANH><<<grid, 256, 0, st>>>(p); break;
  }
  note_launch();
  return check_launch("linear_fwd_kernel");
}

template <typename T>
int backward(const b200gru_linear_args& p, cudaStream_t st) {
  if (p.dx != nullptr) { linear_dx_kernel<T><<<dim3(cdiv(p.K, TILE), cdiv(p.M, TILE)), 256, 0, st>>>(p); note_launch(); }
  if (p.dW != nullptr) { linear_dw_kernel<T><<<dim3(cdiv(p.K, TILE), cdiv(p.N, TILE)), 256, 0, st>>>(p); note_launch(); }
  if (p.db != nullptr) { linear_db_kernel<T><<<cdiv(p.N, 256), 256, 0, st>>>(p); note_launch(); }
  return check_launch("linear backward");
}

bool bad(const b200gru_linear_args* p) {
  return p == nullptr || p->M <= 0 || p->N <= 0 || p->K <= 0 || p->dtype < B200GRU_F32 || p->dtype > B200GRU_F16 ||
         p->activation < B200GRU_ACT_NONE || p->activation > B200GRU_ACT_TANH || p->x == nullptr || p->W == nullptr ||
         p->ldx < 0 || p->ldw < 0 || (p->slope != nullptr && p->lds < p->N);
}

}  // namespace
}  // namespace lin
}  // namespace b200gru

using namespace b200gru;

extern "C" {

size_t b200gru_linear_act_workspace_bytes(const b200gru_linear_args* p, int backward) {
  (void)backward;
  return lin::bad(p) ? (size_t)-1 : 0;
}

int b200gru_linear_act_forward(const b200gru_linear_args* p, void* stream) {
  if (lin::bad(p) || p->y == nullptr || p->ldy < p->N || (p->residual != nullptr && p->ldr < 0)) return B200GRU_INVALID_ARGUMENT;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (p->dtype == B200GRU_F32) return lin::forward<float>(*p, st);
  if (p->dtype == B200GRU_BF16) return lin::forward<__nv_bfloat16>(*p, st);
  return lin::forward<__half>(*p, st);
}

int b200gru_linear_act_backward(const b200gru_linear_args* p, void* stream) {
  if (lin::bad(p) || p->dy == nullptr || p->lddy < 0) return B200GRU_INVALID_ARGUMENT;
  if (p->activation != B200GRU_ACT_NONE && p->slope == nullptr) return B200GRU_INVALID_ARGUMENT;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (p->dtype == B200GRU_F32) return lin::backward<float>(*p, st);
  if (p->dtype == B200GRU_BF16) return lin::backward<__nv_bfloat16>(*p, st);
  return lin::backward<__half>(*p, st);
}

}  // extern "C"
