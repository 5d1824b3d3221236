// y = act(x W^T + bias) + residual and its gradients.
//
//   d = dy * act'(pre)   dx = d W   dW = d^T x   db = sum over rows of d   (the residual's gradient is dy)
//
// Three products of one tensor-core kernel (linear_gemm.cuh); here: the operands' preparation, the joining of K slices, the
// kernel for a few rows, and who runs when.
//
// fp32 operands become two fp16 planes scaled by powers of two.  A scale has to factor out of the sum, so it follows the index
// that is not summed: forward, rows of x and rows of W; dx, rows of d (the scales of W's rows, which are summed here,
// folded into d first); dW, columns of d (the scales of x's rows folded in first).  So x and W need one form each.

#include "linear_gemm.cuh"

namespace b200gru {
namespace lin {

namespace {

inline long long pad8(long long n) { return (n + 7) / 8 * 8; }

// ---- operands ------------------------------------------------------------------------------------------
// Rows that TMA cannot reach where they lie (odd widths, bases or strides) are copied to padded rows, and back.
template <typename T>
__global__ void __launch_bounds__(256) copy_rows_kernel(const T* __restrict__ src, long long ld, T* __restrict__ dst, long long dld,
                                                        int rows, int cols) {
  pdl_launch_dependents();
  pdl_wait();
  const int row = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (row >= rows) return;
  const T* s = src + (long long)row * ld;
  T* d = dst + (long long)row * dld;
#pragma unroll 4
  for (int c = lane; c < cols; c += 32) d[c] = s[c];
}

struct HiLo { __half hi, lo; };
__device__ __forceinline__ HiLo hi_lo(float x) {
  HiLo r;
  r.hi = __float2half_rn(x);
  r.lo = __float2half_rn(x - __half2float(r.hi));
  return r;
}

// Four values of a row from column c on; zeros behind its end.
template <bool VEC>
__device__ __forceinline__ float4 four(const float* row, int c, int cols) {
  if (VEC) return c < cols ? *reinterpret_cast<const float4*>(row + c) : make_float4(0.f, 0.f, 0.f, 0.f);
  return make_float4(c < cols ? row[c] : 0.f, c + 1 < cols ? row[c + 1] : 0.f, c + 2 < cols ? row[c + 2] : 0.f, c + 3 < cols ? row[c + 3] : 0.f);
}
__device__ __forceinline__ void store_planes(__half* d, long long plane, float4 v) {
  const HiLo a = hi_lo(v.x), b = hi_lo(v.y), c = hi_lo(v.z), e = hi_lo(v.w);
  __half h[4] = {a.hi, b.hi, c.hi, e.hi}, l[4] = {a.lo, b.lo, c.lo, e.lo};
  *reinterpret_cast<uint2*>(d) = *reinterpret_cast<uint2*>(h);
  *reinterpret_cast<uint2*>(d + plane) = *reinterpret_cast<uint2*>(l);
}
__device__ __forceinline__ float largest(float4 v, float m) {
  return fmaxf(fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w))), m);
}
__device__ __forceinline__ float4 times(float4 v, float s) { return make_float4(v.x * s, v.y * s, v.z * s, v.w * s); }
__device__ __forceinline__ float4 times(float4 v, float4 s) { return make_float4(v.x * s.x, v.y * s.y, v.z * s.z, v.w * s.w); }

// Rows into two fp16 planes each, scaled so that a row's largest element lies in [2^14, 2^15): 22 significant bits of all elements
// down to 2^-17 of it.  One warp per row; the second read of the row comes from L1.  Up to two matrices in a launch.
struct SplitArgs {
  const float* src; long long ld;
  __half* dst; long long dld, plane;
  int rows, cols, vec;
  float* inv;
};
template <bool VEC>
__device__ __forceinline__ void split_row(const SplitArgs& a, int row, int lane) {
  const float* s = a.src + (long long)row * a.ld;
  float mx = 0.f;
#pragma unroll 4
  for (int c = lane * 4; c < a.cols; c += 128) mx = largest(four<VEC>(s, c, a.cols), mx);
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
  float scale, back;
  pow2_row_scale(mx, &scale, &back);
  if (lane == 0) a.inv[row] = back;
  __half* d = a.dst + (long long)row * a.dld;
#pragma unroll 4
  for (int c = lane * 4; c < a.dld; c += 128) store_planes(d + c, a.plane, times(four<VEC>(s, c, a.cols), scale));
}
__global__ void __launch_bounds__(256) split_rows_kernel(const SplitArgs one, const SplitArgs two) {
  pdl_launch_dependents();
  pdl_wait();
  long long row = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  const bool first = row < one.rows;
  const SplitArgs& a = first ? one : two;
  if (!first) row -= one.rows;
  if (row >= a.rows) return;
  if (a.vec) split_row<true>(a, (int)row, lane);
  else split_row<false>(a, (int)row, lane);
}

// ---- the gradient behind the activation ------------------------------------------------------------------
// d = dy * slope; its column sums (one partial per row slice), and for fp32 the largest |d inv_x| of each column beside them.
// A CTA has 64 x V columns and a slice of rows, four rows at a time.
struct GradArgs {
  int M, N;
  const void* dy; long long lddy;
  const void* slope; long long lds;
  void* d; long long ldd;               // 16-bit types: d, rows padded with zeros; NULL: not wanted
  const float* x_inv;                   // fp32: scales of x's rows
  float* sums; float* tops;             // [slices][ldp]
  long long ldp;
  int rows_per_slice;
};

template <typename T, bool VEC>
__device__ __forceinline__ void grad_values(const GradArgs& a, long long m, int n, float (&v)[Vec<T>::V]) {
  constexpr int V = Vec<T>::V;
  typedef typename SlopeOf<T>::type S;
  const T* dy = static_cast<const T*>(a.dy) + m * a.lddy + n;
  const S* sl = a.slope == nullptr ? nullptr : static_cast<const S*>(a.slope) + m * a.lds + n;
  if (VEC) {
    unpack16<T>(__ldg(reinterpret_cast<const uint4*>(dy)), v);
    if (sl != nullptr) {
      float s[V];
      unpack16<S>(__ldg(reinterpret_cast<const uint4*>(sl)), s);
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] *= s[e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      v[e] = n + e < a.N ? to_float(dy[e]) : 0.f;
      if (sl != nullptr && n + e < a.N) v[e] *= to_float(sl[e]);
    }
  }
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(256) grad_kernel(const GradArgs a) {
  constexpr int V = Vec<T>::V;
  __shared__ float red[3][64][V + 1];
  pdl_launch_dependents();
  pdl_wait();
  const int col = threadIdx.x & 63, grp = threadIdx.x >> 6;
  const int n = (blockIdx.x * 64 + col) * V;
  const int m1 = (int)min((long long)a.M, (long long)(blockIdx.y + 1) * a.rows_per_slice);
  float sum[V], top[V];
#pragma unroll
  for (int e = 0; e < V; ++e) sum[e] = top[e] = 0.f;
  if (n < a.N) {
#pragma unroll 8
    for (int m = blockIdx.y * a.rows_per_slice + grp; m < m1; m += 4) {
      float v[V];
      grad_values<T, VEC>(a, m, n, v);
      const float back = a.x_inv != nullptr ? __ldg(a.x_inv + m) : 0.f;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        sum[e] += v[e];
        top[e] = fmaxf(top[e], fabsf(v[e] * back));
      }
      if (a.d != nullptr) *reinterpret_cast<uint4*>(static_cast<T*>(a.d) + (long long)m * a.ldd + n) = pack16<T>(v);
    }
  }
  for (int pass = 0; pass < (a.tops != nullptr ? 2 : 1); ++pass) {
    float* out = pass == 0 ? a.sums : a.tops;
    if (out == nullptr) continue;
    __syncthreads();
    if (grp > 0) {
#pragma unroll
      for (int e = 0; e < V; ++e) red[grp - 1][col][e] = pass == 0 ? sum[e] : top[e];
    }
    __syncthreads();
    if (grp == 0 && n < a.N) {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        if (n + e >= a.N) continue;
        const float r0 = red[0][col][e], r1 = red[1][col][e], r2 = red[2][col][e];
        out[(long long)blockIdx.y * a.ldp + n + e] = pass == 0 ? ((sum[e] + r0) + r1) + r2 : fmaxf(fmaxf(top[e], r0), fmaxf(r1, r2));
      }
    }
  }
}

// Joins the slices in order: db, and the scales of d's columns.  32 columns x 32 groups of slices a CTA.
template <typename T>
__global__ void __launch_bounds__(1024) grad_columns_kernel(const float* __restrict__ sums, const float* __restrict__ tops, int slices,
                                                            long long ldp, int N, T* __restrict__ db, float* __restrict__ scale,
                                                            float* __restrict__ back) {
  __shared__ float rs[32][33], rt[32][33];
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, grp = threadIdx.x >> 5;
  const int n = blockIdx.x * 32 + lane;
  float s = 0.f, t = 0.f;
  if (n < N) {
#pragma unroll 4
    for (int k = grp; k < slices; k += 32) {
      if (sums != nullptr) s += sums[(long long)k * ldp + n];
      if (tops != nullptr) t = fmaxf(t, tops[(long long)k * ldp + n]);
    }
  }
  rs[grp][lane] = s;
  rt[grp][lane] = t;
  __syncthreads();
  s = rs[lane][grp];                                       // warp `grp` adds column `grp`
  t = rt[lane][grp];
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, off);
    t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, off));
  }
  const int c = blockIdx.x * 32 + grp;
  if (lane == 0 && c < N) {
    if (db != nullptr) db[c] = from_float<T>(s);
    if (tops != nullptr) pow2_row_scale(t, scale + c, back + c);
  }
}

// fp32: d as two planes for dx (rows scaled, W's row scales folded in) and two for dW (columns scaled, x's row scales
// folded in).  One warp per row.
struct GradPlanesArgs {
  GradArgs g;
  const float* w_inv;
  const float* col_scale;
  __half* dx; float* dx_inv;            // NULL: not wanted
  __half* dw;
  long long ld, plane;
};
// HELD: rows of at most 128 * HELD columns stay in registers between the row's maximum and its planes (0: read twice).
template <bool VEC, int HELD>
__global__ void __launch_bounds__(256) grad_planes_kernel(const GradPlanesArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  const int row = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (row >= a.g.M) return;
  auto value = [&](int c) {
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    if (c < a.g.N) grad_values<float, VEC>(a.g, row, c, v);
    return make_float4(v[0], v[1], v[2], v[3]);
  };
  float4 held[HELD > 0 ? HELD : 1];
  if (HELD > 0) {
#pragma unroll
    for (int i = 0; i < HELD; ++i) held[i] = value(lane * 4 + i * 128);
  }
  const float x_inv = a.dw != nullptr ? __ldg(a.g.x_inv + row) : 0.f;
  float scale = 1.f;
  if (a.dx != nullptr) {
    float mx = 0.f;
    auto take = [&](int c, float4 v) {
      if (c < a.g.N) mx = largest(times(v, __ldg(reinterpret_cast<const float4*>(a.w_inv + c))), mx);
    };
    if (HELD > 0) {
#pragma unroll
      for (int i = 0; i < HELD; ++i) take(lane * 4 + i * 128, held[i]);
    } else {
#pragma unroll 4
      for (int c = lane * 4; c < a.g.N; c += 128) take(c, value(c));
    }
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
    float back;
    pow2_row_scale(mx, &scale, &back);
    if (lane == 0) a.dx_inv[row] = back;
  }
  auto put = [&](int c, float4 v) {
    if (c >= a.ld) return;
    const long long at = (long long)row * a.ld + c;
    const bool inside = c < a.g.N;
    if (a.dx != nullptr) store_planes(a.dx + at, a.plane, times(times(v, inside ? __ldg(reinterpret_cast<const float4*>(a.w_inv + c)) : v), scale));
    if (a.dw != nullptr) store_planes(a.dw + at, a.plane, times(times(v, x_inv), inside ? __ldg(reinterpret_cast<const float4*>(a.col_scale + c)) : v));
  };
  if (HELD > 0) {
#pragma unroll
    for (int i = 0; i < HELD; ++i) put(lane * 4 + i * 128, held[i]);
  } else {
#pragma unroll 2
    for (int c = lane * 4; c < a.ld; c += 128) put(c, value(c));
  }
}
template <bool VEC>
void launch_grad_planes(const GradPlanesArgs& q, cudaStream_t st) {
  const dim3 grid((unsigned)cdiv(q.g.M, 8));
  if (q.ld <= 512) launch_pdl(grad_planes_kernel<VEC, 4>, grid, dim3(256), 0, st, q);
  else if (q.ld <= 1024) launch_pdl(grad_planes_kernel<VEC, 8>, grid, dim3(256), 0, st, q);
  else launch_pdl(grad_planes_kernel<VEC, 0>, grid, dim3(256), 0, st, q);
}

// ---- K slices ------------------------------------------------------------------------------------------
// C = epilogue(sum of the slices, in their order).  Four columns a thread.
struct FinishArgs {
  int M, N, splits;
  const float* partial; long long ldp, split_stride;
  int activation, vec;
  const void* bias;
  const void* residual; long long ldr;
  void* C; long long ldc;
  void* slope; long long lds;
};
template <typename T> struct Four { T e[4]; };
template <typename T> struct alignas(4 * sizeof(T)) Aligned { Four<T> f; };

template <typename T>
__global__ void __launch_bounds__(256) finish_kernel(const FinishArgs a) {
  typedef typename SlopeOf<T>::type S;
  pdl_launch_dependents();
  pdl_wait();
  const int quads = cdiv(a.N, 4);                          // not ldp / 4: rows of C may end four columns before the padded ones do
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= (long long)a.M * quads) return;
  const int m = (int)(i / quads), n = (int)(i % quads) * 4;
  const float* p = a.partial + (long long)m * a.ldp + n;
  float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int z = 0; z < a.splits; ++z) {
    const float4 f = __ldcs(reinterpret_cast<const float4*>(p + (long long)z * a.split_stride));
    v[0] += f.x; v[1] += f.y; v[2] += f.z; v[3] += f.w;
  }
  Four<T> y, r;
  Four<S> sl;
  const T* resp = static_cast<const T*>(a.residual) + (long long)m * a.ldr + n;
  if (a.vec && a.residual != nullptr) r = reinterpret_cast<const Aligned<T>*>(resp)->f;
  if (a.bias != nullptr) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (n + e < a.N) v[e] += to_float(static_cast<const T*>(a.bias)[n + e]);
  }
#pragma unroll
  for (int e = 0; e < 4; e += 2) {
    const Activated2 t = activate_as(a.activation, pair(v[e], v[e + 1]));
    const float2 f = split(t.y), g = split(t.slope);
    v[e] = f.x; v[e + 1] = f.y;
    sl.e[e] = from_float<S>(g.x); sl.e[e + 1] = from_float<S>(g.y);
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (a.residual != nullptr && n + e < a.N) v[e] += to_float(a.vec ? r.e[e] : resp[e]);
    y.e[e] = from_float<T>(v[e]);
  }
  T* cp = static_cast<T*>(a.C) + (long long)m * a.ldc + n;
  S* sp = static_cast<S*>(a.slope) + (long long)m * a.lds + n;
  if (a.vec) {
    reinterpret_cast<Aligned<T>*>(cp)->f = y;
    if (a.slope != nullptr) reinterpret_cast<Aligned<S>*>(sp)->f = sl;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (n + e < a.N) {
        cp[e] = y.e[e];
        if (a.slope != nullptr) sp[e] = sl.e[e];
      }
  }
}

// ---- a few rows ----------------------------------------------------------------------------------------
// Bound by one read of W (for each eight rows of x).  A warp has NW rows of W and a slice of K; lanes take 16 bytes each, partial sums of the lanes are
// added by a butterfly, those of the CTA's K slices in their order.  The assignment of k to lanes does not depend on alignment.
// Where it runs (us in a graph, it / the tensor-core products): bf16 1024 -> 4096 2 rows 4.5 / 7.3, 4 rows 6.9 / 7.3, 8 rows
// 10.1 / 7.3; 4096 -> 4096 2 rows 9.7 / 10.3, 4 rows 19.7 / 10.3.  fp32 (whose products need a pass for their planes) 4096 -> 4096
// 8 rows 45 / 65, 512 -> 512 8 rows 3.2 / 9.7.
bool few_rows_apply(int M, int N, int K, bool f32) {
  const double work = (double)M * N * K;
  if (f32) return M <= 8 || (M <= 32 && work <= 8.4e6);
  return M <= 2 || (M <= 8 && work <= 16.8e6);
}

template <typename T, bool VEC>
__device__ __forceinline__ void take(const T* p, int k, int K, float (&v)[Vec<T>::V]) {
  constexpr int V = Vec<T>::V;
  if (VEC) {
    if (k < K) unpack16<T>(__ldg(reinterpret_cast<const uint4*>(p + k)), v);
    else {
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] = 0.f;
    }
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = k + e < K ? to_float(p[k + e]) : 0.f;
  }
}

template <typename T, int MR, int NW, bool VEC>
__global__ void __launch_bounds__(256) few_rows_kernel(const b200gru_linear_args p, int slices) {
  constexpr int V = Vec<T>::V;
  typedef typename SlopeOf<T>::type S;
  __shared__ float part[8][MR * NW];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int groups = 8 / slices, slice = warp % slices;
  const int n0 = (blockIdx.x * groups + warp / slices) * NW;
  const int m0 = blockIdx.y * MR;
  const T* x = static_cast<const T*>(p.x);
  const T* W = static_cast<const T*>(p.W);
  float acc[MR][NW];
#pragma unroll
  for (int i = 0; i < MR; ++i)
#pragma unroll
    for (int j = 0; j < NW; ++j) acc[i][j] = 0.f;
  if (n0 < p.N) {
#pragma unroll 2
    for (int k = (slice * 32 + lane) * V; k < p.K; k += slices * 32 * V) {
      float w[NW][V];
#pragma unroll
      for (int j = 0; j < NW; ++j) take<T, VEC>(W + (long long)min(n0 + j, p.N - 1) * p.ldw, k, p.K, w[j]);
#pragma unroll
      for (int i = 0; i < MR; ++i) {
        float v[V];
        take<T, VEC>(x + (long long)min(m0 + i, p.M - 1) * p.ldx, k, p.K, v);
#pragma unroll
        for (int j = 0; j < NW; ++j)
#pragma unroll
          for (int e = 0; e < V; ++e) acc[i][j] = fmaf(v[e], w[j][e], acc[i][j]);
      }
    }
  }
  float mine = 0.f;                                       // result `lane` of the warp's MR x NW
#pragma unroll
  for (int i = 0; i < MR; ++i)
#pragma unroll
    for (int j = 0; j < NW; ++j) {
      float s = acc[i][j];
#pragma unroll
      for (int off = 16; off >= 1; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
      if (lane == i * NW + j) mine = s;
    }
  if (lane < MR * NW) part[warp][lane] = mine;
  __syncthreads();
  const int m = m0 + lane / NW, n = n0 + lane % NW;
  if (slice != 0 || lane >= MR * NW || m >= p.M || n >= p.N) return;
  float v = 0.f;
  for (int k = 0; k < slices; ++k) v += part[warp + k][lane];
  if (p.bias != nullptr) v += to_float(static_cast<const T*>(p.bias)[n]);
  const Activated2 r = activate_as(p.activation, pair(v, 0.f));
  if (p.slope != nullptr) static_cast<S*>(p.slope)[(long long)m * p.lds + n] = from_float<S>(split(r.slope).x);
  v = split(r.y).x;
  if (p.residual != nullptr) v += to_float(static_cast<const T*>(p.residual)[(long long)m * p.ldr + n]);
  static_cast<T*>(p.y)[(long long)m * p.ldy + n] = from_float<T>(v);
}

template <typename T, int MR, int NW>
int launch_few(const b200gru_linear_args& p, cudaStream_t st) {
  const long long warps = cdiv(p.N, NW);
  int slices = 1;                                         // K slices until every SM has a CTA, while a lane has work
  while (slices < 8 && warps * slices < 8 * 148 && (long long)p.K > (long long)slices * 32 * Vec<T>::V) slices *= 2;
  const dim3 grid((unsigned)((warps * slices + 7) / 8), (unsigned)cdiv(p.M, MR));
  const bool vec = p.K % Vec<T>::V == 0 && on16(p.x, p.M > 1 ? p.ldx : 0, sizeof(T)) && on16(p.W, p.N > 1 ? p.ldw : 0, sizeof(T));
  if (vec) few_rows_kernel<T, MR, NW, true><<<grid, 256, 0, st>>>(p, slices);
  else few_rows_kernel<T, MR, NW, false><<<grid, 256, 0, st>>>(p, slices);
  note_launch();
  return check_launch("few_rows_kernel");
}
template <typename T>
int few_rows(const b200gru_linear_args& p, cudaStream_t st) {
  if (p.M == 1) return launch_few<T, 1, 2>(p, st);
  if (p.M == 2) return launch_few<T, 2, 2>(p, st);
  if (p.M <= 4) return launch_few<T, 4, 2>(p, st);
  return launch_few<T, 8, 2>(p, st);
}

// ---- who runs when ---------------------------------------------------------------------------------------
// Hands out the workspace; without a base it only counts.
struct Carver {
  char* base;
  size_t at;
  template <typename T>
  T* take(long long n) {
    T* p = base == nullptr ? nullptr : reinterpret_cast<T*>(base + at);
    at += align_up((size_t)n * sizeof(T), 256);
    return p;
  }
};

// A matrix as the product kernel reads it.
struct Operand {
  const void* p;
  long long ld, plane;
  float* inv;                  // fp32: what undoes the scale of a row
};

template <typename T>
struct Call {
  const b200gru_linear_args& a;
  Carver ws;
  bool dry;                    // count the workspace only
  cudaStream_t st;
  int rc;

  static constexpr bool F32 = std::is_same<T, float>::value;

  void note(const char* what) {
    note_launch();
    if (rc == B200GRU_OK) rc = check_launch(what);
  }

  // 16-bit rows where they lie, if TMA can read them there.
  Operand operand(const void* src, long long ld, int rows, int cols) {
    Operand o = {src, ld, 0, nullptr};
    if (rows == 1 && (reinterpret_cast<uintptr_t>(src) & 15u) == 0) { o.ld = pad8(cols); return o; }
    if (ld >= cols && on16(src, ld, 2)) return o;
    o.ld = pad8(cols);
    T* d = ws.template take<T>((long long)rows * o.ld);
    o.p = d;
    copy_rows(static_cast<const T*>(src), ld, d, o.ld, rows, cols);
    return o;
  }
  // fp32 rows as planes; the launch follows in split().
  Operand planes(const void* src, long long ld, int rows, int cols, SplitArgs* s) {
    Operand o = {nullptr, pad8(cols), (long long)rows * pad8(cols), nullptr};
    __half* d = ws.template take<__half>(2 * o.plane);
    o.inv = ws.template take<float>(pad8(rows));
    o.p = d;
    *s = {static_cast<const float*>(src), ld, d, o.ld, o.plane, rows, cols, cols % 4 == 0 && on16(src, ld, 4) ? 1 : 0, o.inv};
    return o;
  }
  void split(const SplitArgs& one, const SplitArgs& two) {
    const long long rows = (long long)one.rows + two.rows;
    if (dry || rc != B200GRU_OK || rows == 0) return;
    launch_pdl(split_rows_kernel, dim3((unsigned)((rows + 7) / 8)), dim3(256), 0, st, one, two);
    note("split_rows_kernel");
  }
  // x and W as the products read them (either may not be wanted).
  void operands(bool want_x, bool want_w, Operand* x, Operand* W) {
    if (F32) {
      SplitArgs one, two;
      memset(&one, 0, sizeof(one));
      memset(&two, 0, sizeof(two));
      if (want_x) *x = planes(a.x, a.ldx, a.M, a.K, &one);
      if (want_w) *W = planes(a.W, a.ldw, a.N, a.K, &two);
      split(one, two);
    } else {
      if (want_x) *x = operand(a.x, a.ldx, a.M, a.K);
      if (want_w) *W = operand(a.W, a.ldw, a.N, a.K);
    }
  }

  template <typename U>
  void copy_rows(const U* src, long long ld, U* dst, long long dld, int rows, int cols) {
    if (dry || rc != B200GRU_OK) return;
    launch_pdl(copy_rows_kernel<U>, dim3((unsigned)cdiv(rows, 8)), dim3(256), 0, st, src, ld, dst, dld, rows, cols);
    note("copy_rows_kernel");
  }

  // The product of two operands, in K slices where that fills the GPU better.
  void product(Gemm g) {
    g.planes = F32 ? 2 : 1;
    g.fp16 = F32 || std::is_same<T, __half>::value;
    const Plan plan = plan_gemm(g.M, g.N, g.K, g.planes);
    g.splits = plan.splits;
    if (plan.splits == 1) {
      const long long ld = pad8(g.N);
      if (g.residual != nullptr && (g.ldr < g.N || !on16(g.residual, g.ldr, sizeof(T)))) {
        T* r = ws.template take<T>(g.M * ld);
        copy_rows(static_cast<const T*>(g.residual), g.ldr, r, ld, g.M, g.N);
        g.residual = r; g.ldr = ld;
      }
      T* out = static_cast<T*>(g.C);
      const long long ldc = g.ldc;
      // a tile store writes whole 16-byte pieces: behind rows that end inside one, too
      const bool apart = !on16(g.C, g.ldc, sizeof(T)) || g.N * sizeof(T) % 16 != 0;
      if (apart) { g.C = ws.template take<T>(g.M * ld); g.ldc = ld; }
      typedef typename SlopeOf<T>::type S;
      S* slope = static_cast<S*>(g.slope);
      const long long lds = g.lds;
      const bool slope_apart = !on16(g.slope, g.lds, sizeof(S)) && g.activation != B200GRU_ACT_NONE;
      if (slope_apart) { g.slope = ws.template take<S>(g.M * ld); g.lds = ld; }
      if (!dry && rc == B200GRU_OK) rc = launch_gemm<T>(g, plan, st);
      if (apart) copy_rows(static_cast<const T*>(g.C), ld, out, ldc, g.M, g.N);
      if (slope_apart) copy_rows(static_cast<const S*>(g.slope), ld, slope, lds, g.M, g.N);
      return;
    }
    FinishArgs f;
    memset(&f, 0, sizeof(f));
    f.M = g.M; f.N = g.N; f.splits = plan.splits;
    g.ldp = f.ldp = pad8(g.N);
    f.split_stride = (long long)g.M * g.ldp;
    g.partial = ws.template take<float>(f.split_stride * plan.splits);
    f.partial = g.partial;
    f.activation = g.activation; f.bias = g.bias; f.residual = g.residual; f.ldr = g.ldr;
    f.C = g.C; f.ldc = g.ldc; f.slope = g.slope; f.lds = g.lds;
    f.vec = g.N % 4 == 0 && g.ldc % 4 == 0 && on16(g.C, 0, 1) && on16(g.slope, 0, 1) && g.lds % 4 == 0 && (g.residual == nullptr || (g.ldr % 4 == 0 && on16(g.residual, 0, 1)));
    if (dry || rc != B200GRU_OK) return;
    rc = launch_gemm<void>(g, plan, st);
    if (rc != B200GRU_OK) return;
    const long long quads = (long long)g.M * cdiv(g.N, 4);
    launch_pdl(finish_kernel<T>, dim3((unsigned)((quads + 255) / 256)), dim3(256), 0, st, f);
    note("finish_kernel");
  }

  int forward() {
    if (few_rows_apply(a.M, a.N, a.K, F32)) {
      if (!dry) rc = few_rows<T>(a, st);
      return rc;
    }
    Operand x = {}, W = {};
    operands(true, true, &x, &W);
    Gemm g;
    memset(&g, 0, sizeof(g));
    g.M = a.M; g.N = a.N; g.K = a.K;
    g.A = x.p; g.lda = x.ld; g.a_plane = x.plane; g.row_scale = x.inv;
    g.B = W.p; g.ldb = W.ld; g.b_plane = W.plane; g.col_scale = W.inv;
    g.activation = a.activation; g.bias = a.bias; g.residual = a.residual; g.ldr = a.ldr;
    g.C = a.y; g.ldc = a.ldy; g.slope = a.slope; g.lds = a.lds;
    product(g);
    return rc;
  }

  int backward() {
    const bool act = a.activation != B200GRU_ACT_NONE;
    Operand x = {}, W = {}, dx = {}, dw = {};
    operands(a.dW != nullptr, a.dx != nullptr, &x, &W);

    GradArgs g;
    memset(&g, 0, sizeof(g));
    g.M = a.M; g.N = a.N; g.dy = a.dy; g.lddy = a.lddy; g.slope = act ? a.slope : nullptr; g.lds = a.lds;
    g.ldd = pad8(a.N); g.ldp = pad8(a.N);
    const bool vec = a.N % Vec<T>::V == 0 && on16(a.dy, a.lddy, sizeof(T)) && (!act || on16(a.slope, a.lds, sizeof(typename SlopeOf<T>::type)));
    const bool products = a.dx != nullptr || a.dW != nullptr;
    if (!F32 && products) {
      if (act) {
        T* d = ws.template take<T>((long long)a.M * g.ldd);
        g.d = d;
        dx.p = d; dx.ld = g.ldd;
      } else {
        dx = operand(a.dy, a.lddy, a.M, a.N);
      }
      dw = dx;
    }
    float* scale = nullptr;
    float* back = nullptr;
    const bool columns = F32 && a.dW != nullptr;
    if (a.db != nullptr || columns || g.d != nullptr) {
      const int across = cdiv(a.N, 64 * Vec<T>::V);
      int slices = cdiv(4 * 148, across);                  // four CTAs to an SM (two or eight took longer), 16 rows or more each
      if (slices > cdiv(a.M, 16)) slices = cdiv(a.M, 16);
      g.rows_per_slice = cdiv(cdiv(a.M, slices), 4) * 4;
      slices = cdiv(a.M, g.rows_per_slice);
      if (a.db != nullptr) g.sums = ws.template take<float>(slices * g.ldp);
      if (columns) {
        g.tops = ws.template take<float>(slices * g.ldp);
        scale = ws.template take<float>(g.ldp);
        back = ws.template take<float>(g.ldp);
        g.x_inv = x.inv;
      }
      if (!dry && rc == B200GRU_OK) {
        const dim3 grid((unsigned)across, (unsigned)slices);
        if (vec) launch_pdl(grad_kernel<T, true>, grid, dim3(256), 0, st, g);
        else launch_pdl(grad_kernel<T, false>, grid, dim3(256), 0, st, g);
        note("grad_kernel");
        if (a.db != nullptr || columns) {
          launch_pdl(grad_columns_kernel<T>, dim3((unsigned)cdiv(a.N, 32)), dim3(1024), 0, st, static_cast<const float*>(g.sums),
                     static_cast<const float*>(g.tops), slices, g.ldp, a.N, static_cast<T*>(a.db), scale, back);
          note("grad_columns_kernel");
        }
      }
    }
    if (F32 && products) {
      GradPlanesArgs q;
      memset(&q, 0, sizeof(q));
      q.g = g; q.g.x_inv = x.inv;
      q.w_inv = W.inv; q.col_scale = scale;
      q.ld = pad8(a.N); q.plane = (long long)a.M * q.ld;
      if (a.dx != nullptr) {
        q.dx = ws.template take<__half>(2 * q.plane);
        q.dx_inv = ws.template take<float>(pad8(a.M));
        dx.p = q.dx; dx.ld = q.ld; dx.plane = q.plane; dx.inv = q.dx_inv;
      }
      if (a.dW != nullptr) {
        q.dw = ws.template take<__half>(2 * q.plane);
        dw.p = q.dw; dw.ld = q.ld; dw.plane = q.plane; dw.inv = back;
      }
      if (!dry && rc == B200GRU_OK) {
        if (vec) launch_grad_planes<true>(q, st);
        else launch_grad_planes<false>(q, st);
        note("grad_planes_kernel");
      }
    }
    Gemm m;
    memset(&m, 0, sizeof(m));
    if (a.dx != nullptr) {
      m.M = a.M; m.N = a.K; m.K = a.N;
      m.A = dx.p; m.lda = dx.ld; m.a_plane = dx.plane; m.row_scale = dx.inv;
      m.B = W.p; m.ldb = W.ld; m.b_plane = W.plane; m.b_mn = true;
      m.C = a.dx; m.ldc = a.K;
      product(m);
    }
    if (a.dW != nullptr) {
      memset(&m, 0, sizeof(m));
      m.M = a.N; m.N = a.K; m.K = a.M;
      m.A = dw.p; m.lda = dw.ld; m.a_plane = dw.plane; m.a_mn = true; m.row_scale = dw.inv;
      m.B = x.p; m.ldb = x.ld; m.b_plane = x.plane; m.b_mn = true;
      m.C = a.dW; m.ldc = a.K;
      product(m);
    }
    return rc;
  }
};

template <typename T>
int run(const b200gru_linear_args& a, bool backward, bool dry, size_t* bytes, cudaStream_t st) {
  Call<T> c = {a, {dry ? nullptr : static_cast<char*>(a.workspace), 0}, dry, st, B200GRU_OK};
  const int rc = backward ? c.backward() : c.forward();
  if (bytes != nullptr) *bytes = c.ws.at;
  return rc;
}

int run_as(const b200gru_linear_args& a, bool backward, bool dry, size_t* bytes, cudaStream_t st) {
  if (a.dtype == B200GRU_F32) return run<float>(a, backward, dry, bytes, st);
  if (a.dtype == B200GRU_BF16) return run<__nv_bfloat16>(a, backward, dry, bytes, st);
  return run<__half>(a, backward, dry, bytes, st);
}

// M: a tile of 256 rows that begins inside the matrix ends below 2^31.
bool bad(const b200gru_linear_args* p) {
  return p == nullptr || p->M <= 0 || p->N <= 0 || p->K <= 0 || p->M > 0x7ffffe00 || p->N > 0x3ffffff0 || p->K > 0x3ffffff0 ||
         p->dtype < B200GRU_F32 || p->dtype > B200GRU_F16 || p->activation < B200GRU_ACT_NONE ||
         p->activation > B200GRU_ACT_TANH || p->x == nullptr || p->W == nullptr || p->ldx < 0 || p->ldw < 0 ||
         (p->slope != nullptr && p->lds < p->N);
}

int checked(const b200gru_linear_args* p, bool backward, void* stream) {
  size_t need = 0;
  run_as(*p, backward, true, &need, nullptr);
  if (need > p->workspace_bytes) return B200GRU_WORKSPACE_TOO_SMALL;
  if (need > 0 && (p->workspace == nullptr || (reinterpret_cast<uintptr_t>(p->workspace) & 255u))) return B200GRU_INVALID_ARGUMENT;
  return run_as(*p, backward, false, nullptr, static_cast<cudaStream_t>(stream));
}

}  // namespace

// Cycles of a tile's k-block and tail, of a launch's start and end, of one that joins slices; the cheapest cut of the work.
// Fitted to 16 .. 16384 rows, 120 .. 8192 columns in both types: within 16 % of the best of 30 cuts.
Plan plan_gemm(int M, int N, int K, int planes) {
  const int kb = cdiv(K, 64);
  const double products = planes == 2 ? 3.0 : 1.0;
  Plan best = {1, 128, 1};
  double best_cost = 1e30;
  const struct { int ctas, m, n, units; double per_kb, tail; } cuts[3] = {
      {2, 256, 256, 74, 560.0, 4500.0}, {1, 128, 128, 148, 370.0, 2500.0}, {1, 128, 64, 148, 270.0, 1500.0}};
  for (const auto& c : cuts) {
    const long long tiles = (long long)cdiv(M, c.m) * cdiv(N, c.n);
    for (int want = 1; want <= 64 && want <= kb; ++want) {
      const int per = cdiv(kb, want), splits = cdiv(kb, per);
      if (splits != want || (splits > 1 && per < 4)) continue;
      const double waves = (double)((tiles * splits + c.units - 1) / c.units);
      const double loop = per * c.per_kb * products;       // a tile's tail hides under the next one's products, if those last
      double cost = waves * (loop > c.tail ? loop : c.tail) + 4000.0 + 2500.0 * (c.n / 128.0);
      if (splits > 1) cost += 5000.0 + (double)splits * M * N * 8.0 / 3500.0;      // written and read again
      if (cost < best_cost) { best_cost = cost; best = {c.ctas, c.n, splits}; }
    }
  }
  return best;
}

int read_status(int reset) {
  const int s[4] = {gemm_status<float>(reset), gemm_status<__nv_bfloat16>(reset), gemm_status<__half>(reset), gemm_status<void>(reset)};
  int v = 0;
  for (int i = 0; i < 4; ++i) {
    if (s[i] < 0) return -1;
    v |= s[i];
  }
  return v;
}

}  // namespace lin
}  // namespace b200gru

using namespace b200gru;

extern "C" {

int b200gru_test_linear_plan(int M, int N, int K, int planes, int activation, int* plan) {
  if (M <= 0 || N <= 0 || K <= 0 || (planes != 1 && planes != 2) || plan == nullptr) return B200GRU_INVALID_ARGUMENT;
  const lin::Plan p = lin::plan_gemm(M, N, K, planes);
  const int per = cdiv(cdiv(K, 64), p.splits);
  plan[0] = p.ctas; plan[1] = p.bn; plan[2] = p.splits; plan[3] = per;
  plan[4] = lin::chunk_kblocks(planes, p.splits == 1 && activation != B200GRU_ACT_NONE, per);
  return B200GRU_OK;
}

size_t b200gru_linear_act_workspace_bytes(const b200gru_linear_args* p, int backward) try {
  if (lin::bad(p)) return (size_t)-1;
  size_t n = 0;
  lin::run_as(*p, backward != 0, true, &n, nullptr);
  return n;
} catch (...) {
  return (size_t)-1;
}

int b200gru_linear_act_forward(const b200gru_linear_args* p, void* stream) try {
  if (lin::bad(p) || p->y == nullptr || p->ldy < p->N || (p->residual != nullptr && p->ldr < 0)) return B200GRU_INVALID_ARGUMENT;
  return lin::checked(p, false, stream);
} catch (...) {
  return B200GRU_LAUNCH_FAILURE;
}

int b200gru_linear_act_backward(const b200gru_linear_args* p, void* stream) try {
  if (lin::bad(p) || p->dy == nullptr || p->lddy < 0) return B200GRU_INVALID_ARGUMENT;
  if (p->activation != B200GRU_ACT_NONE && p->slope == nullptr) return B200GRU_INVALID_ARGUMENT;
  return lin::checked(p, true, stream);
} catch (...) {
  return B200GRU_LAUNCH_FAILURE;
}

}  // extern "C"
