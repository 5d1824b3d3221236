// Tensor-core product of linear_act: persistent CTAs (128 x BN tiles) or CTA pairs (256 x 256), epilogue of a tile under the
// products of the next.
//
//   C[M,N] = epilogue( row_scale[m] col_scale[n] sum_p A_p[M,K] B_p[N,K]^T )
//
// Operands: one plane of bf16 or fp16, or (fp32) two row-scaled fp16 planes, of which low x high, high x low and high x high
// are summed in that order.  Either operand K-major (rows of K) or MN-major (rows of M or N, one per k).  The tensor core's
// fp32 accumulator truncates, so sums are built in chunks (32 steps for planes; 256 for 16-bit types, whose results are rounded
// to 2^-9 or 2^-12) in one of two tensor-memory buffers and added to register totals with round-to-nearest.
//
// Roles of a CTA's ten warps: 0 loads k-blocks by TMA, 1 issues tcgen05.mma, 2-9 drain the accumulator (32 rows and half the
// columns each), turn it through a transpose buffer so that rows leave in whole sectors, and apply the epilogue there.  The
// residual of the next columns is requested before the present ones are finished.
#pragma once

#include <cstring>
#include <map>
#include <mutex>
#include <type_traits>
#include <utility>

#include "linear_act.cuh"
#include "tc_common.cuh"

namespace b200gru {
namespace lin {

struct Gemm {
  int M, N, K;
  int planes;                    // 1: bf16 or fp16, 2: fp16 planes
  bool fp16;                     // operand format
  const void* A;
  const void* B;
  bool a_mn, b_mn;               // rows of M or N instead of rows of K
  long long lda, ldb, a_plane, b_plane;        // elements
  const float* row_scale;
  const float* col_scale;
  int splits;                    // K slices; > 1: partial sums to `partial`, no epilogue
  float* partial;                // [splits][M][ldp]
  long long ldp;
  // epilogue
  int activation;
  const void* bias;
  const void* residual; long long ldr;
  void* C; long long ldc;
  void* slope; long long lds;
};

// How a product is cut: CTAs per tile (1: 128 x bn, 2: 256 x 256) and K slices.
struct Plan {
  int ctas, bn, splits;
};
Plan plan_gemm(int M, int N, int K, int planes);
// T: element type of C (float, __nv_bfloat16, __half).
template <typename T>
int launch_gemm(const Gemm& g, const Plan& plan, cudaStream_t st);
template <typename T>
int gemm_status(int reset);

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

// Rows that start on 16-byte boundaries.
inline bool on16(const void* p, long long ld, size_t es) {
  return p == nullptr || ((reinterpret_cast<uintptr_t>(p) & 15u) == 0 && (ld * (long long)es) % 16 == 0);
}

// 16 bytes of a row: V values.
template <typename T> struct Vec;
template <> struct Vec<float> { static constexpr int V = 4; };
template <> struct Vec<__nv_bfloat16> { static constexpr int V = 8; };
template <> struct Vec<__half> { static constexpr int V = 8; };

template <typename T>
__device__ __forceinline__ void unpack16(const uint4& w, float (&v)[Vec<T>::V]) {
  const T* e = reinterpret_cast<const T*>(&w);
#pragma unroll
  for (int i = 0; i < Vec<T>::V; ++i) v[i] = to_float(e[i]);
}
template <typename T>
__device__ __forceinline__ uint4 pack16(const float (&v)[Vec<T>::V]) {
  uint4 w;
  T* e = reinterpret_cast<T*>(&w);
#pragma unroll
  for (int i = 0; i < Vec<T>::V; ++i) e[i] = from_float<T>(v[i]);
  return w;
}

#ifdef B200GRU_LINEAR_GEMM_IMPL

static __device__ int g_lin_status;          // a bounded wait gave up (one word per translation unit)

namespace {

constexpr int BM = 128;                      // rows of A per CTA
constexpr int EPI_WARPS = 8;
constexpr int THREADS = 64 + 32 * EPI_WARPS;
constexpr int MAX_STAGES = 8;

struct Params {
  int M, N;
  int tiles_m, tiles_n, tiles;               // tiles of the K slices included
  int kb_total, kb_per_split;
  int stages, chunk_kb;
  int vec;                                   // rows of every epilogue tensor on 16-byte boundaries, N a multiple of V
  unsigned ab_format;
  const float* row_scale;
  const float* col_scale;
  int activation;
  const void* bias;
  const void* residual; long long ldr;
  void* C; long long ldc;
  void* slope; long long lds;
  float* partial; long long ldp, split_stride;
};

__device__ __forceinline__ uint32_t cta_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void pair_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t at_leader(uint32_t addr) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(addr));
  return r;
}
template <int CTAS>
__device__ __forceinline__ void load_tile(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, uint32_t bar) {
  if (CTAS == 1) {
    tc::tma_load_3d(dst, map, c0, c1, c2, bar);
  } else {                                   // bytes counted on the barrier of the pair's leader
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3, %4}], [%5];"
        ::"r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(bar) : "memory");
  }
}
template <int CTAS>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  if (CTAS == 1) {
    tc::umma<false>(d, a, b, idesc, accumulate);
  } else {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
  }
}
template <int CTAS>
__device__ __forceinline__ void commit(uint32_t bar) {
  if (CTAS == 1) {
    tc::umma_commit(bar);
  } else {
    const uint16_t mask = 3;
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 ::"r"(bar), "h"(mask) : "memory");
  }
}

// Columns that a warp turns at a time: 64 bytes of a row for every type.
template <typename Out> struct Turn { typedef Out T; };
template <> struct Turn<void> { typedef float T; };
template <typename T> constexpr int STEP = 4 * Vec<T>::V;
template <typename T> constexpr int TR_LD = STEP<T> + 4;      // floats per row of the transpose buffer
template <typename T> constexpr int TR_BYTES = EPI_WARPS * 32 * TR_LD<T> * 4;

// Out = void: partial sums in fp32.
template <int CTAS, int BN, bool A_MN, bool B_MN, int PL, typename Out>
__global__ void __launch_bounds__(THREADS, 1)
lin_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const Params p) {
  typedef typename Turn<Out>::T T;
  constexpr bool PARTIAL = std::is_void<Out>::value;
  constexpr int V = Vec<T>::V;
  constexpr int BH = CTAS == 2 ? 128 : BN;               // rows of B per CTA
  constexpr int A_PLANE = BM * 128, B_PLANE = BH * 128, STAGE = PL * (A_PLANE + B_PLANE);
  constexpr int UMMA_K = 16, NC = BN / 2;                // accumulator columns per epilogue thread
  const uint32_t IDESC = tc::umma_idesc(false, A_MN, B_MN, CTAS * BM, BN, p.ab_format);

  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  __shared__ __align__(8) unsigned long long bar_full[MAX_STAGES], bar_empty[MAX_STAGES];
  __shared__ __align__(8) unsigned long long bar_acc_full[2], bar_acc_empty[2];
  __shared__ uint32_t tmem_slot;
  __shared__ int dead;

  const int warp = tc::uniform_warp(), lane = threadIdx.x & 31;
  const uint32_t rank = CTAS == 2 ? cta_rank() : 0;
  const int unit = blockIdx.x / CTAS, units = gridDim.x / CTAS;
  volatile int* deadp = &dead;
  int* status = &g_lin_status;
  pdl_launch_dependents();

  if (threadIdx.x == 0) {
    dead = (*reinterpret_cast<volatile int*>(status) != 0) ? 1 : 0;
    for (int s = 0; s < p.stages; ++s) {
      tc::mbar_init(tc::smem_u32(&bar_full[s]), 1);
      tc::mbar_init(tc::smem_u32(&bar_empty[s]), 1);
    }
    for (int b = 0; b < 2; ++b) {
      tc::mbar_init(tc::smem_u32(&bar_acc_full[b]), 1);
      tc::mbar_init(tc::smem_u32(&bar_acc_empty[b]), CTAS * EPI_WARPS);
    }
    tc::mbar_fence_init();
    tc::tma_prefetch_map(&tmA);
    tc::tma_prefetch_map(&tmB);
  }
  if (warp == 1) {
    if (CTAS == 1) {
      tc::tmem_alloc(tc::smem_u32(&tmem_slot), 2 * BN);
    } else {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc::smem_u32(&tmem_slot)), "r"(2 * BN) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
  }
  tc::tc_fence_before();
  __syncthreads();
  if (CTAS == 2) pair_sync();                             // barriers of both CTAs exist
  tc::tc_fence_after();
  const uint32_t tmem = tmem_slot;
  pdl_wait();

  // tile index -> K slice, row panel, column panel (columns fastest: neighbours share the rows of A)
  auto locate = [&](int t, int& m0, int& n0, int& z, int& kb0, int& nkb) {
    n0 = (t % p.tiles_n) * BN;
    const int r = t / p.tiles_n;
    m0 = (r % p.tiles_m) * CTAS * BM + (int)rank * BM;
    z = r / p.tiles_m;
    kb0 = z * p.kb_per_split;
    nkb = max(0, min(p.kb_total, kb0 + p.kb_per_split) - kb0);
  };

  if (warp == 0) {
    // ---- loader: own rows of A and of B; for a pair the leader's barrier counts the bytes of both CTAs
    bool alive = __all_sync(0xffffffffu, *deadp == 0);
    int s = 0;
    uint32_t parity = 1;                                  // the first round finds every stage free
    bool first = true;
    for (int t = unit; t < p.tiles && alive; t += units) {
      int m0, n0, z, kb0, nkb;
      locate(t, m0, n0, z, kb0, nkb);
      n0 += (int)rank * BH;
      for (int i = 0; i < nkb; ++i) {
        if (!first) alive = __all_sync(0xffffffffu, tc::mbar_wait(tc::smem_u32(&bar_empty[s]), parity, deadp, status));
        if (!alive) break;
        if (tc::elect_one()) {
          const uint32_t own = tc::smem_u32(&bar_full[s]);
          const uint32_t full = CTAS == 2 ? at_leader(own) : own;
          if (rank == 0) tc::mbar_expect_tx(own, (uint32_t)(CTAS * STAGE));
          const uint32_t st = tc::smem_u32(smem) + (uint32_t)(s * STAGE);
          const int k = (kb0 + i) * 64;
#pragma unroll
          for (int pl = 0; pl < PL; ++pl) {
            const uint32_t da = st + (uint32_t)(pl * A_PLANE), db = st + (uint32_t)(PL * A_PLANE + pl * B_PLANE);
            if (A_MN) {
              load_tile<CTAS>(da, &tmA, m0, k, pl, full);
              load_tile<CTAS>(da + 8192, &tmA, m0 + 64, k, pl, full);
            } else {
              load_tile<CTAS>(da, &tmA, k, m0, pl, full);
            }
            if (B_MN) {
#pragma unroll
              for (int c = 0; c < BH / 64; ++c) load_tile<CTAS>(db + c * 8192, &tmB, n0 + c * 64, k, pl, full);
            } else {
              load_tile<CTAS>(db, &tmB, k, n0, pl, full);
            }
          }
        }
        __syncwarp();
        if (++s == p.stages) { s = 0; parity ^= 1u; first = false; }
      }
    }
  } else if (warp == 1) {
    if (rank == 0) {
      // ---- issuer
      constexpr uint64_t A_STEP = (A_MN ? UMMA_K * 128 : 32) >> 4, B_STEP = (B_MN ? UMMA_K * 128 : 32) >> 4;
      const uint64_t da0 = tc::umma_smem_desc(tc::smem_u32(smem), A_MN ? 8192 : 16, 1024);
      const uint64_t db0 = tc::umma_smem_desc(tc::smem_u32(smem), B_MN ? 8192 : 16, 1024);
      bool alive = __all_sync(0xffffffffu, *deadp == 0);
      int s = 0, c = 0;                                   // ring stage, chunks so far
      uint32_t parity = 0;
      for (int t = unit; t < p.tiles && alive; t += units) {
        int m0, n0, z, kb0, nkb;
        locate(t, m0, n0, z, kb0, nkb);
        for (int i0 = 0; i0 < nkb && alive; i0 += p.chunk_kb, ++c) {
          const int buf = c & 1;
          if (c >= 2) alive = __all_sync(0xffffffffu, tc::mbar_wait(tc::smem_u32(&bar_acc_empty[buf]), ((c >> 1) - 1) & 1, deadp, status));
          if (!alive) break;
          tc::tc_fence_after();
          const uint32_t tacc = tmem + (uint32_t)(buf * BN);
          const int i1 = min(nkb, i0 + p.chunk_kb);
          for (int i = i0; i < i1; ++i) {
            alive = __all_sync(0xffffffffu, tc::mbar_wait(tc::smem_u32(&bar_full[s]), parity, deadp, status));
            if (!alive) break;
            tc::tc_fence_after();
            if (tc::elect_one()) {
              const uint64_t a = da0 + (uint32_t)((s * STAGE) >> 4), b = db0 + (uint32_t)((s * STAGE + PL * A_PLANE) >> 4);
              const uint32_t more = i > i0 ? 1u : 0u;
              if (PL == 1) {
#pragma unroll
                for (int kk = 0; kk < 4; ++kk) mma<CTAS>(tacc, a + kk * A_STEP, b + kk * B_STEP, IDESC, kk > 0 ? 1u : more);
              } else {                                    // low x high, high x low, high x high
#pragma unroll
                for (int kk = 0; kk < 4; ++kk)
                  mma<CTAS>(tacc, a + (A_PLANE >> 4) + kk * A_STEP, b + kk * B_STEP, IDESC, kk > 0 ? 1u : more);
#pragma unroll
                for (int kk = 0; kk < 4; ++kk) mma<CTAS>(tacc, a + kk * A_STEP, b + (B_PLANE >> 4) + kk * B_STEP, IDESC, 1u);
#pragma unroll
                for (int kk = 0; kk < 4; ++kk) mma<CTAS>(tacc, a + kk * A_STEP, b + kk * B_STEP, IDESC, 1u);
              }
              commit<CTAS>(tc::smem_u32(&bar_empty[s]));
              if (i == i1 - 1) commit<CTAS>(tc::smem_u32(&bar_acc_full[buf]));
            }
            __syncwarp();
            if (++s == p.stages) { s = 0; parity ^= 1u; }
          }
        }
      }
    }
  } else {
    // ---- epilogue: warp w reads lanes 32 (w % 4) .. of this CTA's accumulator, one half of the columns
    constexpr int ST = STEP<T>, LD = TR_LD<T>;
    const int q = warp & 3, half = (warp - 2) >> 2;
    float* tr = reinterpret_cast<float*>(smem + p.stages * STAGE) + (warp - 2) * 32 * LD;
    const int rsub = lane >> 2, csub = (lane & 3) * V;
    const T* resp = static_cast<const T*>(p.residual);
    typedef typename SlopeOf<T>::type S;
    int c = 0;
    bool ok = __all_sync(0xffffffffu, *deadp == 0);
    for (int t = unit; t < p.tiles && ok; t += units) {
      int m0, n0, z, kb0, nkb;
      locate(t, m0, n0, z, kb0, nkb);
      const int row_base = m0 + q * 32, col_base = n0 + half * NC;
      uint4 res[4];
      const bool prefetch = !PARTIAL && p.vec && resp != nullptr;
      auto request = [&](int j) {                         // the residual of columns col_base + j ..
        const int n = col_base + j + csub;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int m = row_base + k * 8 + rsub;
          res[k] = make_uint4(0, 0, 0, 0);
          if (m < p.M && n < p.N) res[k] = __ldg(reinterpret_cast<const uint4*>(resp + (long long)m * p.ldr + n));
        }
      };
      if (prefetch) request(0);
      float rs[4] = {1.f, 1.f, 1.f, 1.f};
      if (p.row_scale != nullptr) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int m = row_base + k * 8 + rsub;
          if (m < p.M) rs[k] = __ldg(p.row_scale + m);
        }
      }
      float acc[NC];
#pragma unroll
      for (int j = 0; j < NC; ++j) acc[j] = 0.f;
      for (int i0 = 0; i0 < nkb; i0 += p.chunk_kb, ++c) {
        const int buf = c & 1;
        ok = __all_sync(0xffffffffu, tc::mbar_wait(tc::smem_u32(&bar_acc_full[buf]), (c >> 1) & 1, deadp, status));
        if (!ok) break;
        tc::tc_fence_after();
        const uint32_t tsrc = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(buf * BN + half * NC);
#pragma unroll
        for (int c0 = 0; c0 < NC; c0 += 32) {
          uint32_t v[32];
          tc::tmem_ld32(tsrc + (uint32_t)c0, v);
          tc::tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 32; ++j) acc[c0 + j] += __uint_as_float(v[j]);
        }
        tc::tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          const uint32_t own = tc::smem_u32(&bar_acc_empty[buf]);
          if (CTAS == 2) asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(at_leader(own)) : "memory");
          else tc::mbar_arrive(own);
        }
      }
      if (!ok) break;
#pragma unroll
      for (int j = 0; j < NC; j += ST) {
        if (col_base + j >= p.N) break;                    // warp-uniform
        __syncwarp();
#pragma unroll
        for (int e = 0; e < ST; e += 4)
          *reinterpret_cast<float4*>(tr + lane * LD + e) = make_float4(acc[j + e], acc[j + e + 1], acc[j + e + 2], acc[j + e + 3]);
        __syncwarp();
        if (p.vec) {
          const int n = col_base + j + csub;
          uint4 now[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) now[k] = res[k];
          if (prefetch && j + ST < NC) request(j + ST);
          if (n < p.N) {                                   // N is a multiple of V
            float cs[V], bs[V];
#pragma unroll
            for (int e = 0; e < V; ++e) { cs[e] = 1.f; bs[e] = 0.f; }
            if (p.col_scale != nullptr) {
#pragma unroll
              for (int e = 0; e < V; ++e) cs[e] = __ldg(p.col_scale + n + e);
            }
            if (!PARTIAL && p.bias != nullptr) unpack16<T>(__ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(p.bias) + n)), bs);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int m = row_base + k * 8 + rsub;
              if (m < p.M) {
                float v[V];
#pragma unroll
                for (int e = 0; e < V; e += 4) {
                  const float4 f = *reinterpret_cast<const float4*>(tr + (k * 8 + rsub) * LD + csub + e);
                  v[e] = f.x; v[e + 1] = f.y; v[e + 2] = f.z; v[e + 3] = f.w;
                }
                if (PL == 2) {
#pragma unroll
                  for (int e = 0; e < V; ++e) v[e] = v[e] * rs[k] * cs[e];
                }
                if (PARTIAL) {
                  *reinterpret_cast<float4*>(p.partial + (long long)z * p.split_stride + (long long)m * p.ldp + n) = make_float4(v[0], v[1], v[2], v[3]);
                } else {
#pragma unroll
                  for (int e = 0; e < V; ++e) v[e] += bs[e];
                  if (p.activation != B200GRU_ACT_NONE) {
                    float sl[V];
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                      const Activated r = activate_as(p.activation, v[e]);
                      v[e] = r.y;
                      sl[e] = r.slope;
                    }
                    if (p.slope != nullptr)
                      *reinterpret_cast<uint4*>(static_cast<S*>(p.slope) + (long long)m * p.lds + n) = pack16<S>(sl);
                  }
                  if (resp != nullptr) {
                    float rv[V];
                    unpack16<T>(now[k], rv);
#pragma unroll
                    for (int e = 0; e < V; ++e) v[e] += rv[e];
                  }
                  *reinterpret_cast<uint4*>(static_cast<T*>(p.C) + (long long)m * p.ldc + n) = pack16<T>(v);
                }
              }
            }
          }
        } else {
          // rows that lie on no boundary: a column per lane
          const int cl = lane % ST, n = col_base + j + cl;
          if (n < p.N) {
            const float cs = p.col_scale != nullptr ? __ldg(p.col_scale + n) : 1.f;
            const float bs = (!PARTIAL && p.bias != nullptr) ? to_float(static_cast<const T*>(p.bias)[n]) : 0.f;
#pragma unroll 4
            for (int r = lane / ST; r < 32; r += 32 / ST) {
              const int m = row_base + r;
              if (m >= p.M) break;
              float v = tr[r * LD + cl];
              if (PL == 2) v = v * (p.row_scale != nullptr ? __ldg(p.row_scale + m) : 1.f) * cs;
              if (PARTIAL) {
                p.partial[(long long)z * p.split_stride + (long long)m * p.ldp + n] = v;
              } else {
                v += bs;
                if (p.activation != B200GRU_ACT_NONE) {
                  const Activated a = activate_as(p.activation, v);
                  v = a.y;
                  if (p.slope != nullptr) static_cast<S*>(p.slope)[(long long)m * p.lds + n] = from_float<S>(a.slope);
                }
                if (resp != nullptr) v += to_float(resp[(long long)m * p.ldr + n]);
                static_cast<T*>(p.C)[(long long)m * p.ldc + n] = from_float<T>(v);
              }
            }
          }
        }
      }
    }
  }

  if (warp == 0 && lane == 0 && *deadp) {                 // a CTA that gave up: let tile copies in flight land
    const long long start = clock64();
    while (clock64() - start < (1ll << 18)) {
    }
  }
  tc::tc_fence_before();
  __syncthreads();
  if (CTAS == 2) pair_sync();                             // nobody leaves while the other may still signal it
  if (warp == 1) {
    __syncwarp();
    tc::tc_fence_after();
    if (CTAS == 1) tc::tmem_dealloc(tmem, 2 * BN);
    else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2 * BN) : "memory");
  }
}

// CTAs (or pairs) that the device runs at once; 0 when they cannot be launched.
int units_on_device(const void* fn, size_t smem, int ctas) {
  static std::mutex mu;
  static std::map<std::pair<int, const void*>, int> cache;
  int dev = -1;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  std::lock_guard<std::mutex> lk(mu);
  const auto key = std::make_pair(dev, fn);
  auto it = cache.find(key);
  if (it != cache.end()) return it->second;
  int n = 0;
  if (allow_dynamic_smem(fn, smem) == B200GRU_OK) {
    if (ctas == 1) {
      if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) { cudaGetLastError(); n = 0; }
    } else {
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(2); cfg.blockDim = dim3(THREADS); cfg.dynamicSmemBytes = smem;
      cudaLaunchAttribute at[1];
      at[0].id = cudaLaunchAttributeClusterDimension;
      at[0].val.clusterDim.x = 2; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
      cfg.attrs = at; cfg.numAttrs = 1;
      if (cudaOccupancyMaxActiveClusters(&n, fn, &cfg) != cudaSuccess) { cudaGetLastError(); n = 0; }
    }
  }
  cache[key] = n;
  return n;
}

template <int CTAS, int BN, bool A_MN, bool B_MN, int PL, typename Out>
int launch_variant(const Gemm& g, Params p, const CUtensorMap& ta, const CUtensorMap& tb, cudaStream_t st) {
  typedef typename Turn<Out>::T T;
  auto kernel = lin_gemm_kernel<CTAS, BN, A_MN, B_MN, PL, Out>;
  constexpr int BH = CTAS == 2 ? 128 : BN, stage = PL * (BM + BH) * 128;
  p.stages = (226 * 1024 - 1024 - TR_BYTES<T> - 512) / stage;
  if (p.stages > MAX_STAGES) p.stages = MAX_STAGES;
  const size_t smem = (size_t)p.stages * stage + TR_BYTES<T> + 1024;
  const int units = units_on_device(reinterpret_cast<const void*>(kernel), smem, CTAS);
  if (units <= 0) return B200GRU_UNSUPPORTED;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(CTAS * (p.tiles < units ? p.tiles : units)));
  cfg.blockDim = dim3(THREADS); cfg.dynamicSmemBytes = smem; cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = B200GRU_PDL_ALLOWED;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = CTAS; at[1].val.clusterDim.y = 1; at[1].val.clusterDim.z = 1;
  cfg.attrs = at; cfg.numAttrs = CTAS == 2 ? 2 : 1;
  cudaLaunchKernelEx(&cfg, kernel, ta, tb, p);
  note_launch();
  return check_launch("lin_gemm_kernel");
}

template <int CTAS, int BN, int PL, typename Out>
int launch_tile(const Gemm& g, cudaStream_t st) {
  typedef typename Turn<Out>::T T;
  typedef typename SlopeOf<T>::type S;
  Params p;
  memset(&p, 0, sizeof(p));
  p.M = g.M; p.N = g.N;
  p.tiles_m = cdiv(g.M, CTAS * BM); p.tiles_n = cdiv(g.N, BN);
  const long long tiles = (long long)p.tiles_m * p.tiles_n * g.splits;
  if (tiles > 0x3fffffff) return B200GRU_UNSUPPORTED;
  p.tiles = (int)tiles;
  p.kb_total = cdiv(g.K, 64);
  p.kb_per_split = cdiv(p.kb_total, g.splits);
  p.chunk_kb = PL == 2 ? 2 : 64;
  p.ab_format = g.fp16 ? 0u : 1u;
  p.row_scale = g.row_scale; p.col_scale = g.col_scale; p.activation = g.activation; p.bias = g.bias;
  p.residual = g.residual; p.ldr = g.ldr; p.C = g.C; p.ldc = g.ldc; p.slope = g.slope; p.lds = g.lds;
  p.partial = g.partial; p.ldp = g.ldp; p.split_stride = (long long)g.M * g.ldp;
  if (std::is_void<Out>::value) p.vec = 1;                // partial rows are padded to 16 bytes
  else p.vec = g.N % Vec<T>::V == 0 && on16(g.C, g.ldc, sizeof(T)) && on16(g.residual, g.ldr, sizeof(T)) &&
               on16(g.bias, 0, sizeof(T)) && on16(g.slope, g.lds, sizeof(S));
  if (std::is_void<Out>::value) p.N = (int)g.ldp;         // and written to their padded end

  constexpr int BH = CTAS == 2 ? 128 : BN;
  const CUtensorMapDataType dt = g.fp16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  alignas(64) CUtensorMap ta, tb;
  const unsigned long long a_rows = g.a_mn ? g.K : g.M, b_rows = g.b_mn ? g.K : g.N;
  const unsigned long long a_pl = PL > 1 ? (unsigned long long)g.a_plane * 2 : a_rows * g.lda * 2;
  const unsigned long long b_pl = PL > 1 ? (unsigned long long)g.b_plane * 2 : b_rows * g.ldb * 2;
  int rc = tc::make_tensor_map_3d(&ta, dt, g.A, g.a_mn ? g.M : g.K, a_rows, PL, (unsigned long long)g.lda * 2, a_pl, 64, g.a_mn ? 64 : BM);
  if (rc) return rc;
  rc = tc::make_tensor_map_3d(&tb, dt, g.B, g.b_mn ? g.N : g.K, b_rows, PL, (unsigned long long)g.ldb * 2, b_pl, 64, g.b_mn ? 64 : BH);
  if (rc) return rc;
  if (!g.a_mn && !g.b_mn) return launch_variant<CTAS, BN, false, false, PL, Out>(g, p, ta, tb, st);
  if (!g.a_mn && g.b_mn) return launch_variant<CTAS, BN, false, true, PL, Out>(g, p, ta, tb, st);
  if (g.a_mn && g.b_mn) return launch_variant<CTAS, BN, true, true, PL, Out>(g, p, ta, tb, st);
  return B200GRU_UNSUPPORTED;
}

template <int PL, typename Out>
int launch_plan(const Gemm& g, const Plan& plan, cudaStream_t st) {
  if (plan.ctas == 2) return launch_tile<2, 256, PL, Out>(g, st);
  if (plan.bn == 128) return launch_tile<1, 128, PL, Out>(g, st);
  return launch_tile<1, 64, PL, Out>(g, st);
}

int unit_status(int reset) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_lin_status, sizeof(int)) != cudaSuccess) return -1;
  if (reset && v != 0) {
    const int none = 0;
    cudaMemcpyToSymbol(g_lin_status, &none, sizeof(int));
  }
  return v;
}

}  // namespace

#endif  // B200GRU_LINEAR_GEMM_IMPL

}  // namespace lin
}  // namespace b200gru
