// Tensor-core product of linear_act: persistent CTAs (128 x BN tiles) or CTA pairs (256 x 256), epilogue of a tile under the
// products of the next.
//
//   C[M,N] = epilogue( row_scale[m] col_scale[n] sum_p A_p[M,K] B_p[N,K]^T )
//
// Operands: one plane of bf16 or fp16, or (fp32) two row-scaled fp16 planes, of which low x high, high x low and high x high
// are summed in that order.  Either operand K-major (rows of K) or MN-major (rows of M or N, one per k).  The tensor core's
// fp32 accumulator truncates, so sums are built in chunks (24 steps for planes; 512 for 16-bit types: 512 losses of 2^-23 stay
// a quarter of half a step of fp16) in one of two tensor-memory buffers and added to register totals with round-to-nearest.
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

// 32 lanes x 32 consecutive columns back into tensor memory.
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
      ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
        "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]),
        "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]),
        "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31]) : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// First row and column of a warp's part of a tile, and its K slice.
struct Corner {
  int row, col, z;
};

// The residual of 32 rows and the lane's V columns from n on, four rows a lane.
template <typename T>
__device__ __forceinline__ void request_residual(const Params& p, const Corner& at, int n, int lane, uint4 (&res)[4]) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int m = at.row + k * 8 + (lane >> 2);
    res[k] = make_uint4(0, 0, 0, 0);
    if (m < p.M && n < p.N) res[k] = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(p.residual) + (long long)m * p.ldr + n));
  }
}

// STEP columns from column j of the warp's part on, which lie in the transpose buffer as rows: scales, bias, activation,
// residual, and out.
template <int ACT, int PL, typename Out>
__device__ __forceinline__ void store_step(const Params& p, const float* tr, const Corner& at, int j, int lane, const uint4 (&res)[4]) {
  typedef typename Turn<Out>::T T;
  typedef typename SlopeOf<T>::type S;
  constexpr bool PARTIAL = std::is_void<Out>::value;
  constexpr int V = Vec<T>::V, ST = STEP<T>, LD = TR_LD<T>;
  if (p.vec) {
    const int rsub = lane >> 2, csub = (lane & 3) * V, n = at.col + j + csub;
    if (n >= p.N) return;                                  // N is a multiple of V
    float cs[V], bs[V];
    if (PL == 2) {
#pragma unroll
      for (int e = 0; e < V; ++e) cs[e] = p.col_scale != nullptr ? __ldg(p.col_scale + n + e) : 1.f;
    }
    if (!PARTIAL) {
#pragma unroll
      for (int e = 0; e < V; ++e) bs[e] = 0.f;
      if (p.bias != nullptr) unpack16<T>(__ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(p.bias) + n)), bs);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int m = at.row + k * 8 + rsub;
      if (m >= p.M) continue;
      float v[V];
#pragma unroll
      for (int e = 0; e < V; e += 4) {
        const float4 f = *reinterpret_cast<const float4*>(tr + (k * 8 + rsub) * LD + csub + e);
        v[e] = f.x; v[e + 1] = f.y; v[e + 2] = f.z; v[e + 3] = f.w;
      }
      if (PL == 2) {
        const float rs = p.row_scale != nullptr ? __ldg(p.row_scale + m) : 1.f;
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = v[e] * rs * cs[e];
      }
      if (PARTIAL) {
        *reinterpret_cast<float4*>(p.partial + (long long)at.z * p.split_stride + (long long)m * p.ldp + n) = make_float4(v[0], v[1], v[2], v[3]);
        continue;
      }
      float sl[V];
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const Activated r = activate<ACT>(v[e] + bs[e]);
        v[e] = r.y;
        sl[e] = r.slope;
      }
      if (ACT != B200GRU_ACT_NONE && p.slope != nullptr)
        *reinterpret_cast<uint4*>(static_cast<S*>(p.slope) + (long long)m * p.lds + n) = pack16<S>(sl);
      if (p.residual != nullptr) {
        float rv[V];
        unpack16<T>(res[k], rv);
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] += rv[e];
      }
      *reinterpret_cast<uint4*>(static_cast<T*>(p.C) + (long long)m * p.ldc + n) = pack16<T>(v);
    }
  } else {
    // rows that lie on no boundary: a column per lane
    const int cl = lane % ST, n = at.col + j + cl;
    if (n >= p.N) return;
    const float cs = p.col_scale != nullptr ? __ldg(p.col_scale + n) : 1.f;
    const float bs = (!PARTIAL && p.bias != nullptr) ? to_float(static_cast<const T*>(p.bias)[n]) : 0.f;
#pragma unroll 4
    for (int r = lane / ST; r < 32; r += 32 / ST) {
      const int m = at.row + r;
      if (m >= p.M) break;
      float v = tr[r * LD + cl];
      if (PL == 2) v = v * (p.row_scale != nullptr ? __ldg(p.row_scale + m) : 1.f) * cs;
      if (PARTIAL) {
        p.partial[(long long)at.z * p.split_stride + (long long)m * p.ldp + n] = v;
        continue;
      }
      const Activated a = activate<ACT>(v + bs);
      v = a.y;
      if (ACT != B200GRU_ACT_NONE && p.slope != nullptr) static_cast<S*>(p.slope)[(long long)m * p.lds + n] = from_float<S>(a.slope);
      if (p.residual != nullptr) v += to_float(static_cast<const T*>(p.residual)[(long long)m * p.ldr + n]);
      static_cast<T*>(p.C)[(long long)m * p.ldc + n] = from_float<T>(v);
    }
  }
}

// The tail of a tile from tensor memory: 32 columns at a time, the next ones requested before these are finished.
template <int ACT, int PL, int NC, typename Out>
__device__ __forceinline__ void from_tmem(const Params& p, float* tr, uint32_t src, const Corner& at, int lane) {
  typedef typename Turn<Out>::T T;
  constexpr int ST = STEP<T>, LD = TR_LD<T>, V = Vec<T>::V;
  const bool ahead = !std::is_void<Out>::value && p.vec && p.residual != nullptr;
  uint4 res[4];
  if (ahead) request_residual<T>(p, at, at.col + (lane & 3) * V, lane, res);
#pragma unroll 1
  for (int c0 = 0; c0 < NC; c0 += 32) {
    if (at.col + c0 >= p.N) break;                         // warp-uniform
    uint32_t v[32];
    tc::tmem_ld32(src + (uint32_t)c0, v);
    tc::tmem_ld_wait();
#pragma unroll
    for (int s = 0; s < 32; s += ST) {
      if (at.col + c0 + s >= p.N) break;
      __syncwarp();
#pragma unroll
      for (int e = 0; e < ST; e += 4)
        *reinterpret_cast<uint4*>(tr + lane * LD + e) = make_uint4(v[s + e], v[s + e + 1], v[s + e + 2], v[s + e + 3]);
      __syncwarp();
      uint4 now[4];
      if (ahead) {
#pragma unroll
        for (int k = 0; k < 4; ++k) now[k] = res[k];
        if (c0 + s + ST < NC) request_residual<T>(p, at, at.col + c0 + s + ST + (lane & 3) * V, lane, res);
      }
      store_step<ACT, PL, Out>(p, tr, at, c0 + s, lane, now);
    }
  }
}
// The same from totals in registers.
template <int ACT, int PL, int NC, typename Out>
__device__ __forceinline__ void from_registers(const Params& p, float* tr, const float (&acc)[NC], const Corner& at, int lane) {
  typedef typename Turn<Out>::T T;
  constexpr int ST = STEP<T>, LD = TR_LD<T>, V = Vec<T>::V;
  const bool ahead = !std::is_void<Out>::value && p.vec && p.residual != nullptr;
  uint4 res[4];
  if (ahead) request_residual<T>(p, at, at.col + (lane & 3) * V, lane, res);
#pragma unroll
  for (int j = 0; j < NC; j += ST) {
    if (at.col + j >= p.N) break;                          // warp-uniform
    __syncwarp();
#pragma unroll
    for (int e = 0; e < ST; e += 4)
      *reinterpret_cast<float4*>(tr + lane * LD + e) = make_float4(acc[j + e], acc[j + e + 1], acc[j + e + 2], acc[j + e + 3]);
    __syncwarp();
    uint4 now[4];
    if (ahead) {
#pragma unroll
      for (int k = 0; k < 4; ++k) now[k] = res[k];
      if (j + ST < NC) request_residual<T>(p, at, at.col + j + ST + (lane & 3) * V, lane, res);
    }
    store_step<ACT, PL, Out>(p, tr, at, j, lane, now);
  }
}

// Out = void: partial sums in fp32.
template <int CTAS, int BN, bool A_MN, bool B_MN, int PL, int ACT, typename Out>
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
    constexpr int LD = TR_LD<T>;
    const int q = warp & 3, half = (warp - 2) >> 2;
    float* tr = reinterpret_cast<float*>(smem + p.stages * STAGE) + (warp - 2) * 32 * LD;
    int c = 0;
    bool ok = __all_sync(0xffffffffu, *deadp == 0);
    for (int t = unit; t < p.tiles && ok; t += units) {
      int m0, n0, z, kb0, nkb;
      locate(t, m0, n0, z, kb0, nkb);
      Corner at = {m0 + q * 32, n0 + half * NC, z};
      const int chunks = (nkb + p.chunk_kb - 1) / p.chunk_kb;
      auto landed = [&](int buf) {
        const bool there = __all_sync(0xffffffffu, tc::mbar_wait(tc::smem_u32(&bar_acc_full[buf]), (c >> 1) & 1, deadp, status));
        tc::tc_fence_after();
        return there;
      };
      auto release = [&](int buf) {
        tc::tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          const uint32_t own = tc::smem_u32(&bar_acc_empty[buf]);
          if (CTAS == 2) asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(at_leader(own)) : "memory");
          else tc::mbar_arrive(own);
        }
      };
      auto source = [&](int buf) { return tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(buf * BN + half * NC); };
      if (PL == 1 && chunks == 1) {
        // one chunk: results go from tensor memory to the transpose buffer, 32 columns at a time
        const int buf = c & 1;
        ok = landed(buf);
        if (!ok) break;
        from_tmem<ACT, PL, NC, Out>(p, tr, source(buf), at, lane);
        release(buf);
        ++c;
        continue;
      }
      float acc[NC];
#pragma unroll
      for (int j = 0; j < NC; ++j) acc[j] = 0.f;
      for (int i = 0; i < chunks; ++i, ++c) {
        const int buf = c & 1;
        ok = landed(buf);
        if (!ok) break;
        if (PL == 2) {
#pragma unroll
          for (int c0 = 0; c0 < NC; c0 += 16) {
            uint32_t v[16];
            tc::tmem_ld16(source(buf) + (uint32_t)c0, v);
            tc::tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 16; ++j) acc[c0 + j] += __uint_as_float(v[j]);
          }
        } else {
#pragma unroll
          for (int c0 = 0; c0 < NC; c0 += 32) {
            uint32_t v[32];
            tc::tmem_ld32(source(buf) + (uint32_t)c0, v);
            tc::tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 32; ++j) acc[c0 + j] += __uint_as_float(v[j]);
            if (i == chunks - 1) {                        // the totals go back: the tail is the same as above
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] = __float_as_uint(acc[c0 + j]);
              tmem_st32(source(buf) + (uint32_t)c0, v);
            }
          }
        }
        if (PL == 1 && i == chunks - 1) {
          tmem_st_wait();
          from_tmem<ACT, PL, NC, Out>(p, tr, source(buf), at, lane);
        }
        release(buf);
      }
      if (!ok) break;
      // planes: chunks are short, so the totals stay in registers and the buffer is free at once
      if (PL == 2) from_registers<ACT, PL, NC, Out>(p, tr, acc, at, lane);
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

template <int CTAS, int BN, bool A_MN, bool B_MN, int PL, int ACT, typename Out>
int launch_variant(const Gemm& g, Params p, const CUtensorMap& ta, const CUtensorMap& tb, cudaStream_t st) {
  typedef typename Turn<Out>::T T;
  auto kernel = lin_gemm_kernel<CTAS, BN, A_MN, B_MN, PL, ACT, Out>;
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
  p.chunk_kb = PL == 2 ? 2 : 128;
  p.ab_format = g.fp16 ? 0u : 1u;
  p.row_scale = g.row_scale; p.col_scale = g.col_scale; p.bias = g.bias;
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
  constexpr int NONE = B200GRU_ACT_NONE;
  if (g.a_mn && g.b_mn) return launch_variant<CTAS, BN, true, true, PL, NONE, Out>(g, p, ta, tb, st);
  if (!g.a_mn && g.b_mn) return launch_variant<CTAS, BN, false, true, PL, NONE, Out>(g, p, ta, tb, st);
  if (g.a_mn) return B200GRU_UNSUPPORTED;
  if constexpr (!std::is_void<Out>::value) {              // one kernel for each activation: chosen once an element, it cost 30 products
    switch (g.activation) {
      case B200GRU_ACT_RELU: return launch_variant<CTAS, BN, false, false, PL, B200GRU_ACT_RELU, Out>(g, p, ta, tb, st);
      case B200GRU_ACT_SILU: return launch_variant<CTAS, BN, false, false, PL, B200GRU_ACT_SILU, Out>(g, p, ta, tb, st);
      case B200GRU_ACT_GELU: return launch_variant<CTAS, BN, false, false, PL, B200GRU_ACT_GELU, Out>(g, p, ta, tb, st);
      case B200GRU_ACT_SIGMOID: return launch_variant<CTAS, BN, false, false, PL, B200GRU_ACT_SIGMOID, Out>(g, p, ta, tb, st);
      case B200GRU_ACT_TANH: return launch_variant<CTAS, BN, false, false, PL, B200GRU_ACT_TANH, Out>(g, p, ta, tb, st);
    }
  }
  return launch_variant<CTAS, BN, false, false, PL, NONE, Out>(g, p, ta, tb, st);
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
