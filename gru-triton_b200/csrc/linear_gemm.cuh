// Tensor-core product of linear_act: persistent CTAs (128 x BN tiles) or CTA pairs (256 x 256), epilogue of a tile under the
// products of the next.
//
//   C[M,N] = epilogue( row_scale[m] col_scale[n] sum_p A_p[M,K] B_p[N,K]^T )
//
// Operands: one plane of bf16 or fp16, or (fp32) two row-scaled fp16 planes, of which low x high, high x low and high x high
// are summed in that order.  Either operand K-major (rows of K) or MN-major (rows of M or N, one per k).
//
// The tensor core's fp32 accumulator truncates: a sum of K terms loses up to 2^-23 of itself at each of its K / 16 steps, always
// towards zero.  So sums are built in chunks, in one of two tensor-memory buffers, and the chunks added with round-to-nearest.
// Planes: 24 steps.  16-bit types without an activation (gates of a recurrence, whose fp32 state carries every rounding of a
// gate on; gradients): 8 steps where K is at most 512, 16 up to 2048, then 32, added in registers.  With an activation 64 steps, added into the
// next buffer: its epilogue is long, and reading chunks between would hold the products up (32768 x 1024 -> 4096 bf16, gelu: 196 us;
// 241 with 32 steps, 304 with 16; none: 198 us with 16, 177 with one chunk).  Share of bf16 results that are not the rounding of the exact
// sum, K 512 / 1024 / 4096: 1.0 / 1.8 / 3.4e-4 (one chunk: 2.8 / 5.6 / 23e-4; fp32 multiply-adds: 1.2 / 1.7 / 3.7e-4).
//
// Roles of a CTA's ten warps: 0 loads k-blocks by TMA, 1 issues tcgen05.mma, 2-9 drain the accumulator (32 rows and half the
// columns each; a lane has a row).  Results, slopes and residual move as TMA tiles of 32 rows x 128 bytes through swizzled
// shared memory of the warp's own: the residual of the next columns lands while these are computed, and results are added
// in its place.  (Rows turned through shared memory and stored by the warp cost as many instructions again as the activation.)
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
// K-blocks of 64 terms in a chunk (see above).
inline int chunk_kblocks(int planes, bool activation, int kb_per_split) {
  if (planes == 2) return 2;
  if (activation) return 16;
  return kb_per_split <= 8 ? 2 : kb_per_split <= 32 ? 4 : 8;
}
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
template <int B, int L> struct Vec<Slope16<B, L>> { static constexpr int V = 8; };

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
  int with_residual, with_slope;
  int out_mask;                              // 1: two result buffers a warp in turn, 0: one (beside one for slopes)
  unsigned ab_format;
  const float* row_scale;
  const float* col_scale;
  const void* bias;
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

// How a warp's results leave: groups of 32 rows x 128 bytes (64 for a 64-wide tile of a 16-bit type).
template <typename Out> struct Leaves { typedef Out T; };
template <> struct Leaves<void> { typedef float T; };
template <typename T, int NC>
struct Group {
  static constexpr int COLS = 128 / (int)sizeof(T) < NC ? 128 / (int)sizeof(T) : NC;
  static constexpr int ROW_BYTES = COLS * (int)sizeof(T), BYTES = 32 * ROW_BYTES, COUNT = NC / COLS;
  // Byte of 16-byte piece c of row r: the swizzle of TMA tiles this wide.
  static __device__ __forceinline__ uint32_t piece(int r, int c) {
    return (uint32_t)(r * ROW_BYTES + ((c ^ (ROW_BYTES == 128 ? r & 7 : (r >> 1) & 3)) << 4));
  }
};
constexpr int WARP_OUT = 4096;               // bytes of a warp's tile buffer
constexpr int WARP_COEF = 128 * 8;           // its columns' bias and scale

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
// At most N of this thread's latest tile stores may still be reading shared memory.
template <int N>
__device__ __forceinline__ void stores_read() { asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory"); }

// A warp's shared memory, and how many groups it has sent: group i uses buffer i & 1.
struct Lane {
  unsigned char* out;                        // result tiles
  unsigned char* slopes;                     // slope tile
  float* coef;                               // bias[NC], scale[NC]
  uint32_t bar[2];                           // the residual of a buffer has landed
  int lane;
  int sent;
};
struct Corner { int row, col, z; };          // first row and column of the warp's part of a tile, its K slice

template <typename T, int COLS>
__device__ __forceinline__ void fetch_residual(const Params& p, const CUtensorMap* map, const Lane& w, int i, int row, int col) {
  if (w.lane == 0) {
    tc::mbar_expect_tx(w.bar[i & 1], 32 * COLS * sizeof(T));
    tc::tma_load_3d(tc::smem_u32(w.out + (i & 1) * WARP_OUT), map, col, row, 0, w.bar[i & 1]);
  }
}

// 32 columns from column c of the group on: scales, bias, activation, residual; into the buffers.  KEEP: slopes too.
template <int ACT, int PL, typename Out, int NC, bool KEEP>
__device__ __forceinline__ void finish_some(const Params& p, const Lane& w, unsigned char* out, const P2* v, float rs, int col, int c) {
  typedef typename Leaves<Out>::T T;
  typedef typename SlopeOf<T>::type S;
  typedef Group<T, NC> G;
  constexpr int V = Vec<T>::V;
  const bool add = !std::is_void<Out>::value && p.with_residual;
#pragma unroll
  for (int e = 0; e < 32; e += V) {
    P2 x[V / 2], sl[V / 2];
#pragma unroll
    for (int k = 0; k < V / 2; ++k) {
      x[k] = v[e / 2 + k];
      if (PL == 2) {
        const float2 cs = *reinterpret_cast<const float2*>(w.coef + NC + col + e + 2 * k);
        x[k] = mul2(mul2(x[k], both(rs)), pair(cs.x, cs.y));
      }
    }
    if (!std::is_void<Out>::value) {
#pragma unroll
      for (int k = 0; k < V / 2; k += 2) {
        const float4 b = *reinterpret_cast<const float4*>(w.coef + col + e + 2 * k);
        const Activated2 r0 = activate<ACT>(add2(x[k], pair(b.x, b.y))), r1 = activate<ACT>(add2(x[k + 1], pair(b.z, b.w)));
        x[k] = r0.y; x[k + 1] = r1.y;
        sl[k] = r0.slope; sl[k + 1] = r1.slope;
      }
    }
    const uint32_t at = G::piece(w.lane, (c + e) / V);
    if (KEEP) {
      float f[V];
#pragma unroll
      for (int k = 0; k < V / 2; ++k) { const float2 s = split(sl[k]); f[2 * k] = s.x; f[2 * k + 1] = s.y; }
      *reinterpret_cast<uint4*>(w.slopes + at) = pack16<S>(f);
    }
    if (add) {
      float f[V];
      unpack16<T>(*reinterpret_cast<const uint4*>(out + at), f);
#pragma unroll
      for (int k = 0; k < V / 2; ++k) x[k] = add2(x[k], pair(f[2 * k], f[2 * k + 1]));
    }
    float f[V];
#pragma unroll
    for (int k = 0; k < V / 2; ++k) { const float2 y = split(x[k]); f[2 * k] = y.x; f[2 * k + 1] = y.y; }
    *reinterpret_cast<uint4*>(out + at) = pack16<T>(f);
  }
}

template <int ACT, int PL, typename Out, int NC>
__device__ __forceinline__ void finish_columns(const Params& p, const Lane& w, unsigned char* out, const P2* v, float rs, int col, int c) {
  if (ACT != B200GRU_ACT_NONE && p.with_slope) finish_some<ACT, PL, Out, NC, true>(p, w, out, v, rs, col, c);
  else finish_some<ACT, PL, Out, NC, false>(p, w, out, v, rs, col, c);
}

// Before a group's columns are written: its buffer is free, its residual there, the next group's requested.
template <typename Out, int NC>
__device__ __forceinline__ bool open_group(const Params& p, const CUtensorMap* tmR, Lane& w, const Corner& next, bool more, volatile int* dead, int* status) {
  typedef typename Leaves<Out>::T T;
  typedef Group<T, NC> G;
  if (!std::is_void<Out>::value && p.with_residual) {
    if (w.lane == 0) stores_read<0>();
    __syncwarp();
    if (more) fetch_residual<T, G::COLS>(p, tmR, w, w.sent + 1, next.row, next.col);
    return __all_sync(0xffffffffu, tc::mbar_wait(w.bar[w.sent & 1], (uint32_t)(w.sent >> 1) & 1u, dead, status));
  }
  if (w.lane == 0) {
    if (p.with_slope) stores_read<0>();
    else stores_read<1>();
  }
  __syncwarp();
  return true;
}
// Tile store whose lines leave L2 before others: results pass through, the operands are read again (6 % of 32768 x 2048 -> 4096 with
// gelu, 9 % where slopes are kept).
__device__ __forceinline__ void store_tile(const CUtensorMap* map, int c0, int c1, int c2, uint32_t src, uint64_t policy) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group.L2::cache_hint [%0, {%1, %2, %3}], [%4], %5;"
               ::"l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(src), "l"(policy) : "memory");
}
// The group's results (and slopes) start on their way.
template <typename Out, int NC>
__device__ __forceinline__ void close_group(const Params& p, const CUtensorMap* tmC, const CUtensorMap* tmS, Lane& w, const Corner& at, int col) {
  tc::fence_async_smem();
  __syncwarp();
  if (w.lane == 0) {
    const uint32_t from = tc::smem_u32(w.out + (w.sent & p.out_mask) * WARP_OUT);
    if (std::is_void<Out>::value) {
      tc::tma_store_3d(tmC, at.col + col, at.row, at.z, from);       // read again at once
    } else {
      uint64_t policy;
      asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
      store_tile(tmC, at.col + col, at.row, 0, from, policy);
      if (p.with_slope) store_tile(tmS, at.col + col, at.row, 0, tc::smem_u32(w.slopes), policy);
    }
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
  }
  ++w.sent;
}

// Out = void: partial sums in fp32.  IN_REGISTERS: where the chunks of a tile are added up.
template <int CTAS, int BN, bool A_MN, bool B_MN, int PL, int ACT, typename Out, bool IN_REGISTERS>
__global__ void __launch_bounds__(THREADS, 1)
lin_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                const __grid_constant__ CUtensorMap tmC, const __grid_constant__ CUtensorMap tmS,
                const __grid_constant__ CUtensorMap tmR, const Params p) {
  typedef typename Leaves<Out>::T T;
  constexpr int BH = CTAS == 2 ? 128 : BN;               // rows of B per CTA
  constexpr int A_PLANE = BM * 128, B_PLANE = BH * 128, STAGE = PL * (A_PLANE + B_PLANE);
  constexpr int UMMA_K = 16, NC = BN / 2;                // accumulator columns per epilogue thread
  constexpr bool PARTIAL = std::is_void<Out>::value;
  const uint32_t IDESC = tc::umma_idesc(false, A_MN, B_MN, CTAS * BM, BN, p.ab_format);

  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  __shared__ __align__(8) unsigned long long bar_full[MAX_STAGES], bar_empty[MAX_STAGES];
  __shared__ __align__(8) unsigned long long bar_acc_full[2], bar_acc_empty[2], bar_res[EPI_WARPS][2];
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
      for (int w = 0; w < EPI_WARPS; ++w) tc::mbar_init(tc::smem_u32(&bar_res[w][b]), 1);
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

  // tile index -> K slice, row panel, column panel.  Tiles run down bands of eight row panels, column by column: what runs at
  // a time is about as high as wide, and reads the least of A and B (8192^3 bf16, where a row of tiles would draw all of B
  // through L2: 929 -> 855 us).
  auto locate = [&](int t, int& m0, int& n0, int& z, int& kb0, int& nkb) {
    constexpr int BAND = 8;
    const int plane = p.tiles_m * p.tiles_n;
    z = t / plane;
    const int r = t - z * plane, band = r / (BAND * p.tiles_n), first = band * BAND;
    const int high = min(BAND, p.tiles_m - first), i = r - band * BAND * p.tiles_n;
    n0 = (i / high) * BN;
    m0 = (first + i % high) * CTAS * BM + (int)rank * BM;
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
    typedef Group<T, NC> G;
    const int q = warp & 3, half = (warp - 2) >> 2, me = warp - 2;
    unsigned char* tail = smem + p.stages * STAGE;           // buffers of the warps, 1024-byte aligned
    Lane w;
    const int buffers = 1 + p.out_mask + p.with_slope;
    w.out = tail + me * buffers * WARP_OUT;
    w.slopes = w.out + (1 + p.out_mask) * WARP_OUT;
    w.coef = reinterpret_cast<float*>(tail + EPI_WARPS * buffers * WARP_OUT + me * WARP_COEF);
    w.bar[0] = tc::smem_u32(&bar_res[me][0]); w.bar[1] = tc::smem_u32(&bar_res[me][1]);
    w.lane = lane; w.sent = 0;
    int c = 0;
    bool ok = __all_sync(0xffffffffu, *deadp == 0);
    // the next tile from t on in which this warp has columns (a narrow matrix ends before its half of the tile)
    auto next_tile = [&](int t, Corner& at) {
      for (; t < p.tiles; t += units) {
        int m0, n0, z, kb0, nkb;
        locate(t, m0, n0, z, kb0, nkb);
        at = Corner{m0 + q * 32, n0 + half * NC, z};
        if (at.col < p.N) return true;
      }
      return false;
    };
    Corner then = {0, 0, 0};
    if (!PARTIAL && p.with_residual && ok && next_tile(unit, then)) fetch_residual<T, G::COLS>(p, &tmR, w, 0, then.row, then.col);
    for (int t = unit; t < p.tiles && ok; t += units) {
      int m0, n0, z, kb0, nkb;
      locate(t, m0, n0, z, kb0, nkb);
      const Corner at = {m0 + q * 32, n0 + half * NC, z};
      bool last = true;
      if (!PARTIAL && p.with_residual) last = !next_tile(t + units, then);
      const int chunks = (nkb + p.chunk_kb - 1) / p.chunk_kb;
      // bias and scales of the columns; the row's scale
      __syncwarp();
      for (int j = lane; j < NC; j += 32) {
        const int n = at.col + j;
        if (!PARTIAL) w.coef[j] = (p.bias != nullptr && n < p.N) ? to_float(static_cast<const T*>(p.bias)[n]) : 0.f;
        if (PL == 2) w.coef[NC + j] = (p.col_scale != nullptr && n < p.N) ? __ldg(p.col_scale + n) : 1.f;
      }
      __syncwarp();
      float rs = 1.f;
      if (PL == 2 && p.row_scale != nullptr && at.row + lane < p.M) rs = __ldg(p.row_scale + at.row + lane);
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
          // relaxed: a release would wait for results on their way to memory
          if (CTAS == 2) asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(at_leader(own)) : "memory");
          else tc::mbar_arrive(own);
        }
      };
      auto source = [&](int buf) { return tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(buf * BN + half * NC); };
      auto open = [&](int g) {
        const bool here = g + 1 < G::COUNT && at.col + (g + 1) * G::COLS < p.N;
        return open_group<Out, NC>(p, &tmR, w, here ? Corner{at.row, at.col + (g + 1) * G::COLS, 0} : then, here || !last, deadp, status);
      };
      auto close = [&](int g) { close_group<Out, NC>(p, &tmC, &tmS, w, at, g * G::COLS); };
      if (!IN_REGISTERS) {
        // One chunk, or few long ones: a total of more is summed in registers and put back, so that the way out is one: from tensor
        // memory, the next 32 columns requested before these are finished.
        const int buf0 = c & 1;
        ok = landed(buf0);
        if (!ok) break;
        int buf = buf0;
        for (int i = 1; i < chunks; ++i) {                   // add this buffer's sums to the next one's
          ++c;
          ok = landed(buf ^ 1);
          if (!ok) break;
#pragma unroll 1
          for (int c0 = 0; c0 < NC; c0 += 32) {
            uint32_t v[32], u[32];
            tc::tmem_ld32(source(buf) + (uint32_t)c0, v);
            tc::tmem_ld32(source(buf ^ 1) + (uint32_t)c0, u);
            tc::tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 32; ++j) u[j] = __float_as_uint(__uint_as_float(v[j]) + __uint_as_float(u[j]));
            tmem_st32(source(buf ^ 1) + (uint32_t)c0, u);
          }
          tmem_st_wait();
          release(buf);
          buf ^= 1;
        }
        if (!ok) break;
        uint32_t v[32];
        tc::tmem_ld32(source(buf), v);
#pragma unroll 1
        for (int g = 0; g < G::COUNT; ++g) {
          if (at.col + g * G::COLS >= p.N) break;            // warp-uniform
          ok = open(g);
          unsigned char* out = w.out + (w.sent & p.out_mask) * WARP_OUT;
#pragma unroll
          for (int c0 = 0; c0 < G::COLS; c0 += 32) {
            const int col = g * G::COLS + c0;
            tc::tmem_ld_wait();
            P2 x[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) x[j] = pair(__uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1]));
            if (col + 32 < NC) tc::tmem_ld32(source(buf) + (uint32_t)(col + 32), v);
            finish_columns<ACT, PL, Out, NC>(p, w, out, x, rs, col, c0);
          }
          close(g);
        }
        tc::tmem_ld_wait();
        release(buf);
        ++c;
      } else {
        // chunks are short, so the totals stay in registers and a buffer is free at once
        P2 acc[NC / 2];
#pragma unroll
        for (int j = 0; j < NC / 2; ++j) acc[j] = both(0.f);
        for (int i = 0; i < chunks; ++i, ++c) {
          const int buf = c & 1;
          ok = landed(buf);
          if (!ok) break;
#pragma unroll
          for (int c0 = 0; c0 < NC; c0 += 16) {
            uint32_t v[16];
            tc::tmem_ld16(source(buf) + (uint32_t)c0, v);
            tc::tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 16; j += 2)
              acc[(c0 + j) / 2] = add2(acc[(c0 + j) / 2], pair(__uint_as_float(v[j]), __uint_as_float(v[j + 1])));
          }
          release(buf);
        }
        if (!ok) break;
#pragma unroll
        for (int g = 0; g < G::COUNT; ++g) {
          if (at.col + g * G::COLS >= p.N) break;            // warp-uniform
          if (ok) ok = open(g);
          unsigned char* out = w.out + (w.sent & p.out_mask) * WARP_OUT;
#pragma unroll
          for (int c0 = 0; c0 < G::COLS; c0 += 32)
            finish_columns<ACT, PL, Out, NC>(p, w, out, acc + (g * G::COLS + c0) / 2, rs, g * G::COLS + c0, c0);
          close(g);
        }
      }
    }
    // shared memory is read, and results are in memory, before the CTA ends; a residual that nobody took has landed
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
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

struct Maps {
  alignas(64) CUtensorMap a, b, c, slope, residual;
};

template <int CTAS, int BN, bool A_MN, bool B_MN, int PL, int ACT, typename Out, bool IN_REGISTERS>
int launch_kernel(Params p, const Maps& m, cudaStream_t st) {
  auto kernel = lin_gemm_kernel<CTAS, BN, A_MN, B_MN, PL, ACT, Out, IN_REGISTERS>;
  constexpr int BH = CTAS == 2 ? 128 : BN, stage = PL * (BM + BH) * 128;
  const int tail = EPI_WARPS * ((1 + p.out_mask + p.with_slope) * WARP_OUT + WARP_COEF);
  p.stages = (227 * 1024 - 1024 - 512 - tail) / stage;       // 512: barriers
  if (p.stages > MAX_STAGES) p.stages = MAX_STAGES;
  const size_t smem = (size_t)p.stages * stage + tail + 1024;
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
  cudaLaunchKernelEx(&cfg, kernel, m.a, m.b, m.c, m.slope, m.residual, p);
  note_launch();
  return check_launch("lin_gemm_kernel");
}

// Short chunks are added in registers; one chunk alone leaves from tensor memory at once (16384 x 120 -> 608 bf16: 13.4 us against
// 15.4), and so do the long chunks before an activation.
template <int CTAS, int BN, bool A_MN, bool B_MN, int PL, int ACT, typename Out>
int launch_variant(const Params& p, const Maps& m, cudaStream_t st) {
  if constexpr (PL == 2) return launch_kernel<CTAS, BN, A_MN, B_MN, PL, ACT, Out, true>(p, m, st);
  else if constexpr (ACT != B200GRU_ACT_NONE) return launch_kernel<CTAS, BN, A_MN, B_MN, PL, ACT, Out, false>(p, m, st);
  else if (p.kb_per_split > p.chunk_kb) return launch_kernel<CTAS, BN, A_MN, B_MN, PL, ACT, Out, true>(p, m, st);
  else return launch_kernel<CTAS, BN, A_MN, B_MN, PL, ACT, Out, false>(p, m, st);
}

template <typename T> struct MapType;
template <> struct MapType<float> { static constexpr CUtensorMapDataType value = CU_TENSOR_MAP_DATA_TYPE_FLOAT32; };
template <> struct MapType<__nv_bfloat16> { static constexpr CUtensorMapDataType value = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16; };
template <> struct MapType<__half> { static constexpr CUtensorMapDataType value = CU_TENSOR_MAP_DATA_TYPE_FLOAT16; };
template <int B, int L> struct MapType<Slope16<B, L>> { static constexpr CUtensorMapDataType value = CU_TENSOR_MAP_DATA_TYPE_UINT16; };

template <int CTAS, int BN, int PL, typename Out>
int launch_tile(const Gemm& g, cudaStream_t st) {
  typedef typename Leaves<Out>::T T;
  typedef typename SlopeOf<T>::type S;
  typedef Group<T, BN / 2> G;
  constexpr bool PARTIAL = std::is_void<Out>::value;
  Params p;
  memset(&p, 0, sizeof(p));
  p.M = g.M; p.N = g.N;
  p.tiles_m = cdiv(g.M, CTAS * BM); p.tiles_n = cdiv(g.N, BN);
  const long long tiles = (long long)p.tiles_m * p.tiles_n * g.splits;
  if (tiles > 0x3fffffff) return B200GRU_UNSUPPORTED;
  p.tiles = (int)tiles;
  p.kb_total = cdiv(g.K, 64);
  p.kb_per_split = cdiv(p.kb_total, g.splits);
  p.chunk_kb = chunk_kblocks(PL, !PARTIAL && g.activation != B200GRU_ACT_NONE, p.kb_per_split);
  p.ab_format = g.fp16 ? 0u : 1u;
  p.row_scale = g.row_scale; p.col_scale = g.col_scale; p.bias = g.bias;
  p.with_residual = !PARTIAL && g.residual != nullptr;
  p.with_slope = !PARTIAL && g.slope != nullptr && g.activation != B200GRU_ACT_NONE;
  p.out_mask = p.with_slope && !p.with_residual ? 0 : 1;    // shared memory for a fourth stage of operands

  constexpr int BH = CTAS == 2 ? 128 : BN;
  const CUtensorMapDataType dt = g.fp16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  Maps m;
  memset(&m, 0, sizeof(m));
  const unsigned long long a_rows = g.a_mn ? g.K : g.M, b_rows = g.b_mn ? g.K : g.N;
  const unsigned long long a_pl = PL > 1 ? (unsigned long long)g.a_plane * 2 : a_rows * g.lda * 2;
  const unsigned long long b_pl = PL > 1 ? (unsigned long long)g.b_plane * 2 : b_rows * g.ldb * 2;
  int rc = tc::make_tensor_map_3d(&m.a, dt, g.A, g.a_mn ? g.M : g.K, a_rows, PL, (unsigned long long)g.lda * 2, a_pl, 64, g.a_mn ? 64 : BM);
  if (rc == B200GRU_OK) rc = tc::make_tensor_map_3d(&m.b, dt, g.B, g.b_mn ? g.N : g.K, b_rows, PL, (unsigned long long)g.ldb * 2, b_pl, 64, g.b_mn ? 64 : BH);
  // rows of results; partial sums end at N too, in rows padded for 16-byte alignment
  auto rows_map = [&](CUtensorMap* map, CUtensorMapDataType type, const void* base, long long cols, int slices, long long ld, size_t es) {
    return tc::make_tensor_map_out(map, type, base, cols, g.M, slices, (unsigned long long)ld * es, (unsigned long long)g.M * ld * es,
                                   G::COLS, 32, G::ROW_BYTES);
  };
  if (rc == B200GRU_OK) rc = PARTIAL ? rows_map(&m.c, MapType<T>::value, g.partial, g.N, g.splits, g.ldp, sizeof(T))
                                     : rows_map(&m.c, MapType<T>::value, g.C, g.N, 1, g.ldc, sizeof(T));
  if (rc == B200GRU_OK && p.with_slope) rc = rows_map(&m.slope, MapType<S>::value, g.slope, g.N, 1, g.lds, sizeof(S));
  if (rc == B200GRU_OK && p.with_residual) rc = rows_map(&m.residual, MapType<T>::value, g.residual, g.N, 1, g.ldr, sizeof(T));
  if (rc != B200GRU_OK) return rc;
  constexpr int NONE = B200GRU_ACT_NONE;
  if (g.a_mn && g.b_mn) return launch_variant<CTAS, BN, true, true, PL, NONE, Out>(p, m, st);
  if (!g.a_mn && g.b_mn) return launch_variant<CTAS, BN, false, true, PL, NONE, Out>(p, m, st);
  if (g.a_mn) return B200GRU_UNSUPPORTED;
  if constexpr (!PARTIAL) {                               // one kernel for each activation: chosen once an element, it cost ten products
    switch (g.activation) {
      case B200GRU_ACT_RELU: return launch_variant<CTAS, BN, false, false, PL, B200GRU_ACT_RELU, Out>(p, m, st);
      case B200GRU_ACT_SILU: return launch_variant<CTAS, BN, false, false, PL, B200GRU_ACT_SILU, Out>(p, m, st);
      case B200GRU_ACT_GELU: return launch_variant<CTAS, BN, false, false, PL, B200GRU_ACT_GELU, Out>(p, m, st);
      case B200GRU_ACT_SIGMOID: return launch_variant<CTAS, BN, false, false, PL, B200GRU_ACT_SIGMOID, Out>(p, m, st);
      case B200GRU_ACT_TANH: return launch_variant<CTAS, BN, false, false, PL, B200GRU_ACT_TANH, Out>(p, m, st);
    }
  }
  return launch_variant<CTAS, BN, false, false, PL, NONE, Out>(p, m, st);
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
