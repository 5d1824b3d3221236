// Gated linear recurrence: the GRU update with gates from the input alone.
//
//   z = sigmoid(x)   n = tanh(c) or c   h_t = z h_{t-1} + (1 - z) n        gi[t,b,:] = (x[H], c[H])
//
// Each (row, unit) is a chain of its own whose steps are affine maps h -> z h + u.  Maps compose,
// (A2, b2) o (A1, b1) = (A2 A1, A2 b1 + b2), so time is cut: a thread folds 8 or 16 steps of two units, a CTA a tile (64 steps
// of 64 units; where rows are few 128 of 32), and a cluster of up to 16 CTAs takes that many tiles of the same units at once.
// Maps are joined in the order of time at every level (through shared memory, then through the cluster's), never in the order
// of arrival.
// The backward pass is the same scan in the other direction, G_t = z_t (dout_t + G_{t+1}), with the same products of z; it
// recomputes the states of a tile from the one that the forward kept, so `out` is not read again.
//
// Bound: bytes (forward 3, backward 5 elements of traffic a step and unit).  The gates are computed once and stay in
// registers between the fold and the results; inputs arrive by TMA a few tiles ahead.

#include <cstring>
#include <map>
#include <mutex>
#include <tuple>
#include <type_traits>

#include "gated_scan.cuh"
#include "tc_common.cuh"

namespace b200gru {
namespace gated {

__device__ int g_gated_status;

namespace {

constexpr int STAGES_MAX = 4;

// L threads side by side have the units of a tile (two each), P of them one behind the other its steps (S each).
template <int L, int P, int S>
struct Tile {
  static constexpr int LANES = L, PARTS = P, SEG = S, THREADS = L * P, UNITS = 2 * L, STEPS = P * S, WARPS = THREADS / 32;
};
// Forward: 16 steps a thread, which halves what a round costs beside its elements (2048 x 64 x 1024, bf16: 197 -> 175 us against
// 8); the backward has no registers for more than 8.
typedef Tile<32, 4, 16> Forward;
typedef Tile<32, 8, 8> Backward;
// Few rows: 128 steps of 32 units, which makes twice as many CTAs (32768 x 1 x 1024: 87 us against 165 with 64 units and half the
// CTAs); a warp has two parts, one behind the other.
typedef Tile<16, 16, 8> Narrow;
static_assert(Forward::STEPS == Backward::STEPS, "states lie between tiles of both directions");

// ---- element access: PAIRS = two adjacent units per lane (aligned), else units `lane` and `lane + LANES`
template <typename T> struct Pair;
template <> struct Pair<float> { typedef float2 type; };
template <> struct Pair<__nv_bfloat16> { typedef __nv_bfloat162 type; };
template <> struct Pair<__half> { typedef __half2 type; };

__device__ __forceinline__ P2 unpack(float2 v) { return pair(v.x, v.y); }
__device__ __forceinline__ P2 unpack(__nv_bfloat162 v) {        // a bf16 is the upper half of an fp32
  const uint32_t w = *reinterpret_cast<const uint32_t*>(&v);
  return pair(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ P2 unpack(__half2 v) { return unpack(__half22float2(v)); }
template <typename T> __device__ __forceinline__ typename Pair<T>::type pack(float2 v);
template <> __device__ __forceinline__ float2 pack<float>(float2 v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat162 pack<__nv_bfloat16>(float2 v) { return __float22bfloat162_rn(v); }
template <> __device__ __forceinline__ __half2 pack<__half>(float2 v) { return __float22half2_rn(v); }

// The lane's two units of a row that starts at p (unit 0 of the CTA); `left`: units of the row from there on.
template <bool PAIRS, int LANES, typename T>
__device__ __forceinline__ P2 load_units(const T* p, int lane, int left) {
  if (PAIRS) return 2 * lane < left ? unpack(*reinterpret_cast<const typename Pair<T>::type*>(p + 2 * lane)) : both(0.f);
  return pair(lane < left ? to_float(p[lane]) : 0.f, lane + LANES < left ? to_float(p[lane + LANES]) : 0.f);
}
template <bool PAIRS, int LANES, typename T>
__device__ __forceinline__ void store_units(T* p, int lane, int left, P2 pv) {
  const float2 v = split(pv);
  if (PAIRS) {
    if (2 * lane < left) *reinterpret_cast<typename Pair<T>::type*>(p + 2 * lane) = pack<T>(v);
  } else {
    if (lane < left) p[lane] = from_float<T>(v.x);
    if (lane + LANES < left) p[lane + LANES] = from_float<T>(v.y);
  }
}

// fp32 states of the lane's units; rows of any alignment.
template <bool PAIRS, int LANES>
__device__ __forceinline__ P2 load_state(const float* p, int lane, int left) {
  const int i = PAIRS ? 2 * lane : lane, j = PAIRS ? 2 * lane + 1 : lane + LANES;
  return pair(i < left ? p[i] : 0.f, j < left ? p[j] : 0.f);
}
template <bool PAIRS, int LANES>
__device__ __forceinline__ void store_state(float* p, int lane, int left, P2 pv) {
  const float2 v = split(pv);
  const int i = PAIRS ? 2 * lane : lane, j = PAIRS ? 2 * lane + 1 : lane + LANES;
  if (i < left) p[i] = v.x;
  if (j < left) p[j] = v.y;
}

// A map of two units as it lies in shared memory: 16 bytes.
struct __align__(16) Map {
  P2 A, b;
};
// The map `m` after the map `first`.
__device__ __forceinline__ Map after(const Map& m, const Map& first) { return {mul2(m.A, first.A), fma2(m.A, first.b, m.b)}; }
__device__ __forceinline__ P2 apply(const Map& m, P2 h) { return fma2(m.A, h, m.b); }
__device__ __forceinline__ P2 from_other_half(P2 v) { return P2{__shfl_xor_sync(0xffffffffu, v.v, 16)}; }

// ---- cluster exchange ----------------------------------------------------------------------------
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t at_rank(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
// 16 bytes into a peer's shared memory, counted on a barrier of the peer.
__device__ __forceinline__ void send16(uint32_t dst, const Map& m, uint32_t bar) {
  asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v2.b64 [%0], {%1, %2}, [%3];"
               ::"r"(dst), "l"(m.A.v), "l"(m.b.v), "r"(bar) : "memory");
}

template <typename Cut>
struct Shared {
  Map part[2][Cut::WARPS][Cut::LANES];         // maps of the warps
  P2 carry[2][Cut::LANES];                     // what enters the round
  unsigned long long full[STAGES_MAX];       // a stage of inputs has landed
  unsigned long long joined[2];              // maps of all ranks have landed
  int dead;
};
// Behind the ring of inputs in dynamic shared memory: maps of the cluster's tiles, [2][ranks][LANES].
template <int LANES>
__host__ __device__ constexpr size_t peer_bytes(int ranks) { return ranks > 1 ? (size_t)2 * ranks * LANES * sizeof(Map) : 0; }

// Where a CTA is: its row, first unit, and its rank among the CTAs that share them.
struct Place {
  int b, unit, left, rank, ranks;
};
template <int UNITS>
__device__ __forceinline__ Place place_of(const Args& a, int ranks) {
  Place w;
  w.ranks = ranks;
  w.rank = ranks > 1 ? (int)cluster_rank() : 0;
  const int columns = (a.H + UNITS - 1) / UNITS;
  const unsigned i = blockIdx.x / (unsigned)ranks;
  w.b = (int)(i / (unsigned)columns);
  w.unit = (int)(i % (unsigned)columns) * UNITS;
  w.left = a.H - w.unit;
  return w;
}

template <typename Cut>
__device__ __forceinline__ void set_up(Shared<Cut>& s, int stages, int ranks) {
  constexpr int LANES = Cut::LANES;
  if (threadIdx.x == 0) {
    s.dead = 0;
    for (int i = 0; i < stages; ++i) tc::mbar_init(tc::smem_u32(&s.full[i]), 1);
    for (int i = 0; i < 2; ++i) tc::mbar_init(tc::smem_u32(&s.joined[i]), 1);
    tc::mbar_fence_init();
    if (ranks > 1)
      for (int i = 0; i < 2; ++i) tc::mbar_expect_tx(tc::smem_u32(&s.joined[i]), (uint32_t)(ranks * LANES * sizeof(Map)));
  }
  __syncthreads();
  if (ranks > 1) cluster_barrier();
}

// One part of the threads (all of a CTA's units) sends the CTA's map to every rank.  A slot is used again two rounds later: a
// peer sends its map of the round between only after all its threads have read this round's, so two slots are enough.
template <typename Cut>
__device__ __forceinline__ void send_map(Shared<Cut>& s, Map* peers, const Place& w, int round, Map all, int lane) {
  constexpr int LANES = Cut::LANES;
  const int slot = round & 1;
  const uint32_t to = tc::smem_u32(peers + (slot * w.ranks + w.rank) * LANES + lane), bar = tc::smem_u32(&s.joined[slot]);
  for (int r = 0; r < w.ranks; ++r) send16(at_rank(to, (uint32_t)r), all, at_rank(bar, (uint32_t)r));
}
// What enters this CTA's tile: the round's carry through the maps of the ranks before it.  Part 1 folds on through all of
// them, which is what the next round starts from.
template <typename Cut>
__device__ __forceinline__ P2 join(Shared<Cut>& s, const Map* peers, const Place& w, int round, int part, int lane) {
  constexpr int LANES = Cut::LANES;
  const int slot = round & 1;
  tc::mbar_wait(tc::smem_u32(&s.joined[slot]), (uint32_t)(round >> 1) & 1u, &s.dead, &g_gated_status);
  if (threadIdx.x == 0) tc::mbar_expect_tx(tc::smem_u32(&s.joined[slot]), (uint32_t)(w.ranks * LANES * sizeof(Map)));
  const Map* m = peers + slot * w.ranks * LANES + lane;
  P2 h = s.carry[slot][lane];
  for (int r = 0; r < w.rank; ++r) h = apply(m[r * LANES], h);
  if (part == 1) {
    P2 end = h;
    for (int r = w.rank; r < w.ranks; ++r) end = apply(m[r * LANES], end);
    s.carry[slot ^ 1][lane] = end;
  }
  return h;
}

// What enters this warp: h through the maps of the warps before it (v = 0 .. warp - 1, or the last .. warp + 1 where BACK).
template <bool BACK, int WARPS, int LANES>
__device__ __forceinline__ P2 through(const Map* m, int warp, P2 h) {
  Map all[WARPS];
#pragma unroll
  for (int v = 0; v < WARPS; ++v) all[v] = m[v * LANES];
#pragma unroll
  for (int i = 0; i < WARPS - 1; ++i) {
    const int v = BACK ? WARPS - 1 - i : i;
    if (BACK ? v > warp : v < warp) h = apply(all[v], h);
  }
  return h;
}

// How inputs come: as TMA tiles (rows on 16-byte boundaries); by asynchronous copies of two units, each thread its own; by
// such copies of single fp32 units; or, 16-bit units on odd boundaries, by loads of the threads.
enum { BY_TMA = 0, BY_PAIRS = 1, BY_UNITS = 2 };
template <int MODE> constexpr bool PAIRED = MODE != BY_UNITS;        // a lane has units 2 i and 2 i + 1, not i and i + LANES
template <int MODE, typename T> constexpr bool OWN_COPIES = MODE == BY_PAIRS || (MODE == BY_UNITS && sizeof(T) == 4);
template <int MODE, typename T> constexpr bool BY_LOADS = MODE == BY_UNITS && sizeof(T) != 4;

template <int BYTES, int TO, int FROM>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0 + %2], [%1 + %3], %4;" ::"r"(dst), "l"(src), "n"(TO), "n"(FROM), "n"(BYTES) : "memory");
}
// A thread's rows K .. SEG - 1 of its two units into its own places of a stage; behind the row's end (not ALL) the last step again.
template <bool ALL, int MODE, int SEG, int LANES, typename T, int K = 0>
__device__ __forceinline__ void copy_rows(uint32_t dst, const T* row, long long stride, int left_steps, bool first, bool second) {
  if constexpr (K < SEG) {
    constexpr int TO = K * 2 * LANES * (int)sizeof(T);
    if (MODE == BY_PAIRS) {
      if (first) copy_async<2 * sizeof(T), TO, 0>(dst, row);
    } else {
      if (first) copy_async<4, TO, 0>(dst, row);
      if (second) copy_async<4, TO + LANES * (int)sizeof(T), LANES * (int)sizeof(T)>(dst, row);
    }
    copy_rows<ALL, MODE, SEG, LANES, T, K + 1>(dst, row + (ALL || K + 1 < left_steps ? stride : 0), stride, left_steps, first, second);
  }
}
template <int MODE, int SEG, int LANES, typename T>
__device__ __forceinline__ void copy_own(T* st, const T* p, long long stride, int t0, int len, int lane, int left) {
  const int unit = MODE == BY_PAIRS ? 2 * lane : lane;
  const uint32_t dst = tc::smem_u32(st + unit);
  const T* row = p + (long long)min(t0, len - 1) * stride + unit;
  if (len - t0 >= SEG) copy_rows<true, MODE, SEG, LANES>(dst, row, stride, SEG, unit < left, lane + LANES < left);
  else copy_rows<false, MODE, SEG, LANES>(dst, row, stride, len - t0, unit < left, lane + LANES < left);
}
// A thread's rows of its two units by loads, all of them in flight at once.  Behind the row's end the last step again, beside its
// last unit that unit (such lanes store nothing): predicates kept the loads apart (286 x 33 x 915 bf16, backward: 59 us against
// 86; 43 at 912 units, where TMA brings them).
template <int SEG, int LANES, typename T, typename V>
__device__ __forceinline__ void load_rows(V (&v)[SEG], const T* p, long long stride, int t0, int len, int lane, int left) {
  const T* a = p + min(lane, left - 1);
  const int next = min(lane + LANES, left - 1) - min(lane, left - 1);
#pragma unroll
  for (int k = 0; k < SEG; ++k) {
    const T* row = a + (long long)min(t0 + k, len - 1) * stride;
    v[k].x = row[0];
    v[k].y = row[next];
  }
}
__device__ __forceinline__ void copies_sent() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void copies_landed_but_last() { asm volatile("cp.async.wait_group 1;" ::: "memory"); }

// Stage of the ring and the phase of its barrier, moved on once a round (a division of the round would cost as much as eight
// elements).
struct Ring {
  int stage, phase;
  __device__ __forceinline__ void next(int stages) {
    if (++stage == stages) { stage = 0; phase ^= 1; }
  }
};

// Nobody leaves while a peer may still write here; a CTA that gave up waits for what is in flight.
__device__ __forceinline__ void tear_down(const volatile int* dead, int ranks) {
  __syncwarp();                                            // the barrier is a whole warp's instruction
  if (ranks > 1) cluster_barrier();
  if (*dead) {
    const long long start = clock64();
    while (clock64() - start < (1ll << 18)) {
    }
  }
}

// ---- forward -------------------------------------------------------------------------------------
// A round's phases: gates and maps of the threads | barrier | the state that enters, the results.  CLUSTERED: the gates of the next
// round are computed while the maps of this one travel (two sets of registers); otherwise other CTAs of the SM cover for the
// barrier.
template <typename T, typename Cut, int MODE, bool TANH, bool CLUSTERED>
__global__ void __launch_bounds__(Cut::THREADS, 512 / Cut::THREADS)
gated_fwd_kernel(const __grid_constant__ CUtensorMap map, const Args a, int ranks, int stages) {
  constexpr int UNITS = Cut::UNITS, PARTS = Cut::PARTS, STEPS = Cut::STEPS, LANES = Cut::LANES, SEG = Cut::SEG, WARPS = Cut::WARPS;
  extern __shared__ __align__(128) unsigned char raw[];
  __shared__ Shared<Cut> s;
  T* ring = reinterpret_cast<T*>(raw);                        // [stages][x, c][STEPS][UNITS]
  Map* peers = reinterpret_cast<Map*>(raw + (size_t)stages * 2 * STEPS * UNITS * sizeof(T));
  const int part = threadIdx.x / LANES, lane = threadIdx.x % LANES, warp = tc::uniform_warp();
  const bool second = LANES == 16 && (threadIdx.x & 16) != 0;  // the later of the warp's two parts
  if (!CLUSTERED) ranks = 1;
  const Place w = place_of<UNITS>(a, ranks);
  const int len = row_length(a, w.b);
  const int tiles = (len + STEPS - 1) / STEPS;
  const int rounds = (tiles + ranks - 1) / ranks;
  set_up(s, stages, ranks);

  auto fetch = [&](int round, int stage) {                    // one thread
    const int tile = round * ranks + w.rank;
    if (round >= rounds || tile >= tiles) return;
    const uint32_t bar = tc::smem_u32(&s.full[stage]);
    T* dst = ring + (size_t)stage * 2 * STEPS * UNITS;
    tc::mbar_expect_tx(bar, 2 * STEPS * UNITS * sizeof(T));
    tc::tma_load_3d(tc::smem_u32(dst), &map, w.unit, w.b, tile * STEPS, bar);
    tc::tma_load_3d(tc::smem_u32(dst + STEPS * UNITS), &map, a.H + w.unit, w.b, tile * STEPS, bar);
  };
  if (MODE == BY_TMA && threadIdx.x == 0)
    for (int r = 0; r < stages; ++r) fetch(r, r);

  const T* gp = static_cast<const T*>(a.gi) + (long long)w.b * a.gi_b + w.unit;
  T* op = static_cast<T*>(a.out) + (long long)w.b * a.out_b + w.unit;
  if (part == 0) {
    P2 h = both(0.f);
    if (a.h0 != nullptr) h = load_state<PAIRED<MODE>, LANES>(a.h0 + (long long)w.b * a.h0_b + w.unit, lane, w.left);
    s.carry[0][lane] = h;
  }
  const Constants K = constants();

  Ring at = {0, 0};

  // a thread's own copies: the next round's are sent before this one's are waited for
  auto copy_round = [&](int round, int stage) {
    const int tile = round * ranks + w.rank;
    if (round < rounds && tile < tiles) {
      T* st = ring + (size_t)stage * 2 * STEPS * UNITS + part * SEG * UNITS;
      copy_own<MODE, SEG, LANES>(st, gp, a.gi_t, tile * STEPS + part * SEG, len, lane, w.left);
      copy_own<MODE, SEG, LANES>(st + STEPS * UNITS, gp + a.H, a.gi_t, tile * STEPS + part * SEG, len, lane, w.left);
    }
    copies_sent();
  };
  if (OWN_COPIES<MODE, T>) copy_round(0, 0);

  // gates of a round into z and u, the thread's map into shared memory
  auto open_gates = [&](int round, P2 (&z)[SEG], P2 (&u)[SEG], Map& first) {
    const int tile = round * ranks + w.rank;
    const int t0 = tile * STEPS + part * SEG;
    const int n = len - t0;                                   // steps left from here
    P2 A = both(1.f), b = both(0.f);
    if (OWN_COPIES<MODE, T>) copy_round(round + 1, at.stage ^ 1);
    if (tile < tiles) {
      if (MODE == BY_TMA) tc::mbar_wait(tc::smem_u32(&s.full[at.stage]), (uint32_t)at.phase, &s.dead, &g_gated_status);
      if (OWN_COPIES<MODE, T>) copies_landed_but_last();
      const T* st = ring + (size_t)at.stage * 2 * STEPS * UNITS + part * SEG * UNITS;
      typename Pair<T>::type rx[SEG], rc[SEG];
      if (BY_LOADS<MODE, T>) {
        load_rows<SEG, LANES>(rx, gp, a.gi_t, t0, len, lane, w.left);
        load_rows<SEG, LANES>(rc, gp + a.H, a.gi_t, t0, len, lane, w.left);
      }
#pragma unroll
      for (int k = 0; k < SEG; ++k) {
        P2 x = both(0.f), c = x;
        if (MODE == BY_TMA || OWN_COPIES<MODE, T>) {
          x = load_units<PAIRED<MODE>, LANES>(st + k * UNITS, lane, UNITS);
          c = load_units<PAIRED<MODE>, LANES>(st + (STEPS + k) * UNITS, lane, UNITS);
        } else {
          x = unpack(rx[k]);
          c = unpack(rc[k]);
        }
        const Gates g = gates<TANH, false>(x, c, K);
        z[k] = g.z;
        u[k] = mul2(g.keep, g.n);
      }
      if (n < SEG) {                                          // behind the row's end: the state stays
#pragma unroll
        for (int k = 0; k < SEG; ++k)
          if (k >= n) { z[k] = both(1.f); u[k] = both(0.f); }
      }
      A = z[0];
      b = u[0];
#pragma unroll
      for (int k = 1; k < SEG; ++k) {
        A = mul2(z[k], A);
        b = fma2(z[k], b, u[k]);
      }
    }
    first = Map{A, b};
    if (LANES == 16) {                                        // `first`: the earlier part's map, in both
      const Map other = {from_other_half(A), from_other_half(b)};
      const Map later = second ? first : other;
      if (second) first = other;
      A = mul2(later.A, first.A);
      b = fma2(later.A, first.b, later.b);
    }
    if (!second) s.part[round & 1][warp][lane] = Map{A, b};
  };
  // results of a round from the state that enters its tile
  auto walk = [&](int round, P2 h, const P2 (&z)[SEG], const P2 (&u)[SEG], const Map& first) {
    const int tile = round * ranks + w.rank;
    if (tile >= tiles) return;
    if (a.states != nullptr && part == 0)
      store_state<PAIRED<MODE>, LANES>(a.states + ((long long)tile * a.B + w.b) * a.H + w.unit, lane, w.left, h);
    h = through<false, WARPS, LANES>(&s.part[round & 1][0][lane], warp, h);
    if (second) h = apply(first, h);
    const int t0 = tile * STEPS + part * SEG, n = len - t0;
    char* o = reinterpret_cast<char*>(op + (long long)t0 * a.out_t);
    if (n >= SEG) {
#pragma unroll
      for (int k = 0; k < SEG; ++k) {
        h = fma2(z[k], h, u[k]);
        store_units<PAIRED<MODE>, LANES>(reinterpret_cast<T*>(o), lane, w.left, h);
        o += a.out_step;
      }
    } else {
#pragma unroll
      for (int k = 0; k < SEG; ++k) {
        h = fma2(z[k], h, u[k]);
        if (k < n) store_units<PAIRED<MODE>, LANES>(reinterpret_cast<T*>(o), lane, w.left, h);
        o += a.out_step;
      }
    }
    if (!CLUSTERED && part == PARTS - 1) s.carry[(round & 1) ^ 1][lane] = h;
  };

  auto send = [&](int round) {                                // part 0: the CTA's map to every rank
    Map all = s.part[round & 1][0][lane];
#pragma unroll
    for (int v = 1; v < WARPS; ++v) all = after(s.part[round & 1][v][lane], all);
    send_map(s, peers, w, round, all, lane);
  };
  if (CLUSTERED) {
    auto round_of = [&](int round, const P2 (&z)[SEG], const P2 (&u)[SEG], const Map& m, P2 (&zn)[SEG], P2 (&un)[SEG], Map& mn) {
      __syncthreads();                                        // the stage is read, the threads' maps are there
      if (part == 0) send(round);
      if (MODE == BY_TMA && threadIdx.x == 0) fetch(round + stages, at.stage);
      at.next(stages);
      if (round + 1 < rounds) open_gates(round + 1, zn, un, mn);
      walk(round, join(s, peers, w, round, part, lane), z, u, m);
    };
    P2 za[SEG], ua[SEG], zb[SEG], ub[SEG];
    Map ma, mb;
    if (rounds > 0) open_gates(0, za, ua, ma);
    for (int round = 0; round < rounds; round += 2) {
      round_of(round, za, ua, ma, zb, ub, mb);
      if (round + 1 < rounds) round_of(round + 1, zb, ub, mb, za, ua, ma);
    }
  } else {
    for (int round = 0; round < rounds; ++round) {
      P2 z[SEG], u[SEG];
      Map first;
      open_gates(round, z, u, first);
      __syncthreads();
      if (MODE == BY_TMA && threadIdx.x == 0) fetch(round + stages, at.stage);
      at.next(stages);
      walk(round, s.carry[round & 1][lane], z, u, first);
    }
  }

  // steps behind the row's last, and the state after it
  for (int t = len + w.rank * PARTS + part; t < a.T; t += ranks * PARTS)
    store_units<PAIRED<MODE>, LANES>(op + (long long)t * a.out_t, lane, w.left, both(0.f));
  __syncthreads();
  if (w.rank == 0 && part == 0)
    store_state<PAIRED<MODE>, LANES>(a.h_T + (long long)w.b * a.H + w.unit, lane, w.left, s.carry[rounds & 1][lane]);
  tear_down(&s.dead, ranks);
}

// ---- backward ------------------------------------------------------------------------------------
// Tiles from the last to the first; rank 0 of a round has the latest.  `front` joins the states inside a tile forwards, `part`
// the gradients backwards, both with the same products of z.
template <typename T, typename Cut, int MODE, bool TANH, bool CLUSTERED>
__global__ void __launch_bounds__(Cut::THREADS, 2)
gated_bwd_kernel(const __grid_constant__ CUtensorMap map, const __grid_constant__ CUtensorMap dmap, const Args a, int ranks,
                 int stages) {
  constexpr int UNITS = Cut::UNITS, PARTS = Cut::PARTS, STEPS = Cut::STEPS, LANES = Cut::LANES, SEG = Cut::SEG, WARPS = Cut::WARPS;
  extern __shared__ __align__(128) unsigned char raw[];
  __shared__ Shared<Cut> s;
  __shared__ P2 front[2][WARPS][LANES];
  T* ring = reinterpret_cast<T*>(raw);                        // [stages][x, c, dout][STEPS][UNITS]
  Map* peers = reinterpret_cast<Map*>(raw + (size_t)stages * 3 * STEPS * UNITS * sizeof(T));
  const int part = threadIdx.x / LANES, lane = threadIdx.x % LANES, warp = tc::uniform_warp();
  const bool second = LANES == 16 && (threadIdx.x & 16) != 0;  // the later of the warp's two parts
  if (!CLUSTERED) ranks = 1;
  const Place w = place_of<UNITS>(a, ranks);
  const int len = row_length(a, w.b);
  const int tiles = (len + STEPS - 1) / STEPS;
  const int rounds = (tiles + ranks - 1) / ranks;
  const bool with_dout = a.dout != nullptr;
  set_up(s, stages, ranks);

  auto fetch = [&](int round, int stage) {                    // one thread
    const int tile = tiles - 1 - (round * ranks + w.rank);
    if (round >= rounds || tile < 0) return;
    const uint32_t bar = tc::smem_u32(&s.full[stage]);
    T* dst = ring + (size_t)stage * 3 * STEPS * UNITS;
    tc::mbar_expect_tx(bar, (with_dout ? 3 : 2) * STEPS * UNITS * sizeof(T));
    tc::tma_load_3d(tc::smem_u32(dst), &map, w.unit, w.b, tile * STEPS, bar);
    tc::tma_load_3d(tc::smem_u32(dst + STEPS * UNITS), &map, a.H + w.unit, w.b, tile * STEPS, bar);
    if (with_dout) tc::tma_load_3d(tc::smem_u32(dst + 2 * STEPS * UNITS), &dmap, w.unit, w.b, tile * STEPS, bar);
  };
  if (MODE == BY_TMA && threadIdx.x == 0)
    for (int r = 0; r < stages; ++r) fetch(r, r);

  const T* gp = static_cast<const T*>(a.gi) + (long long)w.b * a.gi_b + w.unit;
  const T* dp = with_dout ? static_cast<const T*>(a.dout) + (long long)w.b * a.dout_b + w.unit : nullptr;
  T* qp = static_cast<T*>(a.dgi) + (long long)w.b * a.dgi_b + w.unit;
  if (part == 0) {
    P2 G = both(0.f);
    if (a.dh_T != nullptr) G = load_state<PAIRED<MODE>, LANES>(a.dh_T + (long long)w.b * a.dh_b + w.unit, lane, w.left);
    s.carry[0][lane] = G;
  }
  const Constants K = constants();

  Ring at = {0, 0};
  auto copy_round = [&](int round, int stage) {
    const int tile = tiles - 1 - (round * ranks + w.rank);
    if (round < rounds && tile >= 0) {
      T* st = ring + (size_t)stage * 3 * STEPS * UNITS + part * SEG * UNITS;
      const int t0 = tile * STEPS + part * SEG;
      copy_own<MODE, SEG, LANES>(st, gp, a.gi_t, t0, len, lane, w.left);
      copy_own<MODE, SEG, LANES>(st + STEPS * UNITS, gp + a.H, a.gi_t, t0, len, lane, w.left);
      if (with_dout) copy_own<MODE, SEG, LANES>(st + 2 * STEPS * UNITS, dp, a.dout_t, t0, len, lane, w.left);
    }
    copies_sent();
  };
  if (OWN_COPIES<MODE, T>) copy_round(0, 0);
  for (int round = 0; round < rounds; ++round) {
    if (OWN_COPIES<MODE, T>) copy_round(round + 1, at.stage ^ 1);
    const int tile = tiles - 1 - (round * ranks + w.rank);
    const int t0 = tile * STEPS + part * SEG;
    const int n = len - t0;                                   // steps left from here
    P2 h = both(0.f);
    // p: candidate, then (h_{t-1} - n) z (1 - z);  q: (1 - z) n'.  Five values a step: a sixth, z (1 - z), would save a
    // multiplication and cost 16 registers (501 x 19 x 607, fp32: 51 us against 48).
    P2 z[SEG], keep[SEG], p[SEG], q[SEG], d[SEG];
    P2 A = both(1.f), f = both(0.f), r = f;
    if (tile >= 0) {
      h = load_state<PAIRED<MODE>, LANES>(a.states + ((long long)tile * a.B + w.b) * a.H + w.unit, lane, w.left);
      if (MODE == BY_TMA) tc::mbar_wait(tc::smem_u32(&s.full[at.stage]), (uint32_t)at.phase, &s.dead, &g_gated_status);
      if (OWN_COPIES<MODE, T>) copies_landed_but_last();
      const T* st = ring + (size_t)at.stage * 3 * STEPS * UNITS + part * SEG * UNITS;
      typename Pair<T>::type rx[SEG], rc[SEG], rd[SEG];
      if (BY_LOADS<MODE, T>) {
        load_rows<SEG, LANES>(rx, gp, a.gi_t, t0, len, lane, w.left);
        load_rows<SEG, LANES>(rc, gp + a.H, a.gi_t, t0, len, lane, w.left);
        if (with_dout) load_rows<SEG, LANES>(rd, dp, a.dout_t, t0, len, lane, w.left);
      }
#pragma unroll
      for (int k = 0; k < SEG; ++k) {
        P2 x = both(0.f), c = x;
        d[k] = x;
        if (MODE == BY_TMA || OWN_COPIES<MODE, T>) {
          x = load_units<PAIRED<MODE>, LANES>(st + k * UNITS, lane, UNITS);
          c = load_units<PAIRED<MODE>, LANES>(st + (STEPS + k) * UNITS, lane, UNITS);
          if (with_dout) d[k] = load_units<PAIRED<MODE>, LANES>(st + (2 * STEPS + k) * UNITS, lane, UNITS);
        } else {
          x = unpack(rx[k]);
          c = unpack(rc[k]);
          if (with_dout) d[k] = unpack(rd[k]);
        }
        const Gates g = gates<TANH, true>(x, c, K);
        z[k] = g.z;
        keep[k] = g.keep;
        p[k] = g.n;
        q[k] = mul2(g.keep, g.slope);
      }
      if (n < SEG) {
#pragma unroll
        for (int k = 0; k < SEG; ++k)
          if (k >= n) {
            z[k] = both(1.f);
            keep[k] = p[k] = d[k] = both(0.f);
          }
      }
#pragma unroll
      for (int k = 0; k < SEG; ++k) {
        A = mul2(z[k], A);
        f = fma2(z[k], f, mul2(keep[k], p[k]));
      }
#pragma unroll
      for (int k = SEG - 1; k >= 0; --k) r = mul2(z[k], add2(d[k], r));
    }
    const int slot = round & 1;
    Map back = {A, r};                                        // gradients: from the later part to the earlier one
    P2 A0 = A, f0 = f;                                        // states: the earlier part's
    if (LANES == 16) {
      const P2 oA = from_other_half(A), orr = from_other_half(r), of = from_other_half(f);
      const Map early = second ? Map{oA, orr} : back, late = second ? back : Map{oA, orr};
      A0 = early.A;
      f0 = second ? of : f;
      const P2 f1 = second ? f : of;
      back = late;                                            // for the earlier part
      if (!second) {
        s.part[slot][warp][lane] = after(early, late);
        front[slot][warp][lane] = fma2(late.A, f0, f1);
      }
    } else {
      s.part[slot][warp][lane] = back;
      front[slot][warp][lane] = f;
    }
    __syncthreads();
    const Map* m = &s.part[slot][0][lane];
    if (CLUSTERED && part == 0) {
      Map all = m[(WARPS - 1) * LANES];
#pragma unroll
      for (int v = WARPS - 2; v >= 0; --v) all = after(m[v * LANES], all);
      send_map(s, peers, w, round, all, lane);
    }
    if (MODE == BY_TMA && threadIdx.x == 0) fetch(round + stages, at.stage);
    at.next(stages);
    for (int v = 0; v < warp; ++v) h = fma2(m[v * LANES].A, h, front[slot][v][lane]);
    if (second) h = fma2(A0, h, f0);
    if (tile >= 0) {
#pragma unroll
      for (int k = 0; k < SEG; ++k) {
        const P2 n = p[k];
        p[k] = mul2(sub2(h, n), mul2(z[k], keep[k]));
        h = fma2(z[k], h, mul2(keep[k], n));
      }
    }
    P2 G = CLUSTERED ? join(s, peers, w, round, part, lane) : s.carry[slot][lane];
    if (tile >= 0) {
      G = through<true, WARPS, LANES>(m, warp, G);
      if (LANES == 16 && !second) G = apply(back, G);
      char* o = reinterpret_cast<char*>(qp + (long long)(t0 + SEG - 1) * a.dgi_t);
#pragma unroll
      for (int k = SEG - 1; k >= 0; --k) {
        const P2 g = add2(G, d[k]);
        G = mul2(z[k], g);
        if (k < n) {
          store_units<PAIRED<MODE>, LANES>(reinterpret_cast<T*>(o), lane, w.left, mul2(g, p[k]));
          store_units<PAIRED<MODE>, LANES>(reinterpret_cast<T*>(o + a.half), lane, w.left, mul2(g, q[k]));
        }
        o -= a.dgi_step;
      }
      if (!CLUSTERED && part == 0) s.carry[slot ^ 1][lane] = G;
    }
  }

  for (int t = len + w.rank * PARTS + part; t < a.T; t += ranks * PARTS) {
    store_units<PAIRED<MODE>, LANES>(qp + (long long)t * a.dgi_t, lane, w.left, both(0.f));
    store_units<PAIRED<MODE>, LANES>(qp + (long long)t * a.dgi_t + a.H, lane, w.left, both(0.f));
  }
  __syncthreads();
  if (a.dh0 != nullptr && w.rank == 0 && part == 0)
    store_state<PAIRED<MODE>, LANES>(a.dh0 + (long long)w.b * a.H + w.unit, lane, w.left, s.carry[rounds & 1][lane]);
  tear_down(&s.dead, ranks);
}

// ---- a few steps -----------------------------------------------------------------------------------
constexpr int SHORT = 8;

// At most SHORT steps: a warp has 64 units of a row and all their steps, nothing to join.
template <typename T, bool PAIRS, bool TANH>
__global__ void __launch_bounds__(128) gated_short_fwd_kernel(const Args a) {
  const int lane = threadIdx.x & 31, columns = (a.H + 63) / 64;
  const long long i = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (i >= (long long)a.B * columns) return;
  const int b = (int)(i / columns), unit = (int)(i % columns) * 64, left = a.H - unit;
  const int len = row_length(a, b);
  const T* gp = static_cast<const T*>(a.gi) + (long long)b * a.gi_b + unit;
  T* op = static_cast<T*>(a.out) + (long long)b * a.out_b + unit;
  P2 h = both(0.f);
  if (a.h0 != nullptr) h = load_state<PAIRS, 32>(a.h0 + (long long)b * a.h0_b + unit, lane, left);
  if (a.states != nullptr) store_state<PAIRS, 32>(a.states + (long long)b * a.H + unit, lane, left, h);
  const Constants K = constants();
  P2 x[SHORT], c[SHORT];
#pragma unroll
  for (int k = 0; k < SHORT; ++k)
    if (k < len) {
      x[k] = load_units<PAIRS, 32>(gp + (long long)k * a.gi_t, lane, left);
      c[k] = load_units<PAIRS, 32>(gp + (long long)k * a.gi_t + a.H, lane, left);
    }
#pragma unroll
  for (int k = 0; k < SHORT; ++k)
    if (k < a.T) {
      P2 o = both(0.f);
      if (k < len) {
        const Gates g = gates<TANH, false>(x[k], c[k], K);
        h = fma2(g.z, h, mul2(g.keep, g.n));
        o = h;
      }
      store_units<PAIRS, 32>(op + (long long)k * a.out_t, lane, left, o);
    }
  store_state<PAIRS, 32>(a.h_T + (long long)b * a.H + unit, lane, left, h);
}

template <typename T, bool PAIRS, bool TANH>
__global__ void __launch_bounds__(128) gated_short_bwd_kernel(const Args a) {
  const int lane = threadIdx.x & 31, columns = (a.H + 63) / 64;
  const long long i = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (i >= (long long)a.B * columns) return;
  const int b = (int)(i / columns), unit = (int)(i % columns) * 64, left = a.H - unit;
  const int len = row_length(a, b);
  const T* gp = static_cast<const T*>(a.gi) + (long long)b * a.gi_b + unit;
  const T* dp = a.dout != nullptr ? static_cast<const T*>(a.dout) + (long long)b * a.dout_b + unit : nullptr;
  T* qp = static_cast<T*>(a.dgi) + (long long)b * a.dgi_b + unit;
  P2 G = both(0.f);
  if (a.dh_T != nullptr) G = load_state<PAIRS, 32>(a.dh_T + (long long)b * a.dh_b + unit, lane, left);
  P2 h = load_state<PAIRS, 32>(a.states + (long long)b * a.H + unit, lane, left);
  const Constants K = constants();
  P2 z[SHORT], p[SHORT], q[SHORT], d[SHORT];
#pragma unroll
  for (int k = 0; k < SHORT; ++k) {
    d[k] = both(0.f);
    if (k < len) {
      const P2 x = load_units<PAIRS, 32>(gp + (long long)k * a.gi_t, lane, left);
      const P2 c = load_units<PAIRS, 32>(gp + (long long)k * a.gi_t + a.H, lane, left);
      if (dp != nullptr) d[k] = load_units<PAIRS, 32>(dp + (long long)k * a.dout_t, lane, left);
      const Gates g = gates<TANH, true>(x, c, K);
      z[k] = g.z;
      p[k] = mul2(sub2(h, g.n), mul2(g.z, g.keep));
      q[k] = mul2(g.keep, g.slope);
      h = fma2(g.z, h, mul2(g.keep, g.n));
    }
  }
#pragma unroll
  for (int k = SHORT - 1; k >= 0; --k)
    if (k < a.T) {
      P2 dx = both(0.f), dc = dx;
      if (k < len) {
        const P2 g = add2(G, d[k]);
        G = mul2(z[k], g);
        dx = mul2(g, p[k]);
        dc = mul2(g, q[k]);
      }
      store_units<PAIRS, 32>(qp + (long long)k * a.dgi_t, lane, left, dx);
      store_units<PAIRS, 32>(qp + (long long)k * a.dgi_t + a.H, lane, left, dc);
    }
  if (a.dh0 != nullptr) store_state<PAIRS, 32>(a.dh0 + (long long)b * a.H + unit, lane, left, G);
}

template <typename T, bool PAIRS, bool TANH>
__global__ void __launch_bounds__(128) gated_step_kernel(const StepArgs a) {
  const int lane = threadIdx.x & 31, columns = (a.H + 63) / 64;
  const long long i = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (i >= (long long)a.B * columns) return;
  const int b = (int)(i / columns), unit = (int)(i % columns) * 64, left = a.H - unit;
  const T* gp = static_cast<const T*>(a.gi) + (long long)b * a.gi_b + unit;
  const P2 x = load_units<PAIRS, 32>(gp, lane, left), c = load_units<PAIRS, 32>(gp + a.H, lane, left);
  P2 h = load_state<PAIRS, 32>(a.h + (long long)b * a.h_b + unit, lane, left);
  const Gates g = gates<TANH, false>(x, c, constants());
  h = fma2(g.z, h, mul2(g.keep, g.n));
  store_state<PAIRS, 32>(a.h_new + (long long)b * a.hn_b + unit, lane, left, h);
  store_units<PAIRS, 32>(static_cast<T*>(a.out) + (long long)b * a.H + unit, lane, left, h);
}

// ---- host ------------------------------------------------------------------------------------------
template <typename T> struct MapType;
template <> struct MapType<float> { static constexpr CUtensorMapDataType value = CU_TENSOR_MAP_DATA_TYPE_FLOAT32; };
template <> struct MapType<__nv_bfloat16> { static constexpr CUtensorMapDataType value = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16; };
template <> struct MapType<__half> { static constexpr CUtensorMapDataType value = CU_TENSOR_MAP_DATA_TYPE_FLOAT16; };

// Whether rows of `units` elements can be fetched as tiles: everything on 16-byte boundaries, no stride 0.
template <typename T>
bool tileable(const void* p, long long st, long long sb, int B) {
  return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && st > 0 && (st * sizeof(T)) % 16 == 0 &&
         (B == 1 || (sb > 0 && (sb * sizeof(T)) % 16 == 0));
}
template <typename T>
bool paired(const void* p, long long st, long long sb) {
  return (reinterpret_cast<uintptr_t>(p) & (2 * sizeof(T) - 1)) == 0 && st % 2 == 0 && sb % 2 == 0;
}
template <typename T, typename Cut>
int tile_map(CUtensorMap* map, const void* p, long long units, const Args& a, long long st, long long sb) {
  const unsigned long long row = a.B == 1 ? 16 : (unsigned long long)sb * sizeof(T);
  return tc::make_tensor_map_rows(map, MapType<T>::value, p, units, a.B, a.T, row, (unsigned long long)st * sizeof(T),
                                  Cut::UNITS, Cut::STEPS);
}

// Few rows: less than 256 CTAs of 64 units.  Measured on both sides (forward / backward, us): 128 CTAs of 64 units over 3000 steps
// 78 / 102, as 256 narrow ones 51 / 82; 160 over 600 steps 27 / 37 and 23 / 35; 256 over 400 steps 23 / 29 and 25 / 35.
bool narrow(int T, int B, int H) { return T > Forward::STEPS && (long long)B * cdiv(H, Forward::UNITS) < 256; }

// CTAs of a row's units: a cluster of them where that makes at most 256 CTAs, up to the row's tiles.  An exchange costs about
// what a tile does, so more pay only where SMs have nothing else (64 narrow CTAs over 2000 steps: 27 / 41 us alone, 18 / 25 in
// clusters of 4, 23 / 29 of 8).  Clusters above 8 find room only while there are few of them: 16 columns over 20000 steps 54 / 82 us
// with 8, 41 / 63 with 12, 53 / 74 with 16; 8 columns 41 / 61, 39 / 59, 33 / 47; 32 columns over 32768 steps 84 / 133 with 8,
// 115 / 176 with 12.  A device that cannot place such a cluster gets 8 (states lie by tiles, so the two directions may differ).
int ranks_for(const Args& a) {
  if (!narrow(a.T, a.B, a.H)) return 1;
  const long long base = (long long)a.B * cdiv(a.H, Narrow::UNITS);
  const int tiles = cdiv(a.T, Narrow::STEPS);
  int ranks = 1;
  while (ranks < 8 && base * ranks * 2 <= 256) ranks *= 2;
  if (base <= 16) ranks = base <= 8 ? 16 : 12;
  return ranks < tiles ? ranks : tiles;
}

// The largest cluster that a test lets the device place; 0: what it can.
bool too_large_for_test(int ranks) {
  const int most = test_kernel_choice(4);
  return most > 0 && ranks > most;
}

// Whether the device can place a cluster of `ranks` CTAs; above eight that depends on its SMs and on what a CTA holds.  Asked once
// for each kernel and size.
bool placeable(const void* fn, int threads, int ranks, size_t smem) {
  static std::mutex mu;
  static std::map<std::tuple<int, const void*, int, size_t>, bool> cache;
  if (too_large_for_test(ranks)) return false;
  int dev = -1;
  if (cudaGetDevice(&dev) != cudaSuccess) return false;
  std::lock_guard<std::mutex> lk(mu);
  const auto key = std::make_tuple(dev, fn, ranks, smem);
  const auto it = cache.find(key);
  if (it != cache.end()) return it->second;
  int n = 0;
  if (allow_dynamic_smem(fn, smem) == B200GRU_OK &&
      cudaFuncSetAttribute(fn, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)ranks); cfg.blockDim = dim3((unsigned)threads); cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)ranks; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
    cfg.attrs = at; cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, fn, &cfg) != cudaSuccess) { cudaGetLastError(); n = 0; }
  } else {
    cudaGetLastError();
  }
  cache[key] = n > 0;
  return n > 0;
}

template <typename... KArgs, typename... CArgs>
int launch_tiles(void (*kernel)(KArgs...), long long blocks, int threads, int ranks, size_t smem, cudaStream_t st, CArgs... args) {
  const void* fn = reinterpret_cast<const void*>(kernel);
  if (allow_dynamic_smem(fn, smem) != B200GRU_OK || too_large_for_test(ranks)) return B200GRU_UNSUPPORTED;
  if (ranks > 8 && cudaFuncSetAttribute(fn, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess)
    return check_launch("cudaFuncSetAttribute(gated scan)");
  if (blocks > 0x7fffffffll) return B200GRU_UNSUPPORTED;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks); cfg.blockDim = dim3((unsigned)threads); cfg.dynamicSmemBytes = smem; cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)ranks; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
  cfg.attrs = at; cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, kernel, args...);
  note_launch();
  return check_launch("gated scan");
}

// Stages of `stage` bytes that fit beside the rest where `ctas` CTAs share an SM's 227 KB.
int stages_for(size_t stage, size_t fixed, int ctas) {
  const size_t room = 227 * 1024 / ctas - 1024 - fixed;
  const int n = (int)(room / stage);
  return n < 1 ? 1 : (n > STAGES_MAX ? STAGES_MAX : n);
}

template <typename T, typename Cut, int MODE, bool TANH>
int forward_cut(const Args& a, const CUtensorMap& map, int ranks, int stages, cudaStream_t st) {
  const long long blocks = (long long)a.B * cdiv(a.H, Cut::UNITS);
  const size_t ring = (size_t)stages * 2 * Cut::STEPS * Cut::UNITS * sizeof(T);
  if constexpr (std::is_same<Cut, Narrow>::value) {
    auto kernel = gated_fwd_kernel<T, Cut, MODE, TANH, true>;
    if (ranks > 8 && !placeable(reinterpret_cast<const void*>(kernel), Cut::THREADS, ranks, ring + peer_bytes<Cut::LANES>(ranks))) ranks = 8;
    if (ranks > 1) return launch_tiles(kernel, blocks * ranks, Cut::THREADS, ranks, ring + peer_bytes<Cut::LANES>(ranks), st, map, a, ranks, stages);
  }
  return launch_tiles(gated_fwd_kernel<T, Cut, MODE, TANH, false>, blocks, Cut::THREADS, 1, ring, st, map, a, 1, stages);
}
template <typename T, typename Cut, bool TANH>
int forward_tiles(const Args& a, cudaStream_t st) {
  const int ranks = ranks_for(a);
  alignas(64) CUtensorMap map;
  memset(&map, 0, sizeof(map));
  if (paired<T>(a.out, a.out_t, a.out_b) && a.H * sizeof(T) % 16 == 0 && tileable<T>(a.gi, a.gi_t, a.gi_b, a.B) &&
      tile_map<T, Cut>(&map, a.gi, 2ll * a.H, a, a.gi_t, a.gi_b) == B200GRU_OK) {
    const size_t stage = (size_t)2 * Cut::STEPS * Cut::UNITS * sizeof(T);
    const int stages = stages_for(stage, sizeof(Shared<Cut>) + peer_bytes<Cut::LANES>(ranks), 512 / Cut::THREADS);
    return forward_cut<T, Cut, BY_TMA, TANH>(a, map, ranks, stages, st);
  }
  if (a.H % 2 == 0 && paired<T>(a.out, a.out_t, a.out_b) && paired<T>(a.gi, a.gi_t, a.gi_b))
    return forward_cut<T, Cut, BY_PAIRS, TANH>(a, map, ranks, 2, st);
  return forward_cut<T, Cut, BY_UNITS, TANH>(a, map, ranks, sizeof(T) == 4 ? 2 : 0, st);
}

template <typename T, typename Cut, int MODE, bool TANH>
int backward_cut(const Args& a, const CUtensorMap& map, const CUtensorMap& dmap, int ranks, int stages, cudaStream_t st) {
  const long long blocks = (long long)a.B * cdiv(a.H, Cut::UNITS);
  const size_t ring = (size_t)stages * 3 * Cut::STEPS * Cut::UNITS * sizeof(T);
  if constexpr (std::is_same<Cut, Narrow>::value) {
    auto kernel = gated_bwd_kernel<T, Cut, MODE, TANH, true>;
    if (ranks > 8 && !placeable(reinterpret_cast<const void*>(kernel), Cut::THREADS, ranks, ring + peer_bytes<Cut::LANES>(ranks))) ranks = 8;
    if (ranks > 1) return launch_tiles(kernel, blocks * ranks, Cut::THREADS, ranks, ring + peer_bytes<Cut::LANES>(ranks), st, map, dmap, a, ranks, stages);
  }
  return launch_tiles(gated_bwd_kernel<T, Cut, MODE, TANH, false>, blocks, Cut::THREADS, 1, ring, st, map, dmap, a, 1, stages);
}
template <typename T, typename Cut, bool TANH>
int backward_tiles(const Args& a, cudaStream_t st) {
  const int ranks = ranks_for(a);
  alignas(64) CUtensorMap map, dmap;
  memset(&map, 0, sizeof(map));
  memset(&dmap, 0, sizeof(dmap));
  if (paired<T>(a.dgi, a.dgi_t, a.dgi_b) && a.H * sizeof(T) % 16 == 0 && tileable<T>(a.gi, a.gi_t, a.gi_b, a.B) &&
      tile_map<T, Cut>(&map, a.gi, 2ll * a.H, a, a.gi_t, a.gi_b) == B200GRU_OK &&
      (a.dout == nullptr || (tileable<T>(a.dout, a.dout_t, a.dout_b, a.B) &&
                             tile_map<T, Cut>(&dmap, a.dout, a.H, a, a.dout_t, a.dout_b) == B200GRU_OK))) {
    const size_t stage = (size_t)3 * Cut::STEPS * Cut::UNITS * sizeof(T);
    const int stages = stages_for(stage, sizeof(Shared<Cut>) + 2 * Cut::THREADS * sizeof(P2) + peer_bytes<Cut::LANES>(ranks), 2);
    return backward_cut<T, Cut, BY_TMA, TANH>(a, map, dmap, ranks, stages, st);
  }
  if (a.H % 2 == 0 && paired<T>(a.dgi, a.dgi_t, a.dgi_b) && paired<T>(a.gi, a.gi_t, a.gi_b) &&
      (a.dout == nullptr || paired<T>(a.dout, a.dout_t, a.dout_b)))
    return backward_cut<T, Cut, BY_PAIRS, TANH>(a, map, dmap, ranks, 2, st);
  return backward_cut<T, Cut, BY_UNITS, TANH>(a, map, dmap, ranks, sizeof(T) == 4 ? 2 : 0, st);
}

template <typename T, bool TANH>
int forward(const Args& a, cudaStream_t st) {
  if (a.T > SHORT) return narrow(a.T, a.B, a.H) ? forward_tiles<T, Narrow, TANH>(a, st) : forward_tiles<T, Forward, TANH>(a, st);
  const unsigned blocks = (unsigned)(((long long)a.B * cdiv(a.H, 64) + 3) / 4);
  if (a.H % 2 == 0 && paired<T>(a.out, a.out_t, a.out_b) && paired<T>(a.gi, a.gi_t, a.gi_b))
    gated_short_fwd_kernel<T, true, TANH><<<blocks, 128, 0, st>>>(a);
  else
    gated_short_fwd_kernel<T, false, TANH><<<blocks, 128, 0, st>>>(a);
  note_launch();
  return check_launch("gated_short_fwd_kernel");
}

template <typename T, bool TANH>
int backward(const Args& a, cudaStream_t st) {
  if (a.T > SHORT) return narrow(a.T, a.B, a.H) ? backward_tiles<T, Narrow, TANH>(a, st) : backward_tiles<T, Backward, TANH>(a, st);
  const unsigned blocks = (unsigned)(((long long)a.B * cdiv(a.H, 64) + 3) / 4);
  if (a.H % 2 == 0 && paired<T>(a.dgi, a.dgi_t, a.dgi_b) && paired<T>(a.gi, a.gi_t, a.gi_b) &&
      (a.dout == nullptr || paired<T>(a.dout, a.dout_t, a.dout_b)))
    gated_short_bwd_kernel<T, true, TANH><<<blocks, 128, 0, st>>>(a);
  else
    gated_short_bwd_kernel<T, false, TANH><<<blocks, 128, 0, st>>>(a);
  note_launch();
  return check_launch("gated_short_bwd_kernel");
}

template <typename T, bool TANH>
int step(const StepArgs& a, cudaStream_t st) {
  const unsigned blocks = (unsigned)(((long long)a.B * cdiv(a.H, 64) + 3) / 4);
  if (a.H % 2 == 0 && paired<T>(a.gi, 0, a.gi_b) && paired<T>(a.out, 0, 0)) gated_step_kernel<T, true, TANH><<<blocks, 128, 0, st>>>(a);
  else gated_step_kernel<T, false, TANH><<<blocks, 128, 0, st>>>(a);
  note_launch();
  return check_launch("gated_step_kernel");
}

}  // namespace

int tile_steps(int T, int B, int H) { return narrow(T, B, H) ? Narrow::STEPS : Forward::STEPS; }

int launch_forward(const Args& a, int dtype, cudaStream_t st) {
  if (dtype == B200GRU_F32) return a.tanh ? forward<float, true>(a, st) : forward<float, false>(a, st);
  if (dtype == B200GRU_BF16) return a.tanh ? forward<__nv_bfloat16, true>(a, st) : forward<__nv_bfloat16, false>(a, st);
  return a.tanh ? forward<__half, true>(a, st) : forward<__half, false>(a, st);
}

int launch_backward(const Args& a, int dtype, cudaStream_t st) {
  if (dtype == B200GRU_F32) return a.tanh ? backward<float, true>(a, st) : backward<float, false>(a, st);
  if (dtype == B200GRU_BF16) return a.tanh ? backward<__nv_bfloat16, true>(a, st) : backward<__nv_bfloat16, false>(a, st);
  return a.tanh ? backward<__half, true>(a, st) : backward<__half, false>(a, st);
}

int launch_step(const StepArgs& a, int dtype, cudaStream_t st) {
  if (dtype == B200GRU_F32) return a.tanh ? step<float, true>(a, st) : step<float, false>(a, st);
  if (dtype == B200GRU_BF16) return a.tanh ? step<__nv_bfloat16, true>(a, st) : step<__nv_bfloat16, false>(a, st);
  return a.tanh ? step<__half, true>(a, st) : step<__half, false>(a, st);
}

int read_status(int reset) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_gated_status, sizeof(int)) != cudaSuccess) return -1;
  if (reset && v != 0) {
    const int none = 0;
    cudaMemcpyToSymbol(g_gated_status, &none, sizeof(int));
  }
  return v;
}

}  // namespace gated
}  // namespace b200gru

using namespace b200gru;

namespace {

// 2 H, and a tile's units behind it, are 32-bit coordinates.
constexpr int MAX_UNITS = 0x40000000 - 64;

// Sizes and pointers that both directions need; every stride is non-negative.
int check_scan(const b200gru_gated_args* p) {
  if (p == nullptr || p->T <= 0 || p->B <= 0 || p->H <= 0 || p->gi == nullptr) return B200GRU_INVALID_ARGUMENT;
  if (p->dtype < B200GRU_F32 || p->dtype > B200GRU_F16) return B200GRU_INVALID_ARGUMENT;
  if (p->lengths != nullptr && p->length_bytes != 4 && p->length_bytes != 8) return B200GRU_INVALID_ARGUMENT;
  if ((long long)p->B * p->H > 0x7fffffffll || p->T > 0x40000000 || p->H > MAX_UNITS) return B200GRU_UNSUPPORTED;
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
  const long long size = p->dtype == B200GRU_F32 ? 4 : 2;
  a.out_step = p->out_t * size; a.dgi_step = p->dgi_t * size; a.half = p->H * size;
  return a;
}

}  // namespace

extern "C" {

size_t b200gru_gated_states_bytes(int T, int B, int H) {
  if (T <= 0 || B <= 0 || H <= 0) return 0;
  return (size_t)cdiv(T, gated::tile_steps(T, B, H)) * B * H * sizeof(float);
}

int b200gru_gated_scan_forward(const b200gru_gated_args* p, void* stream) try {
  const int rc = check_scan(p);
  if (rc) return rc;
  if (p->out == nullptr || p->h_T == nullptr || p->out_t <= 0 || p->out_b <= 0) return B200GRU_INVALID_ARGUMENT;
  return gated::launch_forward(to_args(p), p->dtype, static_cast<cudaStream_t>(stream));
} catch (...) {
  return B200GRU_LAUNCH_FAILURE;
}

int b200gru_gated_scan_backward(const b200gru_gated_args* p, void* stream) try {
  const int rc = check_scan(p);
  if (rc) return rc;
  if (p->states == nullptr || p->dgi == nullptr || p->dgi_t <= 0 || p->dgi_b <= 0) return B200GRU_INVALID_ARGUMENT;
  if (p->dout != nullptr && (p->dout_t < 0 || p->dout_b < 0)) return B200GRU_INVALID_ARGUMENT;
  return gated::launch_backward(to_args(p), p->dtype, static_cast<cudaStream_t>(stream));
} catch (...) {
  return B200GRU_LAUNCH_FAILURE;
}

int b200gru_gated_step(int dtype, int candidate_tanh, int B, int H, const void* gi, long long gi_b, const float* h,
                       long long h_b, void* out, float* h_new, long long hn_b, void* stream) {
  if (dtype < B200GRU_F32 || dtype > B200GRU_F16 || B <= 0 || H <= 0) return B200GRU_INVALID_ARGUMENT;
  if (gi == nullptr || h == nullptr || out == nullptr || h_new == nullptr) return B200GRU_INVALID_ARGUMENT;
  if (gi_b < 0 || h_b < 0 || hn_b < H) return B200GRU_INVALID_ARGUMENT;
  if ((long long)B * H > 0x7fffffffll || H > MAX_UNITS) return B200GRU_UNSUPPORTED;
  gated::StepArgs a;
  a.B = B; a.H = H; a.tanh = candidate_tanh != 0;
  a.gi = gi; a.gi_b = gi_b; a.h = h; a.h_b = h_b; a.out = out; a.h_new = h_new; a.hn_b = hn_b;
  return gated::launch_step(a, dtype, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
