// Products of sorted token rows with their experts' matrices, and the gradients of those products, in bf16 with fp32
// accumulation on the sm_100a tensor cores.  Expert e owns rows [offsets[e], offsets[e + 1]) of a row matrix.
//
//   product      out[r, c] = sum_k rows[r, k] op(W[e])[k, c]     contraction over either axis of the stored matrix
//   weight grad  out[e][m, c] = sum over the expert's rows r of a[r, m] b[r, c]
//
// Nothing is transposed in memory: the matrix descriptors of tcgen05 read an operand whose contraction axis is contiguous
// ("K-major": 64 elements of it are one 128-byte row of a swizzled tile) as well as one whose other axis is ("MN-major": a
// tile is 64 contraction steps of 64 contiguous outputs).  Forward reads W [K, N] MN-major, the gradient of the rows reads
// the same W K-major, the gradient of W reads both row matrices MN-major.
//
// Output columns are the M side of every MMA and output rows the N side: a tile is 256 columns x up to 256 rows on a CTA
// pair (cta_group::2), and an expert's rows are cut into tiles of nearly equal width, any multiple of 32, so that an odd
// load costs no padding to 256 and a few rows cost a stream of weights and little else.  Each CTA loads 128 of the columns
// and half of the rows per 64 contraction steps, 64 bytes per SM and tensor-pipe clock for a full tile, the smallest feed
// that two accumulators in TMEM allow.
//
// Warps of a persistent CTA (256 threads, weight grad 416):
//   0, 3   TMA producers of the column and the row operand
//   1      allocates TMEM; in the even CTA issues the MMAs (M 256, K 16), in the odd one hands out the pair's tiles
//   2      product: clears the rows of no expert
//   last   weight grad: fetches the rows of a contraction that do not fill a step of 16 into a buffer of their own, where
//   2      clears those behind them, which belong to the next expert (or hold what a caller left behind the last one), so
//          that they add nothing, whatever they hold.  (One warp for both waits out each copy before it asks for the next:
//          64 experts of 2048 x 2048, 125 rows each, 152 us, 131 so.)
//   4..    epilogue: groups of four warps take chunks of 32 output rows in turn.  An accumulator lane is an output column, so
//          the 32 values a warp holds of a row are 64 contiguous bytes and go straight out.  Turning a chunk around in
//          shared memory for longer stores costs the tensor pipe operand bandwidth, which the ring's copies and the MMAs
//          use up (4 x 1024 rows, 4096 x 14336, weight grad: 361 us turned, 353 straight; 32 x 16 rows, 4096 x 4096: 248, 194).
// Every wait is bounded; on expiry a code goes to `status`, no more work is issued, and the kernel tears down behind the copies and
// MMAs that are under way and leaves NaN where it has written nothing.
#include <cuda.h>

#include <atomic>
#include <type_traits>

#include "common.cuh"
#include "tcgen05_ptx.cuh"

namespace b200moe {
namespace {

constexpr int kMaxExperts = 1024;
constexpr int kMaxRows = 1 << 30;  // indices of tiles behind the last row stay below 2^31
constexpr int kMaxSize = 1 << 27;  // of a matrix; fewer than 2^20 column tiles
constexpr int kStages = 6;
constexpr int kOperand = 128 * 128;  // bytes of one operand's part of a stage: 128 rows of 128 bytes
constexpr int kStage = 2 * kOperand;
constexpr int kGroup = 8;    // row tiles that are walked together for every column tile: they share a weight tile in L2
constexpr int kTail = 4 * 2048;  // weight grad: 16 contraction rows of either operand, two boxes of 64 outputs each

// n / d for 0 <= n < 2^31 without a division: n * m >> 31 + s with m the reciprocal rounded up (1 <= d < 2^30).
struct Divisor {
  uint32_t d, m;
  int s;
  __device__ __forceinline__ int quotient(int n) const {
    return d == 1 ? n : static_cast<int>(__umulhi(static_cast<uint32_t>(n), m) >> (s - 1));
  }
};
inline Divisor make_divisor(uint32_t d) {
  int s = 0;
  while ((1u << s) < d) ++s;
  return {d, static_cast<uint32_t>(((uint64_t{1} << (31 + s)) / d) + 1), s};
}

struct Params {
  const int32_t* offsets;
  int R, E;
  int rows, cols;  // weight grad: the size of its matrices; product: output columns
  int k;           // product: contraction length
  int row_tiles, col_tiles;  // product: row_tiles unused
  int width;                 // weight grad: rows of a tile
  Divisor per_matrix, per_group;  // tiles of a matrix (weight grad) and of kGroup row tiles
  __nv_bfloat16* out;
  int parts;         // the contraction is cut into this many; above 1, part i's sums go to partial[i]
  float* partial;    // [parts][output rows][cols]
  int64_t out_rows;  // of all experts
  int32_t* status;
  int64_t wait_cycles;  // a wait gives up after as many
  int32_t* taken;  // tiles handed out beyond every pair's first; NULL: pair u walks tiles u, u + pairs, ...
  int queue;       // ... and how many of them a pair holds at most
};

constexpr int kQueue = 4;

struct Sched {
  int first[kMaxExperts + 1];  // first row of expert e
  int tiles[kMaxExperts + 1];  // product: tiles before expert e
  int queue[kQueue];
};

// Epilogue groups of four warps: one for a product, whose stores pass while the next tile's contraction runs, two where that is
// as short as the stores (SHORT; 9216 rows on 6 experts of K x 13376, one group / two: K 64 79 / 64 us, 256 85 / 72; of 512 x 8192
// 68 / 68) and for the weight grad.
template <bool WGRAD, bool SHORT>
struct Config {
  static constexpr int kGroups = WGRAD || SHORT ? 2 : 1;
  static constexpr int kTails = WGRAD ? 2 : 0;
  static constexpr int kThreads = 128 + kGroups * 128 + (WGRAD ? 32 : 0);
  static constexpr int kOffTail = kStages * kStage;
  static constexpr int kOffBar = kOffTail + kTails * kTail;
  static constexpr int kOffSched = kOffBar + 512;
  static constexpr int kSmem = kOffSched + static_cast<int>(sizeof(Sched)) + 1024;
  static_assert(kSmem <= 227 * 1024, "shared memory of expert_linear_kernel");
};

// MN-major tile, 128B swizzle: rows of 64 contiguous outputs, eight contraction steps per 1024 bytes; the second 64
// outputs follow `box` bytes later, behind all steps of the first.
__device__ __forceinline__ uint64_t desc_sw128_mn(uint32_t saddr, uint32_t box = 8192) {
  uint64_t d = static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4);
  d |= static_cast<uint64_t>(box >> 4) << 16;   // leading byte offset: to the next 64 outputs
  d |= static_cast<uint64_t>(1024 >> 4) << 32;  // stride byte offset: to the next eight contraction steps
  d |= static_cast<uint64_t>(1) << 46;
  d |= static_cast<uint64_t>(2) << 61;
  return d;
}

__device__ __forceinline__ bool mbar_try_wait_cluster(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, %3;\n"
      "selp.u32 %0, 1, 0, p;\n"
      "}\n"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity), "r"(kSuspendNs)
      : "memory");
  return ok != 0;
}
// A wait's bound and where it is reported.  What is bounded is a standstill: an accumulator is waited for as long as its contraction
// takes (2^24 slabs are 4 s), so the time starts again with every slab that the ring has taken on since.  These are finitely many.
struct Bound {
  volatile int* abort_flag;     // of the CTA
  const volatile int* started;  // slabs of the CTA's ring so far, modulo 2^32
  int32_t* status;
  int64_t cycles;
};
struct Clock {
  const Bound& bound;
  int seen;
  long long t0;
  // Whether the wait is over without its barrier: its time is up or another warp of the CTA has given up.
  __device__ __forceinline__ bool over(int code) {
    if (*bound.abort_flag) return true;
    const int now = *bound.started;
    if (now != seen) {
      seen = now;
      t0 = clock64();
    }
    if (clock64() - t0 <= bound.cycles) return false;
    *bound.abort_flag = 1;
    atomicCAS(bound.status, 0, code);
    return true;
  }
};
// A whole warp waits.  Its lanes leave together: one that saw the barrier complete beside one that saw the CTA give up would wait
// for it at the next __syncwarp for good.  The part behind the first look (which lasts 20 us) is a call: in line at nine places it
// cost 1 to 2 % (weight gradient of 8 x 16 rows, 4096 x 28672: 410 us, 402 so; of 64 x 125 rows, 2048 x 2048: 153 and 150).
template <bool CLUSTER>
__device__ __forceinline__ bool look(uint64_t* bar, uint32_t parity) {
  return __all_sync(0xffffffffu, CLUSTER ? mbar_try_wait_cluster(bar, parity) : mbar_try_wait(bar, parity));
}
template <bool CLUSTER>
__device__ __noinline__ bool look_on(uint64_t* bar, uint32_t parity, Bound bound, int code) {
  Clock clock{bound, *bound.started, clock64()};
  while (!look<CLUSTER>(bar, parity))
    if (__any_sync(0xffffffffu, clock.over(code))) return false;
  return true;
}
template <bool CLUSTER = false>
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, const Bound& bound, int code) {
  return look<CLUSTER>(bar, parity) || look_on<CLUSTER>(bar, parity, bound, code);
}
// One lane waits, the others do not.
__device__ __forceinline__ bool lane_wait_cluster(uint64_t* bar, uint32_t parity, const Bound& bound, int code) {
  Clock clock{bound, *bound.started, clock64()};
  while (!mbar_try_wait_cluster(bar, parity))
    if (clock.over(code)) return false;
  return true;
}

struct Tile {
  int expert;
  int row0, rows;  // output rows: of the row matrix (product), of the expert's matrix (weight grad)
  int c0;          // first output column
  int k0, k;       // the contraction's range (weight grad: of rows)
  int part;
  // Steps of 16 that the ring brings (a weight grad's ragged end comes through its own buffer), and slabs of four.
  template <bool WGRAD>
  __device__ __forceinline__ int steps() const { return WGRAD ? k >> 4 : (k + 15) >> 4; }
  template <bool WGRAD>
  __device__ __forceinline__ int slabs() const { return (steps<WGRAD>() + 3) >> 2; }
};

// Tiles of a matrix of row_tiles x col_tiles in groups of kGroup row tiles.
__device__ __forceinline__ void grouped_order(const Params& p, int i, int row_tiles, int& rt, int& ct) {
  const int g = p.per_group.quotient(i), r = i - g * kGroup * p.col_tiles;
  const int width = min(kGroup, row_tiles - g * kGroup);
  if (width == kGroup) {
    ct = r / kGroup;
  } else {  // r < 2^23: the product is off by less than one
    ct = static_cast<int>(static_cast<float>(r) * __frcp_rn(static_cast<float>(width)));
    const int rest = r - ct * width;
    ct += rest >= width ? 1 : (rest < 0 ? -1 : 0);
  }
  rt = g * kGroup + r - ct * width;
}

__device__ __forceinline__ int round_up32(int v) { return (v + 31) & ~31; }

template <bool WGRAD>
__device__ __forceinline__ Tile decode_tile(const Params& p, const Sched& s, int tile) {
  Tile t;
  int rt, ct;
  t.part = 0;
  if (p.parts > 1) {
    const int whole = WGRAD ? p.E * p.row_tiles * p.col_tiles : s.tiles[p.E];
    t.part = tile / whole;
    tile -= t.part * whole;
  }
  if constexpr (WGRAD) {
    t.expert = p.per_matrix.quotient(tile);
    grouped_order(p, tile - t.expert * p.row_tiles * p.col_tiles, p.row_tiles, rt, ct);
    t.k0 = s.first[t.expert];
    t.k = s.first[t.expert + 1] - t.k0;
    t.row0 = rt * p.width;
    t.rows = min(p.width, p.rows - t.row0);
  } else {
    int lo = 0, hi = p.E - 1;  // the last expert whose first tile is not behind this one
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (s.tiles[mid] <= tile) lo = mid;
      else hi = mid - 1;
    }
    t.expert = lo;
    const int first = s.first[lo], count = s.first[lo + 1] - first;
    const int row_tiles = (count + 255) >> 8;
    grouped_order(p, tile - s.tiles[lo], row_tiles, rt, ct);
    const int width = round_up32((count + row_tiles - 1) / row_tiles);
    t.row0 = first + rt * width;
    t.rows = min(width, count - rt * width);
    t.k0 = 0;
    t.k = p.k;
  }
  t.c0 = ct * 256;
  if (p.parts > 1) {  // whole slabs to every part, what is left of the last one to the last part
    const int64_t slabs = (t.k + 63) >> 6;
    const int from = static_cast<int>(slabs * t.part / p.parts) * 64;
    const int to = min(static_cast<int>(slabs * (t.part + 1) / p.parts) * 64, t.k);
    t.k0 += from;
    t.k = to - from;
  }
  return t;
}

// Arrive at a barrier of the odd CTA, which hands out the tiles.  What it announces is that a load has returned (its value has
// decided a branch), so it orders nothing: a release would wait for the epilogue's stores.
__device__ __forceinline__ void mbar_arrive_odd_relaxed(uint64_t* bar) {
  uint32_t remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_u32(bar)), "r"(1));
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(remote) : "memory");
}

// The tiles of a pair, as one warp sees them.
template <bool QUEUE>
struct Walk {
  const Params& p;
  const Sched& s;
  uint64_t *full, *empty;  // of the queue's entries: per CTA, in the odd CTA
  const Bound& bound;
  int unit, n_units, total, i;
  // The next tile, -1 behind the last.
  __device__ __forceinline__ int next() {
    const int at = i++;
    if (!QUEUE || p.taken == nullptr || at == 0) {
      const int64_t tile = unit + static_cast<int64_t>(at) * n_units;
      return tile < total ? static_cast<int>(tile) : -1;
    }
    const int slot = (at - 1) % p.queue;
    if (!warp_wait<true>(&full[slot], (at - 1) / p.queue & 1, bound, 47)) return -1;
    const int tile = *static_cast<const volatile int*>(&s.queue[slot]);
    __syncwarp();
    if (tile >= total) return -1;
    if ((threadIdx.x & 31) == 0) mbar_arrive_odd_relaxed(&empty[slot]);
    return tile;
  }
};

// 0x7fff7fff is NaN as fp32 and as two bf16.  A call, by the whole CTA, since in line it cost the weight gradient 1 %.
__device__ __noinline__ void fill_nan(void* at, int64_t bytes) {
  for (int64_t i = threadIdx.x; i < bytes / 16; i += blockDim.x)
    static_cast<uint4*>(at)[i] = make_uint4(0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu);
}

// Row boxes of a product: 128, 64, 32 and 16 rows (a tile's half is any multiple of 16).  Weight grad: of the row and the
// column operand 64 contraction rows in size[0] and the kernel's own column map, 16 in size[2] and size[3].
struct RowMaps { CUtensorMap size[4]; };

// COL_MN: the column operand is MN-major (always so for the weight grad, whose row operand is too).
template <bool WGRAD, bool COL_MN, bool SHORT>
__global__ void __launch_bounds__(Config<WGRAD, SHORT>::kThreads, 1) __cluster_dims__(2, 1, 1)
expert_linear_kernel(const __grid_constant__ CUtensorMap col_map, const __grid_constant__ RowMaps row_map, const Params p) {
  using C = Config<WGRAD, SHORT>;
  constexpr int kGroups = C::kGroups, kThreads = C::kThreads;
  constexpr uint32_t kTmemCols = 512;
  constexpr uint32_t kIdesc = make_idesc_bf16(256, 0) | (COL_MN ? 1u << 15 : 0u) | (WGRAD ? 1u << 16 : 0u);  // N per tile

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kOffBar);
  uint64_t* full = bars;
  uint64_t* empty = bars + kStages;
  uint64_t* tmem_full = bars + 2 * kStages;
  uint64_t* tmem_empty = tmem_full + 2;
  uint64_t* tail_full = tmem_full + 4;   // a ragged end landed (per CTA),
  uint64_t* tail_ready = tmem_full + 6;  // is cleared in both CTAs (even CTA),
  uint64_t* tail_empty = tmem_full + 8;  // and has been used
  uint64_t* queue_full = tmem_full + 10;
  uint64_t* queue_empty = queue_full + kQueue;
  uint32_t* tmem_ptr = reinterpret_cast<uint32_t*>(queue_empty + kQueue);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_ptr + 1);
  volatile int* started = abort_flag + 1;
  Sched& s = *reinterpret_cast<Sched*>(smem + C::kOffSched);

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
  const int lane = threadIdx.x & 31;
  const int rank = static_cast<int>(cluster_cta_rank());
  const int unit = blockIdx.x >> 1, n_units = gridDim.x >> 1;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tmem_full[a], 1);
      mbar_init(&tmem_empty[a], 2 * 4 * kGroups);
      mbar_init(&tail_full[a], 1);
      mbar_init(&tail_ready[a], 2);
      mbar_init(&tail_empty[a], 1);
    }
    for (int a = 0; a < kQueue; ++a) {
      mbar_init(&queue_full[a], 1);
      mbar_init(&queue_empty[a], 2 * (4 * kGroups + 2) + 1);  // every warp that walks the tiles
    }
    *abort_flag = *started = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_ptr)),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  const int32_t* offsets = p.offsets;
  grid_enter(offsets);
  if (blockIdx.x == 0 && threadIdx.x == 0) *p.status = 0;
  // Row ranges; whatever the offsets hold, no range leaves [0, R) and none is negative.
  for (int e = threadIdx.x; e <= p.E; e += kThreads) s.first[e] = min(max(offsets[e], 0), p.R);
  __syncthreads();
  if (warp == 0) {
    int top = 0, run = 0;
    for (int e0 = 0; e0 <= p.E; e0 += 32) {
      const int e = e0 + lane;
      int at = e <= p.E ? s.first[e] : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, at, o);
        if (lane >= o) at = max(at, u);
      }
      at = max(at, top);
      int before = __shfl_up_sync(0xffffffffu, at, 1);
      if (lane == 0) before = e == 0 ? at : top;
      top = __shfl_sync(0xffffffffu, at, 31);
      int tiles = ((at - before + 255) >> 8) * p.col_tiles;  // of expert e - 1
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, tiles, o);
        if (lane >= o) tiles += u;
      }
      if (e <= p.E) {
        s.first[e] = at;
        s.tiles[e] = run + tiles;
      }
      run += __shfl_sync(0xffffffffu, tiles, 31);
    }
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // the peer's barriers exist before anything signals them
  tc_fence_after();
  const uint32_t tmem_base = *tmem_ptr;
  const int total = (WGRAD ? p.E * p.row_tiles * p.col_tiles : s.tiles[p.E]) * p.parts;
  const Bound bound{abort_flag, started, p.status, p.wait_cycles};
  Walk<!WGRAD> walk{p, s, queue_full, queue_empty, bound, unit, n_units, total, 0};

  if (warp == 0) {
    // ------------------------------------------------------------ producer of the column operand
    const bool leader = elect_one();
    int stage = 0;
    uint32_t phase = 0, taken_on = 0;
    bool ok = true;
    for (int tile = walk.next(); tile >= 0 && ok; tile = walk.next()) {
      const Tile t = decode_tile<WGRAD>(p, s, tile);
      const int slabs = t.slabs<WGRAD>(), c = t.c0 + rank * 128;
      // the even CTA's barrier counts both CTAs' bytes
      const uint32_t bytes = 2 * kOperand + (WGRAD ? (t.rows > 128 ? 2 : 1) * kOperand : round_up32(t.rows) * 128);
      for (int kb = 0; kb < slabs; ++kb) {
        if (!warp_wait(&empty[stage], phase ^ 1u, bound, 41)) { ok = false; break; }
        uint8_t* dst = smem + stage * kStage;
        if (leader) {
          *started = static_cast<int>(++taken_on);
          if (rank == 0) mbar_expect_tx(&full[stage], bytes);
          if constexpr (WGRAD) {
            tma2_load_2d(dst, &col_map, c, t.k0 + kb * 64, &full[stage]);
            tma2_load_2d(dst + 8192, &col_map, c + 64, t.k0 + kb * 64, &full[stage]);
          } else if constexpr (COL_MN) {
            tma2_load_3d(dst, &col_map, c, t.k0 + kb * 64, t.expert, &full[stage]);
            tma2_load_3d(dst + 8192, &col_map, c + 64, t.k0 + kb * 64, t.expert, &full[stage]);
          } else {
            tma2_load_3d(dst, &col_map, t.k0 + kb * 64, c, t.expert, &full[stage]);
          }
        }
        if (++stage == kStages) { stage = 0; phase ^= 1u; }
      }
    }
  } else if (warp == 3) {
    // ------------------------------------------------------------ producer of the row operand
    const bool leader = elect_one();
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int tile = walk.next(); tile >= 0 && ok; tile = walk.next()) {
      const Tile t = decode_tile<WGRAD>(p, s, tile);
      const int slabs = t.slabs<WGRAD>();
      const int half = round_up32(t.rows) >> 1;
      const int r = t.row0 + rank * half;
      for (int kb = 0; kb < slabs; ++kb) {
        if (!warp_wait(&empty[stage], phase ^ 1u, bound, 41)) { ok = false; break; }
        uint8_t* dst = smem + stage * kStage + kOperand;
        if (leader) {
          if constexpr (WGRAD) {
            tma2_load_2d(dst, &row_map.size[0], r, t.k0 + kb * 64, &full[stage]);
            if (t.rows > 128) tma2_load_2d(dst + 8192, &row_map.size[0], r + 64, t.k0 + kb * 64, &full[stage]);
          } else {
            const int k = t.k0 + kb * 64;
            int at = 0;
            if (half & 128) { tma2_load_2d(dst, &row_map.size[0], k, r, &full[stage]); at = 128; }
            if (half & 64) { tma2_load_2d(dst + at * 128, &row_map.size[1], k, r + at, &full[stage]); at += 64; }
            if (half & 32) { tma2_load_2d(dst + at * 128, &row_map.size[2], k, r + at, &full[stage]); at += 32; }
            if (half & 16) tma2_load_2d(dst + at * 128, &row_map.size[3], k, r + at, &full[stage]);
          }
        }
        if (++stage == kStages) { stage = 0; phase ^= 1u; }
      }
    }
  } else if (warp == 1 && rank == 0) {
    // ------------------------------------------------------------ MMA issuer
    const bool leader = elect_one();
    int stage = 0, it = 0, ends = 0;
    uint32_t phase = 0;
    bool ok = true;
    Tile t;
    int tile = walk.next();
    if (tile >= 0) t = decode_tile<WGRAD>(p, s, tile);
    const auto advance = [&] {
      tile = walk.next();
      if (tile >= 0) t = decode_tile<WGRAD>(p, s, tile);
    };
    while (tile >= 0 && ok) {
      const int k = t.k, slabs = t.slabs<WGRAD>(), last = t.steps<WGRAD>() - 4 * (slabs - 1);
      const uint32_t idesc = kIdesc | (static_cast<uint32_t>(round_up32(t.rows) >> 3) << 17);
      if (slabs == 0) advance();
      if (WGRAD && k == 0) continue;
      const int acc = it & 1;
      if (!warp_wait(&tmem_empty[acc], ((it >> 1) & 1) ^ 1u, bound, 42)) break;
      tc_fence_after();
      const uint32_t d_tmem = tmem_base + acc * 256;
      for (int kb = 0; kb < slabs; ++kb) {
        if (!warp_wait(&full[stage], phase, bound, 43)) { ok = false; break; }
        tc_fence_after();
        const uint32_t sc = smem_u32(smem + stage * kStage), sr = sc + kOperand;
        const uint64_t c_desc = COL_MN ? desc_sw128_mn(sc) : desc_sw128(sc);
        const uint64_t r_desc = WGRAD ? desc_sw128_mn(sr) : desc_sw128(sr);
        if (leader) {
          const int steps = kb == slabs - 1 ? last : 4;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (i < steps)  // 16 contraction steps: 32 bytes along a K-major row, 16 rows of an MN-major tile
              tc2_mma_bf16(d_tmem, c_desc + i * (COL_MN ? 128 : 2), r_desc + i * (WGRAD ? 128 : 2), idesc, (kb | i) != 0);
          }
          tc2_commit_pair(&empty[stage]);
        }
        if (kb == slabs >> 1) advance();  // while the tensor pipe has work
        if (++stage == kStages) { stage = 0; phase ^= 1u; }
      }
      if constexpr (WGRAD) if (ok && (k & 15) != 0) {
        const int b = ends % C::kTails;
        if (!warp_wait<true>(&tail_ready[b], ends / C::kTails & 1, bound, 44)) break;
        tc_fence_after();
        const uint32_t sc = smem_u32(smem + C::kOffTail + b * kTail);
        if (leader) {
          tc2_mma_bf16(d_tmem, desc_sw128_mn(sc, 2048), desc_sw128_mn(sc + 4096, 2048), idesc, slabs != 0);
          tc2_commit_pair(&tail_empty[b]);
        }
        ++ends;
      }
      if (ok && leader) tc2_commit_pair(&tmem_full[acc]);
      ++it;
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ tiles: one ticket after the other, for both CTAs
    if (!WGRAD && p.taken != nullptr && lane == 0) {
      for (int i = 0, tile = 0; tile < total; ++i) {
        const int slot = i % p.queue;
        if (!lane_wait_cluster(&queue_empty[slot], (i / p.queue & 1) ^ 1u, bound, 48)) break;
        tile = n_units + atomicAdd(p.taken, 1);
        *static_cast<volatile int*>(&s.queue[slot]) = tile;
        uint32_t remote;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_u32(&s.queue[slot])), "r"(0));
        asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(remote), "r"(tile) : "memory");
        mbar_arrive(&queue_full[slot]);
        mbar_arrive_leader(&queue_full[slot]);
      }
    }
    __syncwarp();
  } else if (!WGRAD && warp == 2) {
    // ------------------------------------------------------------ rows of no expert, beside the tiles
    if (p.parts == 1) {
      const int lo = s.first[0], hi = s.first[p.E], none = lo + p.R - hi;
      for (int i = blockIdx.x; i < none; i += gridDim.x) {
        uint4* row = reinterpret_cast<uint4*>(p.out + static_cast<int64_t>(i < lo ? i : i - lo + hi) * p.cols);
#pragma unroll 8
        for (int c = lane; c < p.cols >> 3; c += 32) row[c] = make_uint4(0, 0, 0, 0);
      }
    }
  } else if (WGRAD && warp == 2) {
    if constexpr (WGRAD) {
    // ------------------------------------------------------------ ragged ends
    int ends = 0;
    for (int tile = walk.next(); tile >= 0; tile = walk.next()) {
      const int rest = decode_tile<WGRAD>(p, s, tile).k & 15;
      if (rest == 0) continue;
      const int b = ends % C::kTails;
      uint8_t* base = smem + C::kOffTail + b * kTail;
      if (!warp_wait(&tail_full[b], ends / C::kTails & 1, bound, 45)) break;
      // 32 lanes clear 512 bytes: a row of all four boxes
      for (int r = rest; r < 16; ++r)
        *reinterpret_cast<uint4*>(base + (lane >> 3) * 2048 + r * 128 + (lane & 7) * 16) = make_uint4(0, 0, 0, 0);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive_leader(&tail_ready[b]);
      ++ends;
    }
    }
  } else if (WGRAD && warp == kThreads / 32 - 1) {
    if constexpr (WGRAD) {
    // ------------------------------------------------------------ producer of ragged ends
    const bool leader = elect_one();
    int ends = 0;
    for (int tile = walk.next(); tile >= 0; tile = walk.next()) {
      const Tile t = decode_tile<WGRAD>(p, s, tile);
      if ((t.k & 15) == 0) continue;
      const int b = ends % C::kTails;
      uint8_t* base = smem + C::kOffTail + b * kTail;
      if (!warp_wait(&tail_empty[b], (ends / C::kTails & 1) ^ 1u, bound, 49)) break;
      if (leader) {
        const int c = t.c0 + rank * 128, r = t.row0 + rank * (round_up32(t.rows) >> 1), k = t.k0 + (t.k & ~15);
        mbar_expect_tx(&tail_full[b], kTail);
        tma_load_2d(base, &row_map.size[3], c, k, &tail_full[b]);
        tma_load_2d(base + 2048, &row_map.size[3], c + 64, k, &tail_full[b]);
        tma_load_2d(base + 4096, &row_map.size[2], r, k, &tail_full[b]);
        tma_load_2d(base + 6144, &row_map.size[2], r + 64, k, &tail_full[b]);
      }
      ++ends;
    }
    }
  } else if (warp >= 4) {
    // ------------------------------------------------------------ epilogue
    const int q = warp & 3, group = (warp - 4) >> 2;
    int it = 0;
    for (int tile = walk.next(); tile >= 0; tile = walk.next()) {
      const Tile t = decode_tile<WGRAD>(p, s, tile);
      const int64_t row0 = (WGRAD ? static_cast<int64_t>(t.expert) * p.rows : 0) + t.row0;
      if (WGRAD && t.k == 0) {  // an expert without rows, or a part without: zeros, eight columns per thread
        const int c = t.c0 + rank * 128 + (lane & 15) * 8;
        for (int r = (warp - 4) * 2 + (lane >> 4); r < t.rows && c < p.cols; r += 8 * kGroups) {
          if (p.parts == 1) {
            *reinterpret_cast<uint4*>(p.out + (row0 + r) * p.cols + c) = make_uint4(0, 0, 0, 0);
          } else {
            uint4* o = reinterpret_cast<uint4*>(p.partial + (t.part * p.out_rows + row0 + r) * p.cols + c);
            o[0] = o[1] = make_uint4(0, 0, 0, 0);
          }
        }
        continue;
      }
      const int col = t.c0 + rank * 128 + q * 32 + lane;
      const int acc = it & 1;
      if (!warp_wait(&tmem_full[acc], (it >> 1) & 1, bound, 46)) break;
      __syncwarp();
      tc_fence_after();
      ++it;
      const uint32_t taddr = tmem_base + acc * 256 + (static_cast<uint32_t>(q * 32) << 16);
      const int chunks = (t.rows + 31) >> 5;
      // also a group without a chunk in this tile has to hand the accumulator back
      if (group >= chunks && lane == 0) mbar_arrive_leader_relaxed(&tmem_empty[acc]);
      __nv_bfloat16* out = p.out + (row0 + group * 32) * p.cols + col;
      for (int c = group; c < chunks; c += kGroups) {
        uint32_t v[32];
        tc_ld32_nowait(taddr + c * 32, v);
        tc_wait_ld();
        if (c + kGroups >= chunks) {  // the group's last look at this accumulator
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_leader_relaxed(&tmem_empty[acc]);
        }
        const int rows = min(32, t.rows - c * 32);
        if (col < p.cols && p.parts > 1) {
          float* o = p.partial + (t.part * p.out_rows + row0 + c * 32) * p.cols + col;
#pragma unroll
          for (int j = 0; j < 32; ++j, o += p.cols)
            if (j < rows) *o = __uint_as_float(v[j]);
        } else if (col < p.cols) {
          __nv_bfloat16* o = out;
          if (rows == 32) {
#pragma unroll
            for (int j = 0; j < 32; ++j, o += p.cols) *o = __float2bfloat16_rn(__uint_as_float(v[j]));
          } else {
#pragma unroll
            for (int j = 0; j < 32; ++j, o += p.cols)
              if (j < rows) *o = __float2bfloat16_rn(__uint_as_float(v[j]));
          }
        }
        __syncwarp();
        out += static_cast<int64_t>(kGroups) * 32 * p.cols;
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  // A pair that has given up may have copies and MMAs under way whose end nothing awaits, of microseconds: they get a hundred times
  // that before shared memory and TMEM go.  (A CTA whose waits all came through has none of its own.)
  if (*abort_flag)
    for (int i = 0; i < 2000; ++i) __nanosleep(1000);
  __syncwarp();
  cluster_sync_all();  // the peer may still read this CTA's shared memory until here
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(kTmemCols) : "memory");
  }
  // Which tiles the pair still owed is not known here: all of the result (or of the parts' sums) becomes NaN, behind the pair's own
  // stores, so that whatever is missing is one.
  if (*abort_flag) {
    const int64_t values = p.parts * p.out_rows * p.cols;
    if (p.parts > 1) fill_nan(p.partial, values * 4);
    else fill_nan(p.out, values * 2);
  }
}

// out = the parts' sums, added up in their order.  Eight columns per thread; rows of no expert (a product's: `offsets`) are zero.
__global__ void __launch_bounds__(256) join_parts_kernel(const float* partial, int parts, int64_t rows, int cols, const int32_t* offsets,
                                                         int E, __nv_bfloat16* out) {
  __shared__ int s_last;
  grid_enter(partial, offsets);
  int64_t lo = 0, hi = rows;
  if (offsets != nullptr) {  // the experts' rows go from the first offset to the largest one
    if (threadIdx.x == 0) s_last = 0;
    __syncthreads();
    int last = 0;
    for (int e = threadIdx.x; e <= E; e += 256) last = max(last, offsets[e]);
    atomicMax(&s_last, last);
    __syncthreads();
    lo = min(max(static_cast<int64_t>(offsets[0]), int64_t{0}), rows);
    hi = min(static_cast<int64_t>(s_last), rows);
  }
  const int64_t pieces = rows * (cols >> 3), stride = rows * cols;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < pieces; i += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t row = i / (cols >> 3);
    uint4 result = make_uint4(0, 0, 0, 0);
    if (row >= lo && row < hi) {
      float sum[8] = {};
#pragma unroll 4
      for (int part = 0; part < parts; ++part) {
        const float4* f = reinterpret_cast<const float4*>(partial + part * stride + i * 8);
        const float4 a = __ldcg(f), b = __ldcg(f + 1);
        sum[0] += a.x; sum[1] += a.y; sum[2] += a.z; sum[3] += a.w;
        sum[4] += b.x; sum[5] += b.y; sum[6] += b.z; sum[7] += b.w;
      }
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(sum[2 * j], sum[2 * j + 1]);
        w[j] = *reinterpret_cast<const uint32_t*>(&v);
      }
      result = make_uint4(w[0], w[1], w[2], w[3]);
    }
    *reinterpret_cast<uint4*>(out + i * 8) = result;
  }
}

// Parts to cut a contraction of `slabs` into where its `tiles` leave more than half of the CTA pairs idle: as many as there are
// pairs for, of eight slabs at least.  The join costs a launch, so each part has to save 48 slabs of about 0.25 us.  Without /
// with: 64 rows on 2 experts of 28672 x 512 105 / 26 us, 454 on 9 of 21304 x 560 85 / 55, weight gradient of 65536 rows on 2 of
// 256 x 512 152 / 36; 64 rows on one of 4096 x 4096, two parts, 22.0 / 24.6, which is why the bound is there.
int split_parts(int64_t tiles, int64_t slabs) {
  const int64_t units = sm_count() / 2;
  if (tiles * 2 > units) return 1;
  const int64_t parts = units / tiles < slabs / 8 ? units / tiles : slabs / 8;
  return parts > 1 && slabs - slabs / parts >= 48 ? static_cast<int>(parts) : 1;
}
int64_t product_tiles(int R, int E, int n) { return (ceil_div64(R, 256) + (E < R ? E : R)) * ceil_div64(n, 256); }
int64_t weight_grad_tiles(int E, int M, int N) { return E * ceil_div64(M, 256) * ceil_div64(N, 256); }

// bf16 matrix (or `batch` of them) with `cols` contiguous; boxes of 64 columns (128 bytes) x box_rows.
int make_map(CUtensorMap* map, const void* base, int64_t cols, int64_t rows, int64_t pitch, int64_t batch,
             int64_t batch_pitch, int box_rows) {
  EncodeTiledFn enc = get_encode_fn();
  B200MOE_REQUIRE(enc != nullptr, B200MOE_ERR_CUDA, "cuTensorMapEncodeTiled is not available from this driver");
  const cuuint32_t rank = batch > 0 ? 3 : 2;
  cuuint64_t dims[3] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows), static_cast<cuuint64_t>(batch > 0 ? batch : 1)};
  cuuint64_t strides[2] = {static_cast<cuuint64_t>(pitch) * 2, static_cast<cuuint64_t>(batch_pitch) * 2};
  cuuint32_t box[3] = {64, static_cast<cuuint32_t>(box_rows), 1};
  cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank, const_cast<void*>(base), dims, strides, box, estr,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  B200MOE_REQUIRE(r == CUDA_SUCCESS, B200MOE_ERR_CUDA, "cuTensorMapEncodeTiled failed with code %d", static_cast<int>(r));
  return B200MOE_OK;
}

template <bool WGRAD, bool COL_MN, bool SHORT>
int launch(const CUtensorMap& cols, const RowMaps& rows, const Params& p, int64_t tiles, cudaStream_t st) {
  auto kern = expert_linear_kernel<WGRAD, COL_MN, SHORT>;
  using C = Config<WGRAD, SHORT>;
  B200MOE_CUDA_OK(ensure_dynamic_smem(reinterpret_cast<const void*>(kern), C::kSmem));
  const int64_t units = sm_count() / 2, work = tiles * p.parts;
  B200MOE_CUDA_OK(launch_overlapped(kern, dim3(static_cast<unsigned>(2 * (work < units ? work : units))), C::kThreads, C::kSmem, st,
                                    cols, rows, p));
  B200MOE_LAUNCH_OK("expert_linear_kernel");
  if (p.parts > 1) {
    const int64_t pieces = p.out_rows * (p.cols / 8), ctas = ceil_div64(pieces, 256), most = static_cast<int64_t>(sm_count()) * 8;
    B200MOE_CUDA_OK(launch_overlapped(join_parts_kernel, dim3(static_cast<unsigned>(ctas < most ? ctas : most)), 256, 0, st,
                                      static_cast<const float*>(p.partial), p.parts, p.out_rows, p.cols,
                                      WGRAD ? static_cast<const int32_t*>(nullptr) : p.offsets, p.E, p.out));
    B200MOE_LAUNCH_OK("join_parts_kernel");
  }
  return B200MOE_OK;
}

std::atomic<int64_t> wait_cycles{kWaitCycles};

bool rows_ok(const void* p, int64_t pitch, int cols) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && pitch % 8 == 0 && pitch >= cols && pitch < (int64_t{1} << 38);
}

}  // namespace
}  // namespace b200moe

using namespace b200moe;

extern "C" int64_t b200moe_expert_wait_cycles(int64_t cycles) { return wait_cycles.exchange(cycles); }

extern "C" size_t b200moe_expert_product_workspace_bytes(int contract_last, int R, int E, int D0, int D1) {
  if (R <= 0 || E <= 0 || D0 <= 0 || D1 <= 0) return 0;
  const int k = contract_last ? D1 : D0, n = contract_last ? D0 : D1;
  const int parts = split_parts(product_tiles(R, E, n), ceil_div64(k, 64));
  return parts > 1 ? static_cast<size_t>(parts) * R * n * sizeof(float) : 0;
}

extern "C" size_t b200moe_expert_weight_grad_workspace_bytes(int R, int E, int M, int N) {
  if (R <= 0 || E <= 0 || M <= 0 || N <= 0) return 0;
  const int parts = split_parts(weight_grad_tiles(E, M, N), R / (static_cast<int64_t>(E) * 64));
  return parts > 1 ? static_cast<size_t>(parts) * E * M * N * sizeof(float) : 0;
}

extern "C" int b200moe_expert_product(const void* rows_bf16, int64_t rows_pitch, const void* weight_bf16, int64_t w_pitch,
                                      int64_t w_expert_pitch, int contract_last, const int32_t* expert_offsets, int R, int E,
                                      int D0, int D1, void* out_bf16, void* workspace, size_t workspace_bytes, int32_t* status,
                                      b200moe_stream_t stream) {
  B200MOE_REQUIRE(rows_bf16 && weight_bf16 && expert_offsets && out_bf16 && status, B200MOE_ERR_INVALID,
                  "expert_product: null pointer argument");
  B200MOE_REQUIRE(R > 0 && R <= kMaxRows && E > 0 && E <= kMaxExperts, B200MOE_ERR_INVALID,
                  "expert_product: need at least one row and at most 2^30, and between 1 and %d experts", kMaxExperts);
  B200MOE_REQUIRE(D0 > 0 && D1 > 0 && D0 % 8 == 0 && D1 % 8 == 0 && D0 <= kMaxSize && D1 <= kMaxSize, B200MOE_ERR_INVALID,
                  "expert_product: both sizes of a weight matrix must be positive multiples of 8, at most 2^27, got %d x %d", D0, D1);
  const int k = contract_last ? D1 : D0, n = contract_last ? D0 : D1;
  B200MOE_REQUIRE(rows_ok(rows_bf16, rows_pitch, k) && rows_ok(weight_bf16, w_pitch, D1) &&
                      rows_ok(weight_bf16, w_expert_pitch, D1),
                  B200MOE_ERR_INVALID, "expert_product: rows and weights must start on 16-byte boundaries");
  B200MOE_REQUIRE((reinterpret_cast<uintptr_t>(out_bf16) & 15) == 0, B200MOE_ERR_INVALID,
                  "expert_product: out must be 16-byte aligned");
  Params p{};
  p.offsets = expert_offsets;
  p.R = R;
  p.E = E;
  p.cols = n;
  p.k = k;
  p.col_tiles = (n + 255) / 256;
  p.per_matrix = p.per_group = make_divisor(static_cast<uint32_t>(kGroup * p.col_tiles));
  p.out = static_cast<__nv_bfloat16*>(out_bf16);
  p.status = status;
  p.wait_cycles = wait_cycles.load();
  const int64_t most_tiles = product_tiles(R, E, n);
  p.parts = split_parts(most_tiles, ceil_div64(k, 64));
  p.partial = static_cast<float*>(workspace);
  p.out_rows = R;
  B200MOE_REQUIRE(p.parts == 1 || (workspace != nullptr && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0 &&
                                   workspace_bytes >= b200moe_expert_product_workspace_bytes(contract_last, R, E, D0, D1)),
                  B200MOE_ERR_WORKSPACE, "expert_product: workspace too small or not 16-byte aligned");
  B200MOE_REQUIRE(most_tiles < (int64_t{1} << 30), B200MOE_ERR_INVALID, "expert_product: too many output tiles");
  CUtensorMap cols;
  RowMaps rows;
  int rc = make_map(&cols, weight_bf16, D1, D0, w_pitch, E, w_expert_pitch, contract_last ? 128 : 64);
  for (int i = 0; i < 4 && rc == B200MOE_OK; ++i) rc = make_map(&rows.size[i], rows_bf16, k, R, rows_pitch, 0, 0, 128 >> i);
  if (rc != B200MOE_OK) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  // Row tiles of an expert share its weight tiles in L2 as long as they run side by side.  A fixed walk drifts apart, since
  // tiles differ in width; handed out in order as pairs come free they stay together (32 experts of 7168 x 4096, 32768
  // rows, skewed: 5.6 -> 2.8 GB from DRAM, 1533 -> 1356 us; its row gradient 3.6 -> 2.4 GB, 1440 -> 1342 us).  The drift is a few
  // tiles, so it costs nothing until the operands are many times L2, while the counter's memset and the queue cost 4 us and more.
  // Fixed / handed out by the operands' size, two or more row tiles per expert: 71 MB (16000 rows, 256 x 32768) 422 / 440 us, 95 MB
  // (64000 rows) 1352 / 1439, 160 MB (8192 rows, 2048 x 4096) 97 / 100, 320 MB (4096 x 4096) 190 / 195 and its row gradient 209 / 217,
  // 576 MB (4096 x 8192) 415 / 418, 605 MB (24000 rows, 2048 x 4096) 372 / 381, 737 MB (skewed) 780 / 776, 960 MB (4096 x 14336)
  // 758 / 753, 1.2 GB (skewed) 1569 / 1549, 2.0 GB (24000 rows, 7168 x 4096) 1339 / 1292 and 1294 / 1246: half a gigabyte is where loss
  // turns into gain.  One row tile per expert has nothing to share.  The weight gradient's short contractions lose everywhere
  // (4 x 1024 rows, 4096 x 14336: 353 and 367 us).
  // The queue holds two tiles, four where contractions are too short to hide a ticket's way (256 x 32768 above: 462 us with two,
  // 440 with four; from 1024 on the two are within 2 % of each other, either way).
  const int64_t bytes = 2 * (static_cast<int64_t>(E) * D0 * D1 + static_cast<int64_t>(R) * k);
  if (R >= 512 * static_cast<int64_t>(E) && bytes >= (int64_t{1} << 29) && most_tiles >= 4 * (sm_count() / 2)) {
    p.taken = status + 1;
    p.queue = k >= 1024 ? 2 : kQueue;
    B200MOE_CUDA_OK(cudaMemsetAsync(p.taken, 0, sizeof(int32_t), st));
  }
  const auto go = [&](auto brief) {
    constexpr bool S = decltype(brief)::value;
    return contract_last ? launch<false, false, S>(cols, rows, p, most_tiles, st) : launch<false, true, S>(cols, rows, p, most_tiles, st);
  };
  return k <= 384 ? go(std::true_type{}) : go(std::false_type{});
}

extern "C" int b200moe_expert_weight_grad(const void* a_bf16, int64_t a_pitch, const void* b_bf16, int64_t b_pitch,
                                          const int32_t* expert_offsets, int R, int E, int M, int N, void* out_bf16,
                                          void* workspace, size_t workspace_bytes, int32_t* status, b200moe_stream_t stream) {
  B200MOE_REQUIRE(a_bf16 && b_bf16 && expert_offsets && out_bf16 && status, B200MOE_ERR_INVALID,
                  "expert_weight_grad: null pointer argument");
  B200MOE_REQUIRE(R > 0 && R <= kMaxRows && E > 0 && E <= kMaxExperts, B200MOE_ERR_INVALID,
                  "expert_weight_grad: need at least one row and at most 2^30, and between 1 and %d experts", kMaxExperts);
  B200MOE_REQUIRE(M > 0 && N > 0 && M % 8 == 0 && N % 8 == 0 && M <= kMaxSize && N <= kMaxSize, B200MOE_ERR_INVALID,
                  "expert_weight_grad: both sizes of a weight matrix must be positive multiples of 8, at most 2^27, got %d x %d", M, N);
  B200MOE_REQUIRE(rows_ok(a_bf16, a_pitch, M) && rows_ok(b_bf16, b_pitch, N), B200MOE_ERR_INVALID,
                  "expert_weight_grad: rows must start on 16-byte boundaries");
  B200MOE_REQUIRE((reinterpret_cast<uintptr_t>(out_bf16) & 15) == 0, B200MOE_ERR_INVALID,
                  "expert_weight_grad: out must be 16-byte aligned");
  Params p{};
  p.offsets = expert_offsets;
  p.R = R;
  p.E = E;
  p.rows = M;
  p.cols = N;
  p.row_tiles = (M + 255) / 256;
  p.col_tiles = (N + 255) / 256;
  // even tiles, as in a product (110 rows each on 145 experts of 320 x 7192: 294 us, with tiles of 256 rows 372; of 4096 x 14336 alike)
  p.width = ((M + p.row_tiles - 1) / p.row_tiles + 31) & ~31;
  p.out = static_cast<__nv_bfloat16*>(out_bf16);
  p.status = status;
  p.wait_cycles = wait_cycles.load();
  const int64_t tiles = weight_grad_tiles(E, M, N);
  p.parts = split_parts(tiles, R / (static_cast<int64_t>(E) * 64));
  p.partial = static_cast<float*>(workspace);
  p.out_rows = static_cast<int64_t>(E) * M;
  B200MOE_REQUIRE(p.parts == 1 || (workspace != nullptr && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0 &&
                                   workspace_bytes >= b200moe_expert_weight_grad_workspace_bytes(R, E, M, N)),
                  B200MOE_ERR_WORKSPACE, "expert_weight_grad: workspace too small or not 16-byte aligned");
  B200MOE_REQUIRE(tiles < (int64_t{1} << 30), B200MOE_ERR_INVALID, "expert_weight_grad: too many output tiles");
  p.per_matrix = make_divisor(static_cast<uint32_t>(p.row_tiles * p.col_tiles));
  p.per_group = make_divisor(static_cast<uint32_t>(kGroup * p.col_tiles));
  CUtensorMap cols;
  RowMaps rows;
  int rc = make_map(&cols, b_bf16, N, R, b_pitch, 0, 0, 64);
  if (rc == B200MOE_OK) rc = make_map(&rows.size[0], a_bf16, M, R, a_pitch, 0, 0, 64);
  if (rc == B200MOE_OK) rc = make_map(&rows.size[2], a_bf16, M, R, a_pitch, 0, 0, 16);
  if (rc == B200MOE_OK) rc = make_map(&rows.size[3], b_bf16, N, R, b_pitch, 0, 0, 16);
  if (rc != B200MOE_OK) return rc;
  rows.size[1] = rows.size[0];  // never used
  return launch<true, true, false>(cols, rows, p, tiles, static_cast<cudaStream_t>(stream));
}
