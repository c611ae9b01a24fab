// Products of sorted token rows with their experts' matrices, and the gradients of those products, in bf16 with fp32
// accumulation on the sm_100a tensor cores.  Expert e owns rows [offsets[e], offsets[e + 1]) of a row matrix.
//
//   product      out[r, n] = sum_k rows[r, k] op(W[e])[k, n]     contraction over either axis of the stored matrix
//   weight grad  out[e][m, n] = sum over the expert's rows r of a[r, m] b[r, n]
//
// Nothing is transposed in memory: the matrix descriptors of tcgen05 read an operand whose contraction axis is contiguous
// ("K-major": 64 elements of it are one 128-byte row of a swizzled tile) as well as one whose other axis is ("MN-major": a
// tile is 64 contraction steps of 64 contiguous outputs).  Forward reads W [K, N] MN-major, the gradient of the rows reads
// the same W K-major, the gradient of W reads both row matrices MN-major.
//
// A tile is 256 x 256 outputs on a CTA pair (cta_group::2): each CTA loads 128 rows of either operand per 64 contraction
// steps (32 KB), i.e. 64 bytes per SM and tensor-pipe clock, the smallest feed that two accumulators in TMEM allow.
//
// Warps of a persistent CTA (384 threads):
//   0, 3   TMA producers of the A and the B operand
//   1      allocates TMEM; in the even CTA issues the MMAs (M 256, N 256, K 16)
//   2      weight grad: clears the rows of a contraction's last 16 that belong to the next expert (or hold what a caller
//          left behind the last one), so that they add nothing, whatever they hold
//   4..11  epilogue: accumulator lane = output row, two warps per 32 lanes take 128 columns each
// Every wait is bounded; on expiry a code goes to `status`, no more work is issued and the kernel tears down.
#include <cuda.h>

#include "common.cuh"
#include "tcgen05_ptx.cuh"

namespace b200moe {
namespace {

constexpr int kMaxExperts = 1024;
constexpr int kThreads = 384;
constexpr int kStages = 6;
constexpr int kOperand = 128 * 128;  // bytes of one operand's part of a stage: 128 rows of 128 bytes
constexpr int kStage = 2 * kOperand;
constexpr int kGroup = 8;  // row tiles that are walked together for every column tile: they share a weight tile in L2

struct Params {
  const int32_t* offsets;
  int R, E;
  int m, n;         // weight grad: its matrix; product: n output columns
  int k;            // product: contraction length
  int m_tiles, n_tiles;  // product: m_tiles unused
  __nv_bfloat16* out;
  int wide_stores;  // output rows start on 32-byte boundaries
  int32_t* status;
};

struct Sched {
  int first[kMaxExperts + 1];  // first row of expert e
  int tiles[kMaxExperts + 1];  // product: tiles before expert e
};

constexpr int kOffBar = kStages * kStage;
constexpr int kOffSched = kOffBar + 512;
constexpr int kSmem = kOffSched + static_cast<int>(sizeof(Sched)) + 1024;
static_assert(kSmem <= 227 * 1024, "shared memory of expert_linear_kernel");

// MN-major tile, 128B swizzle: rows of 64 contiguous outputs, eight contraction steps per 1024 bytes; the second 64
// outputs follow 64 steps (8192 bytes) later.
__device__ __forceinline__ uint64_t desc_sw128_mn(uint32_t saddr) {
  uint64_t d = static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4);
  d |= static_cast<uint64_t>(8192 >> 4) << 16;  // leading byte offset: to the next 64 outputs
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
__device__ __forceinline__ bool mbar_wait_cluster(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int32_t* status,
                                                  int code) {
  const long long t0 = clock64();
  while (!mbar_try_wait_cluster(bar, parity)) {
    if (*abort_flag) return false;
    if (clock64() - t0 > kWaitCycles) {
      *abort_flag = 1;
      atomicCAS(status, 0, code);
      return false;
    }
  }
  return true;
}

struct Tile {
  int expert, row0, rows;  // weight grad: the contraction's rows; product: output rows
  int m0, n0;              // first output row of the tile (weight grad: within the matrix) and column
};

// Tiles of a matrix of m_tiles x n_tiles in groups of kGroup row tiles.
__device__ __forceinline__ void grouped_order(int i, int m_tiles, int n_tiles, int& mt, int& nt) {
  const int g = i / (kGroup * n_tiles), r = i - g * kGroup * n_tiles;
  const int width = min(kGroup, m_tiles - g * kGroup);
  nt = r / width;
  mt = g * kGroup + r - nt * width;
}

template <bool WGRAD>
__device__ __forceinline__ Tile decode_tile(const Params& p, const Sched& s, int tile) {
  Tile t;
  int mt, nt;
  if constexpr (WGRAD) {
    const int per = p.m_tiles * p.n_tiles;
    t.expert = tile / per;
    grouped_order(tile - t.expert * per, p.m_tiles, p.n_tiles, mt, nt);
    t.row0 = s.first[t.expert];
    t.rows = s.first[t.expert + 1] - t.row0;
    t.m0 = mt * 256;
  } else {
    int lo = 0, hi = p.E - 1;  // the last expert whose first tile is not behind this one
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (s.tiles[mid] <= tile) lo = mid;
      else hi = mid - 1;
    }
    t.expert = lo;
    const int first = s.first[lo], end = s.first[lo + 1];
    grouped_order(tile - s.tiles[lo], (end - first + 255) >> 8, p.n_tiles, mt, nt);
    t.m0 = 0;
    t.row0 = first + mt * 256;
    t.rows = min(256, end - t.row0);
  }
  t.n0 = nt * 256;
  return t;
}

// B_MN: the B operand is MN-major (always so for the weight grad, whose A operand is too).
template <bool WGRAD, bool B_MN>
__global__ void __launch_bounds__(kThreads, 1) __cluster_dims__(2, 1, 1)
expert_linear_kernel(const __grid_constant__ CUtensorMap a_map, const __grid_constant__ CUtensorMap b_map, const Params p) {
  constexpr bool A_MN = WGRAD;
  constexpr uint32_t kTmemCols = 512;
  constexpr uint32_t kIdesc = make_idesc_bf16(256, 256) | (A_MN ? 1u << 15 : 0u) | (B_MN ? 1u << 16 : 0u);

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kOffBar);
  uint64_t* full = bars;
  uint64_t* empty = bars + kStages;
  uint64_t* tail_full = bars + 2 * kStages;   // a contraction's ragged end landed (per CTA) ...
  uint64_t* tail_ready = bars + 3 * kStages;  // ... and is cleared in both CTAs (even CTA)
  uint64_t* tmem_full = bars + 4 * kStages;
  uint64_t* tmem_empty = bars + 4 * kStages + 2;
  uint32_t* tmem_ptr = reinterpret_cast<uint32_t*>(bars + 4 * kStages + 4);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_ptr + 1);
  Sched& s = *reinterpret_cast<Sched*>(smem + kOffSched);

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
  const int lane = threadIdx.x & 31;
  const int rank = static_cast<int>(cluster_cta_rank());
  const int unit = blockIdx.x >> 1, n_units = gridDim.x >> 1;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
      mbar_init(&tail_full[i], 1);
      mbar_init(&tail_ready[i], 2);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tmem_full[a], 1);
      mbar_init(&tmem_empty[a], 16);
    }
    *abort_flag = 0;
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
      int tiles = ((at - before + 255) >> 8) * p.n_tiles;  // of expert e - 1
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
  const int total = WGRAD ? p.E * p.m_tiles * p.n_tiles : s.tiles[p.E];
  const int k_slabs_fixed = WGRAD ? 0 : (p.k + 63) >> 6;

  if (warp == 0 || warp == 3) {
    // ------------------------------------------------------------ producers
    const bool leader = elect_one();
    const bool is_a = warp == 0;
    const CUtensorMap* map = is_a ? &a_map : &b_map;
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int tile = unit; tile < total && ok; tile += n_units) {
      const Tile t = decode_tile<WGRAD>(p, s, tile);
      const int slabs = WGRAD ? (t.rows + 63) >> 6 : k_slabs_fixed;
      const int out0 = (is_a ? (WGRAD ? t.m0 : t.row0) : t.n0) + rank * 128;  // first of this CTA's 128 outputs
      for (int kb = 0; kb < slabs; ++kb) {
        if (!mbar_wait(&empty[stage], phase ^ 1u, abort_flag, p.status, 41)) { ok = false; break; }
        uint8_t* dst = smem + stage * kStage + (is_a ? 0 : kOperand);
        const bool ragged = WGRAD && kb == slabs - 1 && (t.rows & 15) != 0;
        if (leader) {
          uint64_t* bar = &full[stage];
          if (ragged) {
            bar = &tail_full[stage];
            if (is_a) {
              mbar_expect_tx(bar, kStage);
              if (rank == 0) mbar_arrive(&full[stage]);
            }
          } else if (is_a && rank == 0) {
            mbar_expect_tx(bar, 2 * kStage);
          }
          if constexpr (WGRAD) {
            const int r = t.row0 + kb * 64;
            if (ragged) {
              tma_load_2d(dst, map, out0, r, bar);
              tma_load_2d(dst + 8192, map, out0 + 64, r, bar);
            } else {
              tma2_load_2d(dst, map, out0, r, bar);
              tma2_load_2d(dst + 8192, map, out0 + 64, r, bar);
            }
          } else if (is_a) {
            tma2_load_2d(dst, map, kb * 64, out0, bar);
          } else if constexpr (B_MN) {
            tma2_load_3d(dst, map, out0, kb * 64, t.expert, bar);
            tma2_load_3d(dst + 8192, map, out0 + 64, kb * 64, t.expert, bar);
          } else {
            tma2_load_3d(dst, map, kb * 64, out0, t.expert, bar);
          }
        }
        if (++stage == kStages) { stage = 0; phase ^= 1u; }
      }
    }
    if (!ok) {
      // let copies already in flight land before the CTA retires
      for (int i = 0; i < 2000; ++i) __nanosleep(1000);
    }
  } else if (warp == 1 && rank == 0) {
    // ------------------------------------------------------------ MMA issuer
    const bool leader = elect_one();
    int stage = 0, it = 0;
    uint32_t phase = 0, tail_phase = 0;
    bool ok = true;
    for (int tile = unit; tile < total && ok; tile += n_units) {
      int rows = 0, slabs = k_slabs_fixed, last = ((p.k + 15) >> 4) - 4 * (slabs - 1);
      if constexpr (WGRAD) {
        const int e = tile / (p.m_tiles * p.n_tiles);
        rows = s.first[e + 1] - s.first[e];
        if (rows == 0) continue;
        slabs = (rows + 63) >> 6;
        last = ((rows + 15) >> 4) - 4 * (slabs - 1);
      }
      const int acc = it & 1;
      if (!mbar_wait(&tmem_empty[acc], ((it >> 1) & 1) ^ 1u, abort_flag, p.status, 42)) break;
      tc_fence_after();
      const uint32_t d_tmem = tmem_base + acc * 256;
      for (int kb = 0; kb < slabs; ++kb) {
        if (!mbar_wait(&full[stage], phase, abort_flag, p.status, 43)) { ok = false; break; }
        if (WGRAD && kb == slabs - 1 && (rows & 15) != 0) {
          if (!mbar_wait_cluster(&tail_ready[stage], (tail_phase >> stage) & 1u, abort_flag, p.status, 44)) { ok = false; break; }
          tail_phase ^= 1u << stage;
        }
        tc_fence_after();
        const uint32_t sa = smem_u32(smem + stage * kStage), sb = sa + kOperand;
        const uint64_t a_desc = A_MN ? desc_sw128_mn(sa) : desc_sw128(sa);
        const uint64_t b_desc = B_MN ? desc_sw128_mn(sb) : desc_sw128(sb);
        if (leader) {
          const int steps = kb == slabs - 1 ? last : 4;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if (k < steps)  // 16 contraction steps: 32 bytes along a K-major row, 16 rows of an MN-major tile
              tc2_mma_bf16(d_tmem, a_desc + k * (A_MN ? 128 : 2), b_desc + k * (B_MN ? 128 : 2), kIdesc, (kb | k) != 0);
          }
          tc2_commit_pair(&empty[stage]);
        }
        if (++stage == kStages) { stage = 0; phase ^= 1u; }
      }
      if (ok && leader) tc2_commit_pair(&tmem_full[acc]);
      ++it;
    }
  } else if (WGRAD && warp == 2) {
    // ------------------------------------------------------------ ragged ends
    int stage = 0;
    uint32_t tail_phase = 0;
    bool ok = true;
    for (int tile = unit; tile < total && ok; tile += n_units) {
      const int e = tile / (p.m_tiles * p.n_tiles);
      const int rows = s.first[e + 1] - s.first[e];
      const int slabs = (rows + 63) >> 6;
      const int at = (stage + slabs - 1) % kStages;
      if ((rows & 15) != 0) {
        if (!mbar_wait(&tail_full[at], (tail_phase >> at) & 1u, abort_flag, p.status, 45)) { ok = false; break; }
        tail_phase ^= 1u << at;
        const int from = (rows - 1) % 64 + 1, to = (from + 15) & ~15;  // rows of the slab to clear
        uint8_t* base = smem + at * kStage;
        // four boxes (two of either operand) of 64 rows of 128 bytes: 32 lanes clear 512 bytes of a row
        for (int r = from; r < to; ++r)
          *reinterpret_cast<uint4*>(base + (lane >> 3) * 8192 + r * 128 + (lane & 7) * 16) = make_uint4(0, 0, 0, 0);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive_leader(&tail_ready[at]);
      }
      stage = (stage + slabs) % kStages;
    }
  } else if (warp >= 4) {
    // ------------------------------------------------------------ epilogue
    const int q = warp & 3, half = (warp - 4) >> 2;
    const int lane_row = rank * 128 + q * 32 + lane;
    int it = 0;
    if constexpr (!WGRAD) {
      // rows of no expert
      const int lo = s.first[0], hi = s.first[p.E], none = lo + p.R - hi;
      for (int i = blockIdx.x * 8 + warp - 4; i < none; i += gridDim.x * 8) {
        uint4* row = reinterpret_cast<uint4*>(p.out + static_cast<int64_t>(i < lo ? i : i - lo + hi) * p.n);
        for (int c = lane; c < p.n >> 3; c += 32) row[c] = make_uint4(0, 0, 0, 0);
      }
    }
    for (int tile = unit; tile < total; tile += n_units) {
      const Tile t = decode_tile<WGRAD>(p, s, tile);
      const bool live = WGRAD ? t.m0 + lane_row < p.m : lane_row < t.rows;
      const int64_t out_row = WGRAD ? static_cast<int64_t>(t.expert) * p.m + t.m0 + lane_row : t.row0 + lane_row;
      const int c0 = t.n0 + half * 128;
      __nv_bfloat16* out = p.out + out_row * p.n + c0;
      const int cols = min(128, p.n - c0);
      const bool empty_tile = WGRAD && t.rows == 0;
      const int acc = it & 1;
      if (!empty_tile) {
        if (!mbar_wait(&tmem_full[acc], (it >> 1) & 1, abort_flag, p.status, 46)) break;
        __syncwarp();
        tc_fence_after();
        ++it;
      }
      const uint32_t taddr = tmem_base + acc * 256 + half * 128 + (static_cast<uint32_t>(q * 32) << 16);
#pragma unroll
      for (int c = 0; c < 128; c += 32) {
        uint32_t v[32];
        if (empty_tile) {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = 0;
        } else {
          tc_ld32_nowait(taddr + c, v);
          tc_wait_ld();
        }
        if (live) {
          uint32_t w[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const __nv_bfloat162 b = __floats2bfloat162_rn(__uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1]));
            w[j] = *reinterpret_cast<const uint32_t*>(&b);
          }
          if (p.wide_stores) {  // n and with it every part that is left is a multiple of 16 columns
#pragma unroll
            for (int j = 0; j < 2; ++j)
              if (c + j * 16 < cols)
                st_global_256(out + c + j * 16, w[8 * j], w[8 * j + 1], w[8 * j + 2], w[8 * j + 3], w[8 * j + 4],
                              w[8 * j + 5], w[8 * j + 6], w[8 * j + 7]);
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (c + j * 8 < cols)
                *reinterpret_cast<uint4*>(out + c + j * 8) = make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
          }
        }
        __syncwarp();  // the next load wants the whole warp
      }
      if (!empty_tile) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_leader_relaxed(&tmem_empty[acc]);
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // the peer may still read this CTA's shared memory until here
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(kTmemCols) : "memory");
  }
}

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

template <bool WGRAD, bool B_MN>
int launch(const CUtensorMap& a, const CUtensorMap& b, const Params& p, int64_t tiles, cudaStream_t st) {
  auto kern = expert_linear_kernel<WGRAD, B_MN>;
  B200MOE_CUDA_OK(ensure_dynamic_smem(reinterpret_cast<const void*>(kern), kSmem));
  const int64_t units = sm_count() / 2;
  B200MOE_CUDA_OK(launch_overlapped(kern, dim3(static_cast<unsigned>(2 * (tiles < units ? tiles : units))), kThreads, kSmem,
                                    st, a, b, p));
  B200MOE_LAUNCH_OK("expert_linear_kernel");
  return B200MOE_OK;
}

bool rows_ok(const void* p, int64_t pitch, int cols) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && pitch % 8 == 0 && pitch >= cols && pitch < (int64_t{1} << 38);
}

}  // namespace
}  // namespace b200moe

using namespace b200moe;

extern "C" int b200moe_expert_product(const void* rows_bf16, int64_t rows_pitch, const void* weight_bf16, int64_t w_pitch,
                                      int64_t w_expert_pitch, int contract_last, const int32_t* expert_offsets, int R, int E,
                                      int D0, int D1, void* out_bf16, int32_t* status, b200moe_stream_t stream) {
  B200MOE_REQUIRE(rows_bf16 && weight_bf16 && expert_offsets && out_bf16 && status, B200MOE_ERR_INVALID,
                  "expert_product: null pointer argument");
  B200MOE_REQUIRE(R > 0 && E > 0 && E <= kMaxExperts, B200MOE_ERR_INVALID,
                  "expert_product: need at least one row and between 1 and %d experts", kMaxExperts);
  B200MOE_REQUIRE(D0 > 0 && D1 > 0 && D0 % 8 == 0 && D1 % 8 == 0, B200MOE_ERR_INVALID,
                  "expert_product: both sizes of a weight matrix must be positive multiples of 8, got %d x %d", D0, D1);
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
  p.n = n;
  p.k = k;
  p.n_tiles = (n + 255) / 256;
  p.out = static_cast<__nv_bfloat16*>(out_bf16);
  p.wide_stores = n % 16 == 0 && (reinterpret_cast<uintptr_t>(out_bf16) & 31) == 0;
  p.status = status;
  const int64_t most_tiles = (ceil_div64(R, 256) + (E < R ? E : R)) * p.n_tiles;
  B200MOE_REQUIRE(most_tiles < (int64_t{1} << 30), B200MOE_ERR_INVALID, "expert_product: too many output tiles");
  CUtensorMap a, b;
  int rc = make_map(&a, rows_bf16, k, R, rows_pitch, 0, 0, 128);
  if (rc != B200MOE_OK) return rc;
  rc = make_map(&b, weight_bf16, D1, D0, w_pitch, E, w_expert_pitch, contract_last ? 128 : 64);
  if (rc != B200MOE_OK) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return contract_last ? launch<false, false>(a, b, p, most_tiles, st) : launch<false, true>(a, b, p, most_tiles, st);
}

extern "C" int b200moe_expert_weight_grad(const void* a_bf16, int64_t a_pitch, const void* b_bf16, int64_t b_pitch,
                                          const int32_t* expert_offsets, int R, int E, int M, int N, void* out_bf16,
                                          int32_t* status, b200moe_stream_t stream) {
  B200MOE_REQUIRE(a_bf16 && b_bf16 && expert_offsets && out_bf16 && status, B200MOE_ERR_INVALID,
                  "expert_weight_grad: null pointer argument");
  B200MOE_REQUIRE(R > 0 && E > 0 && E <= kMaxExperts, B200MOE_ERR_INVALID,
                  "expert_weight_grad: need at least one row and between 1 and %d experts", kMaxExperts);
  B200MOE_REQUIRE(M > 0 && N > 0 && M % 8 == 0 && N % 8 == 0, B200MOE_ERR_INVALID,
                  "expert_weight_grad: both sizes of a weight matrix must be positive multiples of 8, got %d x %d", M, N);
  B200MOE_REQUIRE(rows_ok(a_bf16, a_pitch, M) && rows_ok(b_bf16, b_pitch, N), B200MOE_ERR_INVALID,
                  "expert_weight_grad: rows must start on 16-byte boundaries");
  B200MOE_REQUIRE((reinterpret_cast<uintptr_t>(out_bf16) & 15) == 0, B200MOE_ERR_INVALID,
                  "expert_weight_grad: out must be 16-byte aligned");
  Params p{};
  p.offsets = expert_offsets;
  p.R = R;
  p.E = E;
  p.m = M;
  p.n = N;
  p.m_tiles = (M + 255) / 256;
  p.n_tiles = (N + 255) / 256;
  p.out = static_cast<__nv_bfloat16*>(out_bf16);
  p.wide_stores = N % 16 == 0 && (reinterpret_cast<uintptr_t>(out_bf16) & 31) == 0;
  p.status = status;
  const int64_t tiles = static_cast<int64_t>(E) * p.m_tiles * p.n_tiles;
  B200MOE_REQUIRE(tiles < (int64_t{1} << 30), B200MOE_ERR_INVALID, "expert_weight_grad: too many output tiles");
  CUtensorMap a, b;
  int rc = make_map(&a, a_bf16, M, R, a_pitch, 0, 0, 64);
  if (rc != B200MOE_OK) return rc;
  rc = make_map(&b, b_bf16, N, R, b_pitch, 0, 0, 64);
  if (rc != B200MOE_OK) return rc;
  return launch<true, true>(a, b, p, tiles, static_cast<cudaStream_t>(stream));
}
