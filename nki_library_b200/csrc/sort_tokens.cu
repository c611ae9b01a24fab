// Tokens sorted by expert and back: the order of the (token, choice) pairs, the rows in that order, the weighted sum that
// brings the experts' rows back to their tokens, and the gradients of both.
//
// A pair p = t * K + k goes to row (pairs of smaller experts) + (earlier pairs of the same expert); pairs whose id lies
// outside [0, E) get none.  Nothing but counts decides a place, so the order is the same in every run; two equal ids of one
// token are two rows.
#include "common.cuh"
#include "quantize_row.cuh"

namespace b200moe {
namespace {

constexpr int kMaxExperts = 1024;
constexpr int kChunk = 2048;  // pairs per CTA of the sort
constexpr int kSortThreads = 256;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kSpan = kChunk / kSortWarps;  // consecutive pairs of a warp

struct SortArgs {
  const void* index;
  int wide;  // 64-bit ids
  int64_t pairs;
  int E;
};

__device__ __forceinline__ int expert_of(const SortArgs& a, int64_t p) {
  if (p >= a.pairs) return -1;
  const int64_t e = a.wide ? static_cast<const int64_t*>(a.index)[p] : static_cast<const int32_t*>(a.index)[p];
  return e >= 0 && e < a.E ? static_cast<int>(e) : -1;
}

// hist[w * E + e] = pairs of expert e among warp w's.
__device__ __forceinline__ void count_pairs(const SortArgs& a, int64_t p0, int* hist) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = threadIdx.x; i < kSortWarps * a.E; i += kSortThreads) hist[i] = 0;
  __syncthreads();
  for (int i = 0; i < kSpan; i += 32) {
    const int e = expert_of(a, p0 + warp * kSpan + i + lane);
    const unsigned same = __match_any_sync(0xffffffffu, e);
    if (e >= 0 && lane == __ffs(same) - 1) hist[warp * a.E + e] += __popc(same);
    __syncwarp();
  }
  __syncthreads();
}

__global__ void __launch_bounds__(kSortThreads) count_pairs_kernel(SortArgs a, int* chunk_counts) {
  extern __shared__ int hist[];
  grid_enter(a.index);
  count_pairs(a, static_cast<int64_t>(blockIdx.x) * kChunk, hist);
  for (int e = threadIdx.x; e < a.E; e += kSortThreads) {
    int n = 0;
#pragma unroll
    for (int w = 0; w < kSortWarps; ++w) n += hist[w * a.E + e];
    chunk_counts[static_cast<int64_t>(blockIdx.x) * a.E + e] = n;
  }
}

// Every CTA adds the chunks' counts up for itself: its own base per expert costs no third launch.
__global__ void __launch_bounds__(kSortThreads) place_pairs_kernel(SortArgs a, const int* chunk_counts, int32_t* offsets,
                                                                   int32_t* row_of_pair, int32_t* pair_of_row) {
  extern __shared__ int hist[];  // [kSortWarps][E], then base [E]
  __shared__ int s_warp[kSortWarps];
  grid_enter(a.index, chunk_counts);
  int* base = hist + kSortWarps * a.E;
  const int64_t p0 = static_cast<int64_t>(blockIdx.x) * kChunk;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int chunks = gridDim.x;
  count_pairs(a, p0, hist);
  int run = 0;  // rows of the experts before this round's
  for (int e0 = 0; e0 < a.E; e0 += kSortThreads) {
    const int e = e0 + threadIdx.x;
    int before = 0, total = 0;
    if (e < a.E) {
      if (chunks == 1) {
#pragma unroll
        for (int w = 0; w < kSortWarps; ++w) total += hist[w * a.E + e];
      } else {
#pragma unroll 8
        for (int c = 0; c < chunks; ++c) {
          const int n = chunk_counts[static_cast<int64_t>(c) * a.E + e];
          before += c < static_cast<int>(blockIdx.x) ? n : 0;
          total += n;
        }
      }
    }
    int scan = total;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, scan, o);
      if (lane >= o) scan += u;
    }
    if (lane == 31) s_warp[warp] = scan;
    __syncthreads();
    int first = run + scan - total;
    for (int w = 0; w < kSortWarps; ++w) {
      if (w < warp) first += s_warp[w];
      run += s_warp[w];
    }
    if (e < a.E) {
      if (blockIdx.x == 0) offsets[e] = first;
      base[e] = first + before;
    }
    __syncthreads();
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) offsets[a.E] = run;
  // a warp's part of an expert follows those of the warps before it
  for (int e = threadIdx.x; e < a.E; e += kSortThreads) {
    int at = base[e];
#pragma unroll
    for (int w = 0; w < kSortWarps; ++w) {
      const int n = hist[w * a.E + e];
      hist[w * a.E + e] = at;
      at += n;
    }
  }
  __syncthreads();
  for (int i = 0; i < kSpan; i += 32) {
    const int64_t p = p0 + warp * kSpan + i + lane;
    const int e = expert_of(a, p);
    const unsigned same = __match_any_sync(0xffffffffu, e);
    const int at = e >= 0 ? hist[warp * a.E + e] : -1;
    const int row = e >= 0 ? at + __popc(same & ((1u << lane) - 1u)) : -1;
    __syncwarp();
    if (e >= 0 && lane == __ffs(same) - 1) hist[warp * a.E + e] = at + __popc(same);
    __syncwarp();
    if (p < a.pairs) {
      row_of_pair[p] = row;
      if (row >= 0) pair_of_row[row] = static_cast<int32_t>(p);
      if (p >= run) pair_of_row[p] = -1;
    }
  }
}

// ------------------------------------------------------------------ rows
// T elements, V at once: 16 bytes, or one element where rows are not made of whole aligned 16 bytes.
template <typename T, int V>
__device__ __forceinline__ void load(const T* p, float (&v)[V]) {
  if constexpr (V == 1) v[0] = static_cast<float>(*p);
  else if constexpr (sizeof(T) == 2) unpack8_bf16(*reinterpret_cast<const uint4*>(p), v);
  else {
    const float4 f = *reinterpret_cast<const float4*>(p);
    v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
  }
}
template <typename T, int V>
__device__ __forceinline__ void store(T* p, const float (&v)[V]) {
  if constexpr (V == 1) *p = static_cast<T>(v[0]);
  else if constexpr (sizeof(T) == 2) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&b);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  } else *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
}

struct RowArgs {
  int T, K, H, E;
  const int32_t* row_of_pair;
  const int32_t* offsets;
  // Row of the token's k-th pair, -1 if it has none.
  __device__ __forceinline__ int64_t row(int64_t t, int k) const {
    const int r = row_of_pair[t * K + k];
    return r < static_cast<int64_t>(T) * K ? r : -1;
  }
};

// The K rows that a token's CTA clears if they lie behind the last expert's: rows t * K to t * K + K - 1.
template <typename T, int V>
__device__ __forceinline__ void clear_rows_behind(const RowArgs& a, T* rows) {
  const int64_t r0 = static_cast<int64_t>(blockIdx.x) * a.K;
  const float zero[V] = {};
  for (int64_t r = max(r0, static_cast<int64_t>(a.offsets[a.E])); r < r0 + a.K; ++r)
    for (int h = (blockIdx.y * blockDim.x + threadIdx.x) * V; h < a.H; h += gridDim.y * blockDim.x * V) store<T, V>(rows + r * a.H + h, zero);
}

// rows[row_of_pair[t, k]] = hidden[t]
template <typename T, int V>
__global__ void __launch_bounds__(128) sort_rows_kernel(RowArgs a, const T* hidden, int64_t pitch, T* rows) {
  grid_enter(a.row_of_pair, a.offsets, hidden);
  const int64_t t = blockIdx.x;
  for (int h = (blockIdx.y * blockDim.x + threadIdx.x) * V; h < a.H; h += gridDim.y * blockDim.x * V) {
    float v[V];
    load<T, V>(hidden + t * pitch + h, v);
    for (int k = 0; k < a.K; ++k) {
      const int64_t r = a.row(t, k);
      if (r >= 0) store<T, V>(rows + r * a.H + h, v);
    }
  }
  clear_rows_behind<T, V>(a, rows);
}

// out[t] = sum over k of (affinities[t, k]) rows[row_of_pair[t, k]], in fp32, k ascending, rounded once
template <typename T, int V>
__global__ void __launch_bounds__(128) unsort_rows_kernel(RowArgs a, const T* rows, int64_t pitch, const void* affinities,
                                                          int aff_dtype, T* out) {
  grid_enter(a.row_of_pair, rows, affinities);
  const int64_t t = blockIdx.x;
  for (int h = (blockIdx.y * blockDim.x + threadIdx.x) * V; h < a.H; h += gridDim.y * blockDim.x * V) {
    float sum[V] = {};
    for (int k = 0; k < a.K; ++k) {
      const int64_t r = a.row(t, k);
      if (r < 0) continue;
      const float w = affinities != nullptr ? load_as_float(affinities, t * a.K + k, aff_dtype) : 1.0f;
      float v[V];
      load<T, V>(rows + r * pitch + h, v);
#pragma unroll
      for (int i = 0; i < V; ++i) sum[i] = fmaf(w, v[i], sum[i]);
    }
    store<T, V>(out + t * a.H + h, sum);
  }
}

// d rows[r] = a[t, k] d out[t]; d a[t, k] = <d out[t], rows[r]>
template <typename T, int V>
__global__ void __launch_bounds__(256) unsort_backward_kernel(RowArgs a, const T* d_out, int64_t d_pitch, const T* rows,
                                                              int64_t pitch, const void* affinities, int aff_dtype,
                                                              T* d_rows, void* d_affinities) {
  __shared__ float s_dot[8][8];
  grid_enter(a.row_of_pair, a.offsets, d_out, rows, affinities);
  const int64_t t = blockIdx.x;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int k0 = 0; k0 < a.K; k0 += 8) {
    const int n = min(8, a.K - k0);
    int64_t r[8];
    float w[8], dot[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      r[j] = j < n ? a.row(t, k0 + j) : -1;
      w[j] = j < n && affinities != nullptr ? load_as_float(affinities, t * a.K + k0 + j, aff_dtype) : 1.0f;
      dot[j] = 0.f;
    }
    for (int h = threadIdx.x * V; h < a.H; h += blockDim.x * V) {
      float d[V];
      load<T, V>(d_out + t * d_pitch + h, d);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (r[j] < 0) continue;
        if (d_rows != nullptr) {
          float v[V];
#pragma unroll
          for (int i = 0; i < V; ++i) v[i] = w[j] * d[i];
          store<T, V>(d_rows + r[j] * a.H + h, v);
        }
        if (d_affinities != nullptr) {
          float v[V];
          load<T, V>(rows + r[j] * pitch + h, v);
#pragma unroll
          for (int i = 0; i < V; ++i) dot[j] = fmaf(d[i], v[i], dot[j]);
        }
      }
    }
    if (d_affinities != nullptr) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float s = dot[j];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (lane == 0) s_dot[warp][j] = s;
      }
      __syncthreads();
      if (threadIdx.x < static_cast<unsigned>(n)) {
        float s = 0.f;
        for (int i = 0; i < static_cast<int>(blockDim.x >> 5); ++i) s += s_dot[i][threadIdx.x];
        store_from_float(d_affinities, t * a.K + k0 + threadIdx.x, aff_dtype, s);
      }
      __syncthreads();
    }
  }
  if (d_rows != nullptr) clear_rows_behind<T, V>(a, d_rows);
}

bool whole_vectors(const void* p, int64_t pitch_bytes) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && pitch_bytes % 16 == 0;
}

// CTAs over a token's columns: one once the tokens alone give every SM several.
int column_parts(int T, int H, int width) {
  const int parts = (H - 1) / (128 * width) + 1;
  return T >= 8 * sm_count() ? 1 : (parts < 65535 ? parts : 65535);
}

int check_rows(const char* name, int dtype, int T, int K, int H, int64_t pitch) {
  B200MOE_REQUIRE(dtype == B200MOE_F32 || dtype == B200MOE_BF16, B200MOE_ERR_INVALID, "%s: rows must be fp32 or bf16", name);
  B200MOE_REQUIRE(T > 0 && K > 0 && H > 0 && static_cast<int64_t>(T) * K <= INT32_MAX, B200MOE_ERR_INVALID,
                  "%s: need T, K, H > 0 and at most 2^31 - 1 pairs", name);
  B200MOE_REQUIRE(pitch >= 0, B200MOE_ERR_INVALID, "%s: negative row pitch", name);
  return B200MOE_OK;
}

// Calls fn with a value of the element type and the vector width as compile-time constants.
template <typename F>
int with_rows(int dtype, bool wide, const F& fn) {
  using std::integral_constant;
  if (dtype == B200MOE_BF16) {
    if (wide) return fn(__nv_bfloat16{}, integral_constant<int, 8>{});
    return fn(__nv_bfloat16{}, integral_constant<int, 1>{});
  }
  if (wide) return fn(float{}, integral_constant<int, 4>{});
  return fn(float{}, integral_constant<int, 1>{});
}

}  // namespace
}  // namespace b200moe

using namespace b200moe;

extern "C" size_t b200moe_sort_workspace_bytes(int64_t pairs, int E) {
  if (pairs <= kChunk || E <= 0) return 0;
  return static_cast<size_t>(ceil_div64(pairs, kChunk)) * E * sizeof(int);
}

extern "C" int b200moe_sort_pairs(const void* expert_index, int index_bytes, int T, int K, int E, int32_t* expert_offsets,
                                  int32_t* row_of_pair, int32_t* pair_of_row, void* workspace, size_t workspace_bytes,
                                  b200moe_stream_t stream) {
  B200MOE_REQUIRE(expert_index && expert_offsets && row_of_pair && pair_of_row, B200MOE_ERR_INVALID,
                  "sort_pairs: null pointer argument");
  B200MOE_REQUIRE(index_bytes == 4 || index_bytes == 8, B200MOE_ERR_INVALID, "sort_pairs: ids must have 4 or 8 bytes");
  B200MOE_REQUIRE(T > 0 && K > 0 && static_cast<int64_t>(T) * K <= INT32_MAX, B200MOE_ERR_INVALID,
                  "sort_pairs: need T, K > 0 and at most 2^31 - 1 pairs");
  B200MOE_REQUIRE(E > 0 && E <= kMaxExperts, B200MOE_ERR_INVALID, "sort_pairs: between 1 and %d experts, got %d", kMaxExperts, E);
  const SortArgs a{expert_index, index_bytes == 8, static_cast<int64_t>(T) * K, E};
  const int64_t chunks = ceil_div64(a.pairs, kChunk);
  B200MOE_REQUIRE(chunks == 1 || (workspace != nullptr && workspace_bytes >= b200moe_sort_workspace_bytes(a.pairs, E)),
                  B200MOE_ERR_WORKSPACE, "sort_pairs: workspace too small");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const size_t hist = static_cast<size_t>(kSortWarps) * E * sizeof(int);
  const dim3 grid(static_cast<unsigned>(chunks));
  if (chunks > 1) {
    B200MOE_CUDA_OK(launch_overlapped(count_pairs_kernel, grid, kSortThreads, hist, st, a, static_cast<int*>(workspace)));
    B200MOE_LAUNCH_OK("count_pairs_kernel");
  }
  B200MOE_CUDA_OK(launch_overlapped(place_pairs_kernel, grid, kSortThreads, hist + E * sizeof(int), st, a,
                                    static_cast<const int*>(workspace), expert_offsets, row_of_pair, pair_of_row));
  B200MOE_LAUNCH_OK("place_pairs_kernel");
  return B200MOE_OK;
}

extern "C" int b200moe_sort_rows(const void* hidden, int dtype, int64_t pitch, int T, int K, int H, int E,
                                 const int32_t* row_of_pair, const int32_t* expert_offsets, void* rows,
                                 b200moe_stream_t stream) {
  B200MOE_REQUIRE(hidden && row_of_pair && expert_offsets && rows, B200MOE_ERR_INVALID, "sort_rows: null pointer argument");
  int rc = check_rows("sort_rows", dtype, T, K, H, pitch);
  if (rc != B200MOE_OK) return rc;
  B200MOE_REQUIRE(E > 0 && E <= kMaxExperts, B200MOE_ERR_INVALID, "sort_rows: between 1 and %d experts, got %d", kMaxExperts, E);
  const RowArgs a{T, K, H, E, row_of_pair, expert_offsets};
  const int size = dtype == B200MOE_F32 ? 4 : 2;
  const bool wide = whole_vectors(hidden, pitch * size) && whole_vectors(rows, static_cast<int64_t>(H) * size);
  return with_rows(dtype, wide, [&](auto element, auto width) -> int {
    using E_ = decltype(element);
    constexpr int V = decltype(width)::value;
    const int parts = column_parts(T, H, V);
    B200MOE_CUDA_OK(launch_overlapped(sort_rows_kernel<E_, V>, dim3(T, parts), 128, 0, static_cast<cudaStream_t>(stream), a,
                                      static_cast<const E_*>(hidden), pitch, static_cast<E_*>(rows)));
    B200MOE_LAUNCH_OK("sort_rows_kernel");
    return B200MOE_OK;
  });
}

extern "C" int b200moe_unsort_rows(const void* rows, int dtype, int64_t pitch, int T, int K, int H,
                                   const int32_t* row_of_pair, const void* affinities, int aff_dtype, void* out,
                                   b200moe_stream_t stream) {
  B200MOE_REQUIRE(rows && row_of_pair && out, B200MOE_ERR_INVALID, "unsort_rows: null pointer argument");
  int rc = check_rows("unsort_rows", dtype, T, K, H, pitch);
  if (rc != B200MOE_OK) return rc;
  B200MOE_REQUIRE(affinities == nullptr || aff_dtype == B200MOE_F32 || aff_dtype == B200MOE_BF16, B200MOE_ERR_INVALID,
                  "unsort_rows: affinities must be fp32 or bf16");
  const RowArgs a{T, K, H, 0, row_of_pair, nullptr};
  const int size = dtype == B200MOE_F32 ? 4 : 2;
  const bool wide = whole_vectors(rows, pitch * size) && whole_vectors(out, static_cast<int64_t>(H) * size);
  return with_rows(dtype, wide, [&](auto element, auto width) -> int {
    using E_ = decltype(element);
    constexpr int V = decltype(width)::value;
    const int parts = column_parts(T, H, V);
    B200MOE_CUDA_OK(launch_overlapped(unsort_rows_kernel<E_, V>, dim3(T, parts), 128, 0, static_cast<cudaStream_t>(stream), a,
                                      static_cast<const E_*>(rows), pitch, affinities, aff_dtype, static_cast<E_*>(out)));
    B200MOE_LAUNCH_OK("unsort_rows_kernel");
    return B200MOE_OK;
  });
}

extern "C" int b200moe_unsort_rows_backward(const void* d_out, int64_t d_pitch, const void* rows, int64_t pitch, int dtype,
                                            int T, int K, int H, int E, const int32_t* row_of_pair,
                                            const int32_t* expert_offsets, const void* affinities, int aff_dtype,
                                            void* d_rows, void* d_affinities, b200moe_stream_t stream) {
  B200MOE_REQUIRE(d_out && row_of_pair && expert_offsets && (d_rows || d_affinities), B200MOE_ERR_INVALID,
                  "unsort_rows_backward: null pointer argument");
  B200MOE_REQUIRE(d_affinities == nullptr || (rows && affinities), B200MOE_ERR_INVALID,
                  "unsort_rows_backward: the affinities' gradient needs rows and affinities");
  int rc = check_rows("unsort_rows_backward", dtype, T, K, H, pitch);
  if (rc == B200MOE_OK) rc = check_rows("unsort_rows_backward", dtype, T, K, H, d_pitch);
  if (rc != B200MOE_OK) return rc;
  B200MOE_REQUIRE(affinities == nullptr || aff_dtype == B200MOE_F32 || aff_dtype == B200MOE_BF16, B200MOE_ERR_INVALID,
                  "unsort_rows_backward: affinities must be fp32 or bf16");
  B200MOE_REQUIRE(E > 0 && E <= kMaxExperts, B200MOE_ERR_INVALID, "unsort_rows_backward: between 1 and %d experts, got %d",
                  kMaxExperts, E);
  const RowArgs a{T, K, H, E, row_of_pair, expert_offsets};
  const int size = dtype == B200MOE_F32 ? 4 : 2;
  const bool wide = whole_vectors(d_out, d_pitch * size) && (rows == nullptr || whole_vectors(rows, pitch * size)) &&
                    (d_rows == nullptr || whole_vectors(d_rows, static_cast<int64_t>(H) * size)) &&
                    static_cast<int64_t>(H) * size % 16 == 0;
  return with_rows(dtype, wide, [&](auto element, auto width) -> int {
    using E_ = decltype(element);
    constexpr int V = decltype(width)::value;
    B200MOE_CUDA_OK(launch_overlapped(unsort_backward_kernel<E_, V>, dim3(T), 256, 0, static_cast<cudaStream_t>(stream), a,
                                      static_cast<const E_*>(d_out), d_pitch, static_cast<const E_*>(rows), pitch, affinities,
                                      aff_dtype, static_cast<E_*>(d_rows), d_affinities));
    B200MOE_LAUNCH_OK("unsort_backward_kernel");
    return B200MOE_OK;
  });
}
