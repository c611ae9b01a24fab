// Tokens sorted by expert and back: the order of the (token, choice) pairs, the rows in that order, the weighted sum that
// brings the experts' rows back to their tokens, and the gradients of both.
//
// A pair p = t * K + k goes to row (pairs of smaller experts) + (earlier pairs of the same expert); pairs whose id lies
// outside [0, E) get none.  Nothing but counts decides a place, so the order is the same in every run; two equal ids of one
// token are two rows.
#include "common.cuh"
#include "quantize_row.cuh"

#include <initializer_list>
#include <type_traits>

namespace b200moe {
namespace {

constexpr int kMaxExperts = 1024;
constexpr int kChunk = 2048;  // pairs per CTA of the sort
constexpr int kSortThreads = 512;
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

constexpr int kRounds = kSpan / 32;
constexpr int kMostHist = (kSortWarps + 1) * kMaxExperts * static_cast<int>(sizeof(int));

// How many pairs of each expert a chunk has; no order in it, so atomics on shared memory do.
__global__ void __launch_bounds__(kSortThreads) count_pairs_kernel(SortArgs a, int* chunk_counts) {
  extern __shared__ int hist[];
  grid_enter(a.index);
  int expert[kChunk / kSortThreads];
#pragma unroll
  for (int i = 0; i < kChunk / kSortThreads; ++i)
    expert[i] = expert_of(a, static_cast<int64_t>(blockIdx.x) * kChunk + i * kSortThreads + threadIdx.x);
  for (int e = threadIdx.x; e < a.E; e += kSortThreads) hist[e] = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kChunk / kSortThreads; ++i)
    if (expert[i] >= 0) atomicAdd(&hist[expert[i]], 1);
  __syncthreads();
  for (int e = threadIdx.x; e < a.E; e += kSortThreads) chunk_counts[static_cast<int64_t>(blockIdx.x) * a.E + e] = hist[e];
}

// The chunks' counts turned into sums over all chunks up to and with each: eight experts per CTA, a 128th of the chunks per
// thread.  Without it every CTA adds all chunks' counts up, whose time grows with their square; with it there is a third launch.
// Without / with, order of 8 x T pairs: T 32768 and 128 experts 26.6 / 30.6 us, 1024 experts 51 / 31; T 131072 and 8 experts 22.0 /
// 23.6, 128 44.5 / 25.1; T 1048576 and 64 experts 761 / 111.
bool scan_pays(int64_t chunks, int E) { return chunks * (E > 32 ? E : 32) > 32768; }
constexpr int kScanExperts = 8;
constexpr int kScanParts = 128;
__global__ void __launch_bounds__(kScanExperts * kScanParts) scan_counts_kernel(int* chunk_counts, int chunks, int E) {
  __shared__ int s_warp[kScanParts / 4][kScanExperts];
  grid_enter(chunk_counts);
  const int column = threadIdx.x % kScanExperts, part = threadIdx.x / kScanExperts;
  const int e = blockIdx.x * kScanExperts + column, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int per = (chunks + kScanParts - 1) / kScanParts;
  const int c0 = min(part * per, chunks), c1 = e < E ? min(c0 + per, chunks) : c0;
  int* counts = chunk_counts + e;
  int sum = 0;
#pragma unroll 16
  for (int c = c0; c < c1; ++c) sum += counts[static_cast<int64_t>(c) * E];
  int scan = sum;  // of a warp's four parts
#pragma unroll
  for (int o = kScanExperts; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, scan, o);
    if (lane >= o) scan += u;
  }
  if (lane >= 32 - kScanExperts) s_warp[warp][column] = scan;
  __syncthreads();
  int run = scan - sum;
  for (int w = 0; w < warp; ++w) run += s_warp[w][column];
  for (int c = c0; c < c1; c += 16) {
    int n[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) n[i] = c + i < c1 ? counts[static_cast<int64_t>(c + i) * E] : 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      run += n[i];
      if (c + i < c1) counts[static_cast<int64_t>(c + i) * E] = run;
    }
  }
}

// Rows of one chunk's pairs, by a whole CTA; `put(pair, row)` is called once per pair, -1 for none.  Every CTA adds the chunks'
// counts up for itself, unless they are `scanned`.  Returns the number of rows; `offsets` may be NULL.
template <typename Put>
__device__ __forceinline__ int order_chunk(const SortArgs& a, int chunk, int chunks, const int* chunk_counts, bool scanned,
                                           int* hist, int32_t* offsets, const Put& put) {
  __shared__ int s_warp[kSortWarps], s_before[kSortThreads], s_total[kSortThreads];
  int* base = hist + kSortWarps * a.E;  // hist [kSortWarps][E], then base [E]
  const int64_t p0 = static_cast<int64_t>(chunk) * kChunk;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // a lane's pairs, its lanes of equal expert in each round, and hist[w * E + e] = pairs of expert e among warp w's
  int expert[kRounds];
  unsigned same[kRounds];
#pragma unroll
  for (int i = 0; i < kRounds; ++i) expert[i] = expert_of(a, p0 + warp * kSpan + i * 32 + lane);
  for (int i = threadIdx.x; i < kSortWarps * a.E; i += kSortThreads) hist[i] = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kRounds; ++i) {
    const int e = expert[i];
    same[i] = __match_any_sync(0xffffffffu, e);
    if (e >= 0 && lane == __ffs(same[i]) - 1) hist[warp * a.E + e] += __popc(same[i]);
    __syncwarp();
  }
  __syncthreads();
  // `width` experts at a time, every `parts`-th chunk per thread: one memory latency for each of a thread's chunks would be the
  // whole launch (262144 pairs, 128 experts, a thread per expert: 31 us, 15 so)
  int run = 0;  // rows of the experts before e0
  const int width = min(kSortThreads, max(32, 1 << (32 - __clz(a.E - 1)))), parts = kSortThreads / width;
  const int part = threadIdx.x / width, column = threadIdx.x - part * width;
  for (int e0 = 0; e0 < a.E; e0 += width) {
    const int e = e0 + column;
    int before = 0, total = 0;
    if (e < a.E) {
      if (chunks == 1) {
        if (part == 0) {
#pragma unroll
          for (int w = 0; w < kSortWarps; ++w) total += hist[w * a.E + e];
        }
      } else if (scanned) {
        if (part == 0) {
          before = chunk > 0 ? chunk_counts[static_cast<int64_t>(chunk - 1) * a.E + e] : 0;
          total = chunk_counts[static_cast<int64_t>(chunks - 1) * a.E + e];
        }
      } else {
#pragma unroll 16
        for (int c = part; c < chunks; c += parts) {
          const int n = chunk_counts[static_cast<int64_t>(c) * a.E + e];
          before += c < chunk ? n : 0;
          total += n;
        }
      }
    }
    if (parts > 1 && chunks > 1 && !scanned) {
      s_before[threadIdx.x] = before;
      s_total[threadIdx.x] = total;
      __syncthreads();
      if (part == 0) {
        for (int i = 1; i < parts; ++i) {
          before += s_before[threadIdx.x + i * width];
          total += s_total[threadIdx.x + i * width];
        }
      } else {
        total = 0;
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
    if (part == 0 && e < a.E) {
      if (offsets != nullptr) offsets[e] = first;
      base[e] = first + before;
    }
    __syncthreads();
  }
  if (offsets != nullptr && threadIdx.x == 0) offsets[a.E] = run;
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
#pragma unroll
  for (int i = 0; i < kRounds; ++i) {
    const int64_t p = p0 + warp * kSpan + i * 32 + lane;
    const int e = expert[i];
    const int at = e >= 0 ? hist[warp * a.E + e] : -1;
    const int row = e >= 0 ? at + __popc(same[i] & ((1u << lane) - 1u)) : -1;
    __syncwarp();
    if (e >= 0 && lane == __ffs(same[i]) - 1) hist[warp * a.E + e] = at + __popc(same[i]);
    __syncwarp();
    if (p < a.pairs) put(p, row);
  }
  return run;
}

__global__ void __launch_bounds__(kSortThreads) place_pairs_kernel(SortArgs a, const int* chunk_counts, bool scanned,
                                                                   int32_t* offsets, int32_t* row_of_pair) {
  extern __shared__ int hist[];
  grid_enter(a.index, chunk_counts);
  order_chunk(a, blockIdx.x, gridDim.x, chunk_counts, scanned, hist, blockIdx.x == 0 ? offsets : nullptr,
              [&](int64_t p, int row) { row_of_pair[p] = row; });
}

// ------------------------------------------------------------------ rows
// The elements of a row that a thread holds at once, `chunk` by `chunk` of the CTA's: one unit of 16 bytes, or, where rows are
// not made of whole aligned 16 bytes, a few units of 4 or 2 bytes a CTA's width apart.
template <typename T, int UNIT>
struct Piece {
  static constexpr int kUnits = UNIT == 16 ? 1 : 4;  // eight: 252 us for that sum, 804 instead of 317 for its gradients
  static constexpr int kPer = UNIT / static_cast<int>(sizeof(T));  // elements of a unit
  static constexpr int kCount = kUnits * kPer;
  uint32_t raw[UNIT == 16 ? 4 : kUnits];

  __device__ __forceinline__ static int chunk() { return static_cast<int>(blockDim.x) * kCount; }
  // Index of the first element of unit u of the chunk that starts at h; units at H and behind do not exist.
  __device__ __forceinline__ static int index(int h, int u) {
    return h + (u * static_cast<int>(blockDim.x) + static_cast<int>(threadIdx.x)) * kPer;
  }
  // Only loads, so that a caller's next row is asked for before this one is there (shifting 2-byte units on the spot took 387 us
  // instead of 187 for the sum of 48000 rows of 5003).
  __device__ __forceinline__ void fetch(const T* row, int h, int H) {
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      if (index(h, u) >= H) {
        raw[u] = 0;
        if constexpr (UNIT == 16) raw[1] = raw[2] = raw[3] = 0;
        continue;
      }
      const T* p = row + index(h, u);
      if constexpr (UNIT == 16) {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(p));
        raw[0] = v.x; raw[1] = v.y; raw[2] = v.z; raw[3] = v.w;
      } else if constexpr (UNIT == 4) raw[u] = __ldg(reinterpret_cast<const uint32_t*>(p));
      else raw[u] = __ldg(reinterpret_cast<const uint16_t*>(p));
    }
  }
  // Zero in units that do not exist.
  __device__ __forceinline__ void values(float (&v)[kCount]) const {
    if constexpr (sizeof(T) == 2 && UNIT > 2) {
#pragma unroll
      for (int i = 0; i < kCount / 2; ++i) {
        v[2 * i] = __uint_as_float(raw[i] << 16);
        v[2 * i + 1] = __uint_as_float(raw[i] & 0xffff0000u);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kCount; ++i) v[i] = __uint_as_float(sizeof(T) == 2 ? raw[i] << 16 : raw[i]);
    }
  }
  __device__ __forceinline__ static void store(T* row, int h, int H, const float (&v)[kCount]) {
    constexpr int kWords = kCount * static_cast<int>(sizeof(T)) / 4;
    uint32_t w[kWords > 0 ? kWords : 1];
    if constexpr (UNIT > 2) {
#pragma unroll
      for (int i = 0; i < kWords; ++i) {
        if constexpr (sizeof(T) == 2) {
          const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
          w[i] = *reinterpret_cast<const uint32_t*>(&b);
        } else {
          w[i] = __float_as_uint(v[i]);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      if (index(h, u) >= H) continue;
      T* p = row + index(h, u);
      if constexpr (UNIT == 16) *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
      else if constexpr (UNIT == 4) *reinterpret_cast<uint32_t*>(p) = w[u];
      else *p = static_cast<T>(v[u]);
    }
  }
};

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

// A token belongs to a CTA, or (SHORT) to the threads of one threadIdx.y, where a row is too short for a CTA.  Two forms of each
// kernel, because an index that differs between warps costs registers (unsort of 32768 tokens, 361 and 404 us).
template <bool SHORT>
__device__ __forceinline__ int64_t own_token() {
  return SHORT ? static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y : blockIdx.x;
}

// The K rows that a token's threads clear if they lie behind the last expert's: rows t * K to t * K + K - 1.
template <typename T, int UNIT>
__device__ __forceinline__ void clear_rows_behind(const RowArgs& a, int64_t t, T* rows) {
  using P = Piece<T, UNIT>;
  const int64_t r0 = t * a.K;
  const float zero[P::kCount] = {};
  for (int64_t r = max(r0, static_cast<int64_t>(a.offsets[a.E])); r < r0 + a.K; ++r)
    for (int h = blockIdx.y * P::chunk(); h < a.H; h += gridDim.y * P::chunk()) P::store(rows + r * a.H, h, a.H, zero);
}

// rows[row_of_pair[t, k]] = hidden[t].  32768 tokens x 4096 bf16, top-8: 2.4 GB in 396 us, the copy rate.
template <typename T, int UNIT, bool SHORT>
__global__ void __launch_bounds__(128) sort_rows_kernel(RowArgs a, const T* hidden, int64_t pitch, T* rows) {
  using P = Piece<T, UNIT>;
  grid_enter(a.row_of_pair, a.offsets, hidden);
  const int64_t t = own_token<SHORT>();
  if (SHORT && t >= a.T) return;
  for (int h = blockIdx.y * P::chunk(); h < a.H; h += gridDim.y * P::chunk()) {
    P piece;
    float v[P::kCount];
    piece.fetch(hidden + t * pitch, h, a.H);
    piece.values(v);
    for (int k = 0; k < a.K; ++k) {
      const int64_t r = a.row(t, k);
      if (r >= 0) P::store(rows + r * a.H, h, a.H, v);
    }
  }
  clear_rows_behind<T, UNIT>(a, t, rows);
}

// Order and rows in one launch for a few tokens: every CTA works the order out for itself and moves one token's rows.
template <typename T, int UNIT>
__global__ void __launch_bounds__(kSortThreads) sort_few_kernel(SortArgs s, RowArgs a, const T* hidden, int64_t pitch,
                                                                int32_t* offsets, int32_t* row_of_pair, T* rows) {
  using P = Piece<T, UNIT>;
  extern __shared__ int hist[];
  __shared__ int s_row[kChunk];
  grid_enter(s.index, hidden);
  const bool first = blockIdx.x == 0;
  const int64_t t = blockIdx.x;
  P piece;  // on its way while the order is worked out
  piece.fetch(hidden + t * pitch, 0, a.H);
  const int used = order_chunk(s, 0, 1, nullptr, false, hist, first ? offsets : nullptr, [&](int64_t p, int row) {
    s_row[p] = row;
    if (first) row_of_pair[p] = row;
  });
  __syncthreads();
  const float zero[P::kCount] = {};
  for (int h = 0; h < a.H; h += P::chunk()) {
    float v[P::kCount];
    if (h > 0) piece.fetch(hidden + t * pitch, h, a.H);
    piece.values(v);
    for (int k = 0; k < a.K; ++k) {
      const int r = s_row[t * a.K + k];
      if (r >= 0) P::store(rows + static_cast<int64_t>(r) * a.H, h, a.H, v);
      if (t * a.K + k >= used) P::store(rows + (t * a.K + k) * a.H, h, a.H, zero);  // this row lies behind the last expert's
    }
  }
}

// out[t] = sum over k of (affinities[t, k]) rows[row_of_pair[t, k]], in fp32, k ascending, rounded once.  The same 2.4 GB in
// 356 us (343 without weights); one row at a time, 400 (386).
template <typename T, int UNIT, bool SHORT, int ROWS>
__global__ void __launch_bounds__(128) unsort_rows_kernel(RowArgs a, const T* rows, int64_t pitch, const void* affinities,
                                                          int aff_dtype, T* out) {
  using P = Piece<T, UNIT>;
  grid_enter(a.row_of_pair, rows, affinities);
  const int64_t t = own_token<SHORT>();
  if (SHORT && t >= a.T) return;
  for (int h = blockIdx.y * P::chunk(); h < a.H; h += gridDim.y * P::chunk()) {
    float sum[P::kCount] = {};
    for (int k0 = 0; k0 < a.K; k0 += ROWS) {  // ROWS rows on their way before the first is added
      P piece[ROWS];
      float w[ROWS];
      bool live[ROWS];
#pragma unroll
      for (int j = 0; j < ROWS; ++j) {
        const int64_t r = k0 + j < a.K ? a.row(t, k0 + j) : -1;
        live[j] = r >= 0;
        if (!live[j]) continue;
        piece[j].fetch(rows + r * pitch, h, a.H);
        w[j] = affinities != nullptr ? load_as_float(affinities, t * a.K + k0 + j, aff_dtype) : 1.0f;
      }
#pragma unroll
      for (int j = 0; j < ROWS; ++j) {
        if (!live[j]) continue;
        float v[P::kCount];
        piece[j].values(v);
#pragma unroll
        for (int i = 0; i < P::kCount; ++i) sum[i] = fmaf(w[j], v[i], sum[i]);
      }
    }
    P::store(out + t * a.H, h, a.H, sum);
  }
}

// d rows[r] = a[t, k] d out[t]; d a[t, k] = <d out[t], rows[r]>: one pass over a token's rows for both.  32768 tokens x 4096
// bf16, top-8: 4.6 GB in 695 us; with a row's load, product and store one after the other 1121.
template <typename T, int UNIT, bool SHORT, int ROWS>
__global__ void __launch_bounds__(256) unsort_backward_kernel(RowArgs a, const T* d_out, int64_t d_pitch, const T* rows,
                                                              int64_t pitch, const void* affinities, int aff_dtype,
                                                              T* d_rows, void* d_affinities) {
  using P = Piece<T, UNIT>;
  __shared__ float s_dot[8][ROWS];
  grid_enter(a.row_of_pair, a.offsets, d_out, rows, affinities);
  const int64_t t = own_token<SHORT>();
  const int warps = blockDim.x >> 5, lane = threadIdx.x & 31;  // of a token
  const int warp0 = SHORT ? threadIdx.y * warps : 0, warp = warp0 + (threadIdx.x >> 5);
  for (int k0 = 0; k0 < a.K; k0 += ROWS) {
    const int n = !SHORT || t < a.T ? min(ROWS, a.K - k0) : 0;
    int64_t r[ROWS];
    float w[ROWS], dot[ROWS];
#pragma unroll
    for (int j = 0; j < ROWS; ++j) {
      r[j] = j < n ? a.row(t, k0 + j) : -1;
      w[j] = j < n && affinities != nullptr ? load_as_float(affinities, t * a.K + k0 + j, aff_dtype) : 1.0f;
      dot[j] = 0.f;
    }
    for (int h = 0; h < a.H && n > 0; h += P::chunk()) {
      P piece[ROWS], own;  // all rows on their way before the first is used
      own.fetch(d_out + t * d_pitch, h, a.H);
      if (d_affinities != nullptr) {
#pragma unroll
        for (int j = 0; j < ROWS; ++j)
          if (r[j] >= 0) piece[j].fetch(rows + r[j] * pitch, h, a.H);
      }
      float d[P::kCount];
      own.values(d);
#pragma unroll
      for (int j = 0; j < ROWS; ++j) {
        if (r[j] < 0) continue;
        float v[P::kCount];
        if (d_affinities != nullptr) {
          piece[j].values(v);
#pragma unroll
          for (int i = 0; i < P::kCount; ++i) dot[j] = fmaf(d[i], v[i], dot[j]);
        }
        if (d_rows != nullptr) {
#pragma unroll
          for (int i = 0; i < P::kCount; ++i) v[i] = w[j] * d[i];
          P::store(d_rows + r[j] * a.H, h, a.H, v);
        }
      }
    }
    if (d_affinities != nullptr) {
#pragma unroll
      for (int j = 0; j < ROWS; ++j) {
        float s = dot[j];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (lane == 0) s_dot[warp][j] = s;
      }
      __syncthreads();
      if (threadIdx.x < static_cast<unsigned>(n)) {
        float s = 0.f;
        for (int i = 0; i < warps; ++i) s += s_dot[warp0 + i][threadIdx.x];
        store_from_float(d_affinities, t * a.K + k0 + threadIdx.x, aff_dtype, s);
      }
      __syncthreads();
    }
  }
  if (d_rows != nullptr && (!SHORT || t < a.T)) clear_rows_behind<T, UNIT>(a, t, d_rows);
}

// Bytes that the rows of all given matrices can be moved by: 16, 4, or an element's.
struct Rows {
  const void* p;
  int64_t pitch;
};
int common_unit(int dtype, int H, std::initializer_list<Rows> matrices) {
  const int size = dtype == B200MOE_F32 ? 4 : 2;
  uint64_t bits = static_cast<uint64_t>(H) * size;
  for (const Rows& m : matrices)
    if (m.p != nullptr) bits |= reinterpret_cast<uintptr_t>(m.p) | static_cast<uint64_t>(m.pitch * size);
  return bits % 16 == 0 ? 16 : (bits % 4 == 0 ? 4 : size);
}

// With enough tokens to give every SM several CTAs, a CTA of `threads` has as many tokens as their rows leave room for (30000
// rows of 256 bf16, one per token: 33 us with a token per CTA, 14 so); with fewer a token's columns are spread over CTAs.
struct Layout {
  dim3 grid, block;
};
Layout row_layout(int T, int H, int per_thread, int threads, bool spread) {
  const int lanes = ((H - 1) / per_thread + 32) & ~31;
  if (T < 8 * sm_count()) {
    const int parts = spread ? (H - 1) / (per_thread * threads) + 1 : 1;
    return {dim3(T, parts < 65535 ? parts : 65535), dim3(threads)};
  }
  const int x = lanes <= threads / 4 ? (lanes <= 32 ? 32 : threads / 4) : (lanes <= threads / 2 ? threads / 2 : threads);
  const int y = threads / x;
  return {dim3((T + y - 1) / y), dim3(x, y)};
}

int check_rows(const char* name, int dtype, int T, int K, int H, int64_t pitch) {
  B200MOE_REQUIRE(dtype == B200MOE_F32 || dtype == B200MOE_BF16, B200MOE_ERR_INVALID, "%s: rows must be fp32 or bf16", name);
  B200MOE_REQUIRE(T > 0 && K > 0 && H > 0 && H <= (1 << 30) && static_cast<int64_t>(T) * K <= INT32_MAX, B200MOE_ERR_INVALID,
                  "%s: need T, K, H > 0, at most 2^31 - 1 pairs and 2^30 columns", name);
  B200MOE_REQUIRE(pitch >= 0, B200MOE_ERR_INVALID, "%s: negative row pitch", name);
  return B200MOE_OK;
}

int check_sort(const void* expert_index, int index_bytes, int T, int K, int E, const int32_t* expert_offsets,
               const int32_t* row_of_pair) {
  B200MOE_REQUIRE(expert_index && expert_offsets && row_of_pair, B200MOE_ERR_INVALID, "sort_pairs: null pointer argument");
  B200MOE_REQUIRE(index_bytes == 4 || index_bytes == 8, B200MOE_ERR_INVALID, "sort_pairs: ids must have 4 or 8 bytes");
  B200MOE_REQUIRE(T > 0 && K > 0 && static_cast<int64_t>(T) * K <= INT32_MAX, B200MOE_ERR_INVALID,
                  "sort_pairs: need T, K > 0 and at most 2^31 - 1 pairs");
  B200MOE_REQUIRE(E > 0 && E <= kMaxExperts, B200MOE_ERR_INVALID, "sort_pairs: between 1 and %d experts, got %d", kMaxExperts, E);
  return B200MOE_OK;
}

// Calls fn with a value of the element type and the unit its rows move by, both known to the compiler.
template <typename F>
int with_rows(int dtype, int unit, const F& fn) {
  using std::integral_constant;
  if (dtype == B200MOE_F32)
    return unit == 16 ? fn(float{}, integral_constant<int, 16>{}) : fn(float{}, integral_constant<int, 4>{});
  if (unit == 16) return fn(__nv_bfloat16{}, integral_constant<int, 16>{});
  return unit == 4 ? fn(__nv_bfloat16{}, integral_constant<int, 4>{}) : fn(__nv_bfloat16{}, integral_constant<int, 2>{});
}

}  // namespace
}  // namespace b200moe

using namespace b200moe;

extern "C" size_t b200moe_sort_workspace_bytes(int64_t pairs, int E) {
  if (pairs <= kChunk || E <= 0) return 0;
  return static_cast<size_t>(ceil_div64(pairs, kChunk)) * E * sizeof(int);
}

extern "C" int b200moe_sort_pairs(const void* expert_index, int index_bytes, int T, int K, int E, int32_t* expert_offsets,
                                  int32_t* row_of_pair, void* workspace, size_t workspace_bytes, b200moe_stream_t stream) {
  const int rc = check_sort(expert_index, index_bytes, T, K, E, expert_offsets, row_of_pair);
  if (rc != B200MOE_OK) return rc;
  const SortArgs a{expert_index, index_bytes == 8, static_cast<int64_t>(T) * K, E};
  const int64_t chunks = ceil_div64(a.pairs, kChunk);
  B200MOE_REQUIRE(chunks == 1 || (workspace != nullptr && workspace_bytes >= b200moe_sort_workspace_bytes(a.pairs, E)),
                  B200MOE_ERR_WORKSPACE, "sort_pairs: workspace too small");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const size_t hist = static_cast<size_t>(kSortWarps + 1) * E * sizeof(int);
  const dim3 grid(static_cast<unsigned>(chunks));
  if (chunks > 1) {
    B200MOE_CUDA_OK(launch_overlapped(count_pairs_kernel, grid, kSortThreads, E * sizeof(int), st, a, static_cast<int*>(workspace)));
    B200MOE_LAUNCH_OK("count_pairs_kernel");
  }
  const bool scanned = scan_pays(chunks, E);
  if (scanned) {
    B200MOE_CUDA_OK(launch_overlapped(scan_counts_kernel, dim3((E + kScanExperts - 1) / kScanExperts), kScanExperts * kScanParts, 0, st,
                                      static_cast<int*>(workspace), static_cast<int>(chunks), E));
    B200MOE_LAUNCH_OK("scan_counts_kernel");
  }
  B200MOE_CUDA_OK(ensure_dynamic_smem(reinterpret_cast<const void*>(place_pairs_kernel), kMostHist));
  B200MOE_CUDA_OK(launch_overlapped(place_pairs_kernel, grid, kSortThreads, hist, st, a,
                                    static_cast<const int*>(workspace), scanned, expert_offsets, row_of_pair));
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
  return with_rows(dtype, common_unit(dtype, H, {{hidden, pitch}, {rows, H}}), [&](auto element, auto width) -> int {
    using T_ = decltype(element);
    constexpr int U = decltype(width)::value;
    const Layout l = row_layout(T, H, Piece<T_, U>::kCount, 128, true);
    const auto kernel = l.block.y > 1 ? sort_rows_kernel<T_, U, true> : sort_rows_kernel<T_, U, false>;
    B200MOE_CUDA_OK(launch_overlapped(kernel, l.grid, l.block, 0, static_cast<cudaStream_t>(stream), a,
                                      static_cast<const T_*>(hidden), pitch, static_cast<T_*>(rows)));
    B200MOE_LAUNCH_OK("sort_rows_kernel");
    return B200MOE_OK;
  });
}

extern "C" int b200moe_sort_tokens(const void* hidden, int dtype, int64_t pitch, const void* expert_index, int index_bytes, int T,
                                   int K, int H, int E, int32_t* expert_offsets, int32_t* row_of_pair, void* rows,
                                   void* workspace, size_t workspace_bytes, b200moe_stream_t stream) {
  B200MOE_REQUIRE(hidden && rows, B200MOE_ERR_INVALID, "sort_tokens: null pointer argument");
  int rc = check_rows("sort_tokens", dtype, T, K, H, pitch);
  if (rc != B200MOE_OK) return rc;
  rc = check_sort(expert_index, index_bytes, T, K, E, expert_offsets, row_of_pair);
  if (rc != B200MOE_OK) return rc;
  // One launch instead of two where a CTA per token does not repeat the order too often (16 tokens of 4096, 128 experts, top-8: 7.0 us
  // instead of 4.8 + 3.8, and 16.6 instead of 19.3 of host time)
  if (static_cast<int64_t>(T) * K <= kChunk && T <= 128) {
    const SortArgs s{expert_index, index_bytes == 8, static_cast<int64_t>(T) * K, E};
    const RowArgs a{T, K, H, E, nullptr, nullptr};
    return with_rows(dtype, common_unit(dtype, H, {{hidden, pitch}, {rows, H}}), [&](auto element, auto width) -> int {
      using T_ = decltype(element);
      constexpr int U = decltype(width)::value;
      B200MOE_CUDA_OK(ensure_dynamic_smem(reinterpret_cast<const void*>(sort_few_kernel<T_, U>), kMostHist));
      B200MOE_CUDA_OK(launch_overlapped(sort_few_kernel<T_, U>, dim3(T), kSortThreads, (kSortWarps + 1) * E * sizeof(int),
                                        static_cast<cudaStream_t>(stream), s, a, static_cast<const T_*>(hidden), pitch,
                                        expert_offsets, row_of_pair, static_cast<T_*>(rows)));
      B200MOE_LAUNCH_OK("sort_few_kernel");
      return B200MOE_OK;
    });
  }
  rc = b200moe_sort_pairs(expert_index, index_bytes, T, K, E, expert_offsets, row_of_pair, workspace, workspace_bytes, stream);
  return rc != B200MOE_OK ? rc : b200moe_sort_rows(hidden, dtype, pitch, T, K, H, E, row_of_pair, expert_offsets, rows, stream);
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
  return with_rows(dtype, common_unit(dtype, H, {{rows, pitch}, {out, H}}), [&](auto element, auto width) -> int {
    using T_ = decltype(element);
    constexpr int U = decltype(width)::value;
    const Layout l = row_layout(T, H, Piece<T_, U>::kCount, 128, true);
    const auto kernel = l.block.y > 1 ? (K > 4 ? unsort_rows_kernel<T_, U, true, 8> : unsort_rows_kernel<T_, U, true, 4>)
                                      : (K > 4 ? unsort_rows_kernel<T_, U, false, 8> : unsort_rows_kernel<T_, U, false, 4>);
    B200MOE_CUDA_OK(launch_overlapped(kernel, l.grid, l.block, 0, static_cast<cudaStream_t>(stream), a,
                                      static_cast<const T_*>(rows), pitch, affinities, aff_dtype, static_cast<T_*>(out)));
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
  return with_rows(dtype, common_unit(dtype, H, {{d_out, d_pitch}, {rows, pitch}, {d_rows, H}}), [&](auto element, auto width) -> int {
    using T_ = decltype(element);
    constexpr int U = decltype(width)::value;
    const int threads = T >= 8 * sm_count() && H <= 128 * 4 * Piece<T_, U>::kCount ? 128 : 256;
    const Layout l = row_layout(T, H, Piece<T_, U>::kCount, threads, false);
    const auto pick = [&](auto few) {
      constexpr bool S = decltype(few)::value;
      return K > 4 ? unsort_backward_kernel<T_, U, S, 8>
                   : (K > 2 ? unsort_backward_kernel<T_, U, S, 4> : unsort_backward_kernel<T_, U, S, 2>);
    };
    const auto kernel = l.block.y > 1 ? pick(std::true_type{}) : pick(std::false_type{});
    B200MOE_CUDA_OK(launch_overlapped(kernel, l.grid, l.block, 0, static_cast<cudaStream_t>(stream), a,
                                      static_cast<const T_*>(d_out), d_pitch, static_cast<const T_*>(rows), pitch, affinities,
                                      aff_dtype, static_cast<T_*>(d_rows), d_affinities));
    B200MOE_LAUNCH_OK("unsort_backward_kernel");
    return B200MOE_OK;
  });
}
