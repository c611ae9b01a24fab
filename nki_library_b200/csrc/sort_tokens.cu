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
// What a thread holds of a row is 16 bytes.
template <typename T>
constexpr int kPer = 16 / static_cast<int>(sizeof(T));

template <typename T>
__device__ __forceinline__ void unpack(const uint4& raw, float (&v)[kPer<T>]) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 2) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    } else {
      v[i] = __uint_as_float(w[i]);
    }
  }
}
template <typename T>
__device__ __forceinline__ uint4 pack(const float (&v)[kPer<T>]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 2) {
      const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&b);
    } else {
      w[i] = __float_as_uint(v[i]);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Where a matrix lies: bytes [lo, hi) from its first to its last element; 32 bytes around any element of the rows from `first`
// on, `count` of them, are still inside.
struct Span {
  uintptr_t lo, hi;
  int first;
  unsigned count;
  // Whether `size` bytes at `at`, around an element of the row, are inside.
  __device__ __forceinline__ bool around(int row, uintptr_t at, int size) const {
    return static_cast<unsigned>(row - first) < count || (at >= lo && at + size <= hi);
  }
};

// The 8 bytes at an aligned address, zero where they lie outside the matrix.  A call, since it is rare: in line it cost the
// sums 2 to 8 %.
template <typename T>
__device__ __noinline__ uint2 careful(uintptr_t at, uintptr_t lo, uintptr_t hi) {
  if (at >= lo && at + 8 <= hi) return __ldg(reinterpret_cast<const uint2*>(at));
  unsigned long long w = 0;
#pragma unroll 1
  for (int i = 0; i < 8; i += sizeof(T)) {
    const uintptr_t p = at + i;
    if (p < lo || p >= hi) continue;
    if constexpr (sizeof(T) == 2) w |= static_cast<unsigned long long>(__ldg(reinterpret_cast<const uint16_t*>(p))) << (8 * i);
    else w |= static_cast<unsigned long long>(__ldg(reinterpret_cast<const uint32_t*>(p))) << (8 * i);
  }
  return make_uint2(static_cast<uint32_t>(w), static_cast<uint32_t>(w >> 32));
}

// How a row is cut into pieces of 16 bytes that are aligned where they are stored.  WHOLE: rows are whole aligned 16 bytes
// everywhere, pieces start at columns 0, kPer, ...  Otherwise pieces are aligned in the row that is written, so that its first
// and last piece are cut, and a row that lies differently is read as the two or three aligned 8 bytes around each piece.  Sort,
// sum with weights and its gradients of 16000 tokens x 7163 bf16, top-8: 408, 372, 755 us, and 694, 781, 1157 by 2 bytes at a
// time; of 6000 x 5004, 8 experts: 112, 105, 203, and 143, 118, 230 by 4 bytes.  (Short rows of whole 4 bytes lose: 100000 x 130,
// top-8 97, 106, 288 and 68, 141, 204.)
template <typename T, bool WHOLE>
struct Cut {
  // Column of piece p of the row at `row`; pieces with column >= H do not exist.
  __device__ __forceinline__ static int column(const T* row, int p) {
    return p * kPer<T> - (WHOLE ? 0 : static_cast<int>(reinterpret_cast<uintptr_t>(row) & 15) / static_cast<int>(sizeof(T)));
  }
  __device__ __forceinline__ static int pieces(int H) { return (H - 1) / kPer<T> + (WHOLE ? 1 : 2); }

  // kPer elements from any address on.  Only loads, so that a caller's next row is asked for before this one is there.
  struct Read {
    uint2 a, b, c;
    uint32_t m;
    __device__ __forceinline__ void fetch(const T* first, const Span& span, int row) {
      if constexpr (WHOLE) {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(first));
        a = make_uint2(v.x, v.y);
        b = make_uint2(v.z, v.w);
      } else {
        const uintptr_t at = reinterpret_cast<uintptr_t>(first);
        m = static_cast<uint32_t>(at) & 7;
        if (span.around(row, at - m, 24)) {
          const uint2* p = reinterpret_cast<const uint2*>(at - m);
          a = __ldg(p);
          b = __ldg(p + 1);
          if (m != 0) c = __ldg(p + 2);
        } else {
          a = careful<T>(at - m, span.lo, span.hi);
          b = careful<T>(at - m + 8, span.lo, span.hi);
          c = careful<T>(at - m + 16, span.lo, span.hi);
        }
      }
    }
    __device__ __forceinline__ uint4 get() const {
      if constexpr (WHOLE) {
        return make_uint4(a.x, a.y, b.x, b.y);
      } else {
        uint32_t w[6] = {a.x, a.y, b.x, b.y, c.x, c.y};
#pragma unroll
        for (int i = 0; i < 5; ++i) w[i] = m & 4 ? w[i + 1] : w[i];
        if constexpr (sizeof(T) == 2) {
#pragma unroll
          for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], m * 8);  // by 0 or 16, modulo 32
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
      }
    }

    // The same of an aligned address.
    __device__ __forceinline__ void fetch_aligned(const T* first, const Span& span, int row) {
      if (WHOLE || span.around(row, reinterpret_cast<uintptr_t>(first), 16)) {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(first));
        a = make_uint2(v.x, v.y);
        b = make_uint2(v.z, v.w);
      } else {
        a = careful<T>(reinterpret_cast<uintptr_t>(first), span.lo, span.hi);
        b = careful<T>(reinterpret_cast<uintptr_t>(first) + 8, span.lo, span.hi);
      }
    }
    __device__ __forceinline__ uint4 get_aligned() const { return make_uint4(a.x, a.y, b.x, b.y); }

  };

  __device__ __forceinline__ static bool inside(int h, int H) { return WHOLE || (h >= 0 && h + kPer<T> <= H); }
  __device__ __forceinline__ static void store(T* row, int h, int H, const uint4& v) {
    if (inside(h, H)) {
      *reinterpret_cast<uint4*>(row + h) = v;
      return;
    }
    // The first or last bytes of the piece, n of them: at most one store of each size.
    char* p = reinterpret_cast<char*>(row + h);
    const int size = static_cast<int>(sizeof(T)), n = (h < 0 ? h + kPer<T> : H - h) * size;
    if (h < 0 && h + kPer<T> <= H) {
      if (n & 8) *reinterpret_cast<uint2*>(p + 8) = make_uint2(v.z, v.w);
      if (n & 4) *reinterpret_cast<uint32_t*>(p + (n & 8 ? 4 : 12)) = n & 8 ? v.y : v.w;
      if constexpr (sizeof(T) == 2)
        if (n & 2)
          *reinterpret_cast<uint16_t*>(p + 16 - n) =
              static_cast<uint16_t>((n & 8 ? (n & 4 ? v.x : v.y) : (n & 4 ? v.z : v.w)) >> 16);
    } else if (h >= 0) {
      if (n & 8) *reinterpret_cast<uint2*>(p) = make_uint2(v.x, v.y);
      if (n & 4) *reinterpret_cast<uint32_t*>(p + (n & 8)) = n & 8 ? v.z : v.x;
      if constexpr (sizeof(T) == 2)
        if (n & 2)
          *reinterpret_cast<uint16_t*>(p + n - 2) = static_cast<uint16_t>(n & 8 ? (n & 4 ? v.w : v.z) : (n & 4 ? v.y : v.x));
    } else {  // a row that ends in the piece it begins in
#pragma unroll 1
      for (int i = -h; i < H - h; ++i) {
        const uint32_t w = i * size < 8 ? (i * size < 4 ? v.x : v.y) : (i * size < 12 ? v.z : v.w);
        if constexpr (sizeof(T) == 2) *reinterpret_cast<uint16_t*>(p + 2 * i) = static_cast<uint16_t>(w >> (16 * (i & 1)));
        else *reinterpret_cast<uint32_t*>(p + 4 * i) = w;
      }
    }
  }
  // sum + <d, v> over the columns that exist.
  __device__ __forceinline__ static float dot(int h, int H, const float (&d)[kPer<T>], const float (&v)[kPer<T>], float sum) {
    if (inside(h, H)) {
#pragma unroll
      for (int i = 0; i < kPer<T>; ++i) sum = fmaf(d[i], v[i], sum);
    } else {
#pragma unroll
      for (int i = 0; i < kPer<T>; ++i)
        if (static_cast<unsigned>(h + i) < static_cast<unsigned>(H)) sum = fmaf(d[i], v[i], sum);
    }
    return sum;
  }
};

struct RowArgs {
  int T, K, H, E;
  const int32_t* row_of_pair;
  const int32_t* offsets;
  int pairs;
  // Row of the token's k-th pair, -1 if it has none.
  __device__ __forceinline__ int64_t row(int64_t t, int k) const {
    const int r = row_of_pair[t * K + k];
    return r < pairs ? r : -1;
  }
};

// A token belongs to a CTA, or (SHORT) to the threads of one threadIdx.y, where a row is too short for a CTA.  Two forms of each
// kernel, because an index that differs between warps costs registers (unsort of 32768 tokens, 361 and 404 us).
template <bool SHORT>
__device__ __forceinline__ int64_t own_token() {
  return SHORT ? static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y : blockIdx.x;
}

// A thread's pieces of its token's rows.
__device__ __forceinline__ int first_piece() { return static_cast<int>(blockIdx.y * blockDim.x + threadIdx.x); }
__device__ __forceinline__ int piece_stride() { return static_cast<int>(gridDim.y * blockDim.x); }

// The K rows that a token's threads clear if they lie behind the last expert's: rows t * K to t * K + K - 1.
template <typename T, bool WHOLE>
__device__ __forceinline__ void clear_rows_behind(const RowArgs& a, int64_t t, T* rows) {
  using C = Cut<T, WHOLE>;
  const int64_t r0 = t * a.K;
  for (int64_t r = max(r0, static_cast<int64_t>(a.offsets[a.E])); r < r0 + a.K; ++r) {
    T* row = rows + r * a.H;
    for (int p = first_piece(); p < C::pieces(a.H); p += piece_stride()) {
      const int h = C::column(row, p);
      if (h < a.H) C::store(row, h, a.H, make_uint4(0, 0, 0, 0));
    }
  }
}

// One piece of a token's row at hidden, into the rows of K pairs; `row_of(k)` is -1 for none.
template <typename T, bool WHOLE, typename RowOf>
__device__ __forceinline__ void spread_piece(const RowArgs& a, const T* hidden, const Span& span, int t, int p, T* rows,
                                             const RowOf& row_of) {
  using C = Cut<T, WHOLE>;
  if constexpr (WHOLE) {
    const uint4 v = __ldg(reinterpret_cast<const uint4*>(hidden + p * kPer<T>));
    for (int k = 0; k < a.K; ++k) {
      const int64_t r = row_of(k);
      if (r >= 0) *reinterpret_cast<uint4*>(rows + r * a.H + p * kPer<T>) = v;
    }
  } else {
    // each lies differently: read, from L1 after the first, as each needs it
    for (int k = 0; k < a.K; ++k) {
      const int64_t r = row_of(k);
      if (r < 0) continue;
      T* row = rows + r * a.H;
      const int h = C::column(row, p);
      if (h >= a.H) continue;
      typename C::Read piece;
      piece.fetch(hidden + h, span, t);
      C::store(row, h, a.H, piece.get());
    }
  }
}

// rows[row_of_pair[t, k]] = hidden[t].  32768 tokens x 4096 bf16, top-8: 2.4 GB in 402 us, 0.92 of the copy rate.
template <typename T, bool WHOLE, bool SHORT>
__global__ void __launch_bounds__(128) sort_rows_kernel(RowArgs a, const T* hidden, int64_t pitch, Span span, T* rows) {
  grid_enter(a.row_of_pair, a.offsets, hidden);
  const int64_t t = own_token<SHORT>();
  if (SHORT && t >= a.T) return;
  for (int p = first_piece(); p < Cut<T, WHOLE>::pieces(a.H); p += piece_stride())
    spread_piece<T, WHOLE>(a, hidden + t * pitch, span, static_cast<int>(t), p, rows, [&](int k) { return a.row(t, k); });
  clear_rows_behind<T, WHOLE>(a, t, rows);
}

// Order and rows in one launch for a few tokens: every CTA works the order out for itself and moves one token's rows.
template <typename T, bool WHOLE>
__global__ void __launch_bounds__(kSortThreads) sort_few_kernel(SortArgs s, RowArgs a, const T* hidden, int64_t pitch, Span span,
                                                                int32_t* offsets, int32_t* row_of_pair, T* rows) {
  using C = Cut<T, WHOLE>;
  extern __shared__ int hist[];
  __shared__ int s_row[kChunk];
  grid_enter(s.index, hidden);
  const bool first = blockIdx.x == 0;
  const int64_t t = blockIdx.x;
  // on its way while the order is worked out
  if (static_cast<int>(threadIdx.x) * kPer<T> < a.H)
    asm volatile("prefetch.global.L1 [%0];" ::"l"(hidden + t * pitch + threadIdx.x * kPer<T>));
  const int used = order_chunk(s, 0, 1, nullptr, false, hist, first ? offsets : nullptr, [&](int64_t p, int row) {
    s_row[p] = row;
    if (first) row_of_pair[p] = row;
  });
  __syncthreads();
  for (int p = threadIdx.x; p < C::pieces(a.H); p += kSortThreads)
    spread_piece<T, WHOLE>(a, hidden + t * pitch, span, static_cast<int>(t), p, rows,
                           [&](int k) -> int64_t { return s_row[t * a.K + k]; });
  for (int64_t r = max(t * a.K, static_cast<int64_t>(used)); r < (t + 1) * a.K; ++r) {  // behind the last expert's rows
    for (int p = threadIdx.x; p < C::pieces(a.H); p += kSortThreads) {
      const int h = C::column(rows + r * a.H, p);
      if (h < a.H) C::store(rows + r * a.H, h, a.H, make_uint4(0, 0, 0, 0));
    }
  }
}

// out[t] = sum over k of (affinities[t, k]) rows[row_of_pair[t, k]], in fp32, k ascending, rounded once.  The same 2.4 GB in
// 351 us (341 without weights); one row at a time, 400 (386).
template <typename T, bool WHOLE, bool SHORT, int ROWS>
__global__ void __launch_bounds__(128, !WHOLE && SHORT ? 8 : 0)  // 80 registers without the bound, 123 us instead of 106 at 130 columns
unsort_rows_kernel(RowArgs a, const T* rows, int64_t pitch, Span span, const void* affinities, int aff_dtype, T* out) {
  using C = Cut<T, WHOLE>;
  grid_enter(a.row_of_pair, rows, affinities);
  const int64_t t = own_token<SHORT>();
  if (SHORT && t >= a.T) return;
  T* to = out + t * a.H;
  for (int p = first_piece(); p < C::pieces(a.H); p += piece_stride()) {
    const int h = C::column(to, p);
    if (h >= a.H) break;
    float sum[kPer<T>] = {};
    for (int k0 = 0; k0 < a.K; k0 += ROWS) {  // ROWS rows on their way before the first is added
      typename C::Read piece[ROWS];
      float w[ROWS];
      bool live[ROWS];
#pragma unroll
      for (int j = 0; j < ROWS; ++j) {
        const int64_t r = k0 + j < a.K ? a.row(t, k0 + j) : -1;
        live[j] = r >= 0;
        if (!live[j]) continue;
        piece[j].fetch(rows + r * pitch + h, span, static_cast<int>(r));
        w[j] = affinities != nullptr ? load_as_float(affinities, t * a.K + k0 + j, aff_dtype) : 1.0f;
      }
#pragma unroll
      for (int j = 0; j < ROWS; ++j) {
        if (!live[j]) continue;
        float v[kPer<T>];
        unpack<T>(piece[j].get(), v);
#pragma unroll
        for (int i = 0; i < kPer<T>; ++i) sum[i] = fmaf(w[j], v[i], sum[i]);
      }
    }
    C::store(to, h, a.H, pack<T>(sum));
  }
}

// Lane j's result is the sum of v[j] over the warp (j < N, a power of two): lanes share the values out as they add them up.
template <int N>
__device__ __forceinline__ float sum_over_warp(float (&v)[N], int lane) {
#pragma unroll
  for (int n = N / 2; n > 0; n >>= 1) {
    const bool upper = lane & n;
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const float other = __shfl_xor_sync(0xffffffffu, upper ? v[i] : v[i + n], n);
      v[i] = (upper ? v[i + n] : v[i]) + other;
    }
  }
#pragma unroll
  for (int o = N; o < 32; o <<= 1) v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
  return v[0];
}

// d rows[r] = a[t, k] d out[t]; d a[t, k] = <d out[t], rows[r]>: one pass over a token's rows for both.  32768 tokens x 4096
// bf16, top-8: 4.6 GB in 687 us; with a row's load, product and store one after the other 1121.  ALIKE: a row that is read and the
// one that is written in its place lie alike in their 16 bytes (or only one of them is there).
// The cut form lives from occupancy (48 or 64 registers; unbounded at 100, 6000 x 5003, top-8: 334 us, 209 so), the whole one from
// the rows in flight.
template <typename T, bool WHOLE, bool ALIKE, bool SHORT, int ROWS>
__global__ void __launch_bounds__(256, WHOLE || ROWS > 4 ? 0 : (ALIKE && ROWS == 2 ? 5 : 4))
unsort_backward_kernel(RowArgs a, const T* d_out, int64_t d_pitch, Span d_span, const T* rows, int64_t pitch, Span span,
                       const void* affinities, int aff_dtype, T* d_rows, void* d_affinities) {
  using C = Cut<T, WHOLE>;
  __shared__ float s_dot[2][8][ROWS];
  grid_enter(a.row_of_pair, a.offsets, d_out, rows, affinities);
  const int64_t t = own_token<SHORT>();
  const int warps = blockDim.x >> 5, lane = threadIdx.x & 31;  // of a token
  const int warp0 = SHORT ? threadIdx.y * warps : 0, warp = warp0 + (threadIdx.x >> 5);
  int buffer = 0;  // of s_dot: with two, one barrier per ROWS rows
  for (int k0 = 0; k0 < a.K; k0 += ROWS, buffer ^= 1) {
    const int n = !SHORT || t < a.T ? min(ROWS, a.K - k0) : 0;
    int r[ROWS];
    float w[ROWS], dot[ROWS];
#pragma unroll
    for (int j = 0; j < ROWS; ++j) {
      r[j] = j < n ? static_cast<int>(a.row(t, k0 + j)) : -1;
      w[j] = j < n && affinities != nullptr ? load_as_float(affinities, t * a.K + k0 + j, aff_dtype) : 1.0f;
      dot[j] = 0.f;
    }
    // One piece of row j: what `d` of the gradient and `piece` of the row give.
    const auto use = [&](int j, int h, const float (&d)[kPer<T>], const uint4& piece) {
      float v[kPer<T>];
      if (d_affinities != nullptr) {
        unpack<T>(piece, v);
        dot[j] = C::dot(h, a.H, d, v, dot[j]);
      }
      if (d_rows != nullptr) {
#pragma unroll
        for (int i = 0; i < kPer<T>; ++i) v[i] = w[j] * d[i];
        C::store(d_rows + static_cast<int64_t>(r[j]) * a.H, h, a.H, pack<T>(v));
      }
    };
    for (int p = threadIdx.x; p < C::pieces(a.H) && n > 0; p += blockDim.x) {
      typename C::Read piece[ROWS];  // all rows on their way before the first is used
      if constexpr (WHOLE) {
        const int h = p * kPer<T>;
        typename C::Read own;
        own.fetch_aligned(d_out + t * d_pitch + h, d_span, 0);
        if (d_affinities != nullptr) {
#pragma unroll
          for (int j = 0; j < ROWS; ++j)
            if (r[j] >= 0) piece[j].fetch_aligned(rows + static_cast<int64_t>(r[j]) * pitch + h, span, 0);
        }
        float d[kPer<T>];
        unpack<T>(own.get_aligned(), d);
#pragma unroll
        for (int j = 0; j < ROWS; ++j)
          if (r[j] >= 0) use(j, h, d, piece[j].get_aligned());
      } else {
        // cut as the row that is written; the gradient's pieces then differ from row to row and come from L1 after the first
        typename C::Read own[2];
        int h[ROWS];
#pragma unroll
        for (int j = 0; j < ROWS; ++j) {
          h[j] = a.H;
          if (r[j] < 0) continue;
          const T* row = rows + static_cast<int64_t>(r[j]) * pitch;
          h[j] = C::column(d_rows != nullptr ? d_rows + static_cast<int64_t>(r[j]) * a.H : row, p);
          if (h[j] >= a.H || d_affinities == nullptr) continue;
          if constexpr (ALIKE) piece[j].fetch_aligned(row + h[j], span, r[j]);
          else piece[j].fetch(row + h[j], span, r[j]);
        }
        if (h[0] < a.H) own[0].fetch(d_out + t * d_pitch + h[0], d_span, static_cast<int>(t));
#pragma unroll
        for (int j = 0; j < ROWS; ++j) {
          if (j + 1 < ROWS && h[j + 1 < ROWS ? j + 1 : 0] < a.H)
            own[(j + 1) & 1].fetch(d_out + t * d_pitch + h[j + 1 < ROWS ? j + 1 : 0], d_span, static_cast<int>(t));
          if (h[j] >= a.H) continue;
          float d[kPer<T>];
          unpack<T>(own[j & 1].get(), d);
          use(j, h[j], d, ALIKE ? piece[j].get_aligned() : piece[j].get());
        }
      }
    }
    if (d_affinities != nullptr) {
      const float s = sum_over_warp<ROWS>(dot, lane);
      if (lane < ROWS) s_dot[buffer][warp][lane] = s;
      __syncthreads();
      if (threadIdx.x < static_cast<unsigned>(n)) {
        float s = 0.f;
        for (int i = 0; i < warps; ++i) s += s_dot[buffer][warp0 + i][threadIdx.x];
        store_from_float(d_affinities, t * a.K + k0 + threadIdx.x, aff_dtype, s);
      }
    }
  }
  if (d_rows != nullptr && (!SHORT || t < a.T)) clear_rows_behind<T, WHOLE>(a, t, d_rows);
}

struct Rows {
  const void* p;
  int64_t pitch;
};
Span span_of(int dtype, const void* p, int64_t rows, int64_t pitch, int H) {
  const uintptr_t lo = reinterpret_cast<uintptr_t>(p), size = dtype == B200MOE_F32 ? 4 : 2;
  const bool apart = pitch >= H && H * size >= 32 && rows > 2;
  return {lo, lo + static_cast<uintptr_t>((rows - 1) * pitch + H) * size, 1, apart ? static_cast<unsigned>(rows - 2) : 0u};
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
  return {dim3(static_cast<unsigned>(ceil_div64(T, y))), dim3(x, y)};
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

// bf16 rows of whole 4 bytes that are only copied are cut as fp32 ones of half the width, whose pieces have fewer ends (100000 x 130,
// top-8: 97 us instead of 108; 16000 x 1002, top-4: 37.4 and 39.4).
// H may be 2^30, whose bytes pass 32 bits.
constexpr bool copied_as_fp32(uint64_t addresses, int H, int64_t pitch) {
  const uint64_t bits = addresses | (static_cast<uint64_t>(H) * 2) | (static_cast<uint64_t>(pitch) * 2);
  return bits % 4 == 0 && bits % 16 != 0;
}
static_assert(copied_as_fp32(4, 1 << 30, int64_t{1} << 30) && !copied_as_fp32(16, 1 << 30, int64_t{1} << 30) && !copied_as_fp32(2, 8, 8));
void widen_copy(int& dtype, int& H, int64_t& pitch, const void* from, const void* to) {
  if (dtype != B200MOE_BF16 || !copied_as_fp32(reinterpret_cast<uintptr_t>(from) | reinterpret_cast<uintptr_t>(to), H, pitch)) return;
  dtype = B200MOE_F32;
  H /= 2;
  pitch /= 2;
}

// Calls fn with a value of the element type and whether all rows of the matrices are whole aligned 16 bytes, both known to the
// compiler.
template <typename F>
int with_rows(const char* name, int dtype, int H, std::initializer_list<Rows> matrices, const F& fn) {
  const int size = dtype == B200MOE_F32 ? 4 : 2;
  uint64_t at = 0, apart = static_cast<uint64_t>(H) * size;
  for (const Rows& m : matrices) {
    if (m.p == nullptr) continue;
    at |= reinterpret_cast<uintptr_t>(m.p);
    apart |= static_cast<uint64_t>(m.pitch * size);
  }
  B200MOE_REQUIRE(at % size == 0, B200MOE_ERR_INVALID, "%s: rows must start on an element's boundary", name);
  const bool whole = (at | apart) % 16 == 0;
  if (dtype == B200MOE_F32) return whole ? fn(float{}, std::true_type{}) : fn(float{}, std::false_type{});
  return whole ? fn(__nv_bfloat16{}, std::true_type{}) : fn(__nv_bfloat16{}, std::false_type{});
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
  widen_copy(dtype, H, pitch, hidden, rows);
  const RowArgs a{T, K, H, E, row_of_pair, expert_offsets, T * K};
  return with_rows("sort_rows", dtype, H, {{hidden, pitch}, {rows, H}}, [&](auto element, auto whole) -> int {
    using T_ = decltype(element);
    constexpr bool W = decltype(whole)::value;
    const Layout l = row_layout(T, H, kPer<T_>, 128, true);
    const auto kernel = l.block.y > 1 ? sort_rows_kernel<T_, W, true> : sort_rows_kernel<T_, W, false>;
    B200MOE_CUDA_OK(launch_overlapped(kernel, l.grid, l.block, 0, static_cast<cudaStream_t>(stream), a,
                                      static_cast<const T_*>(hidden), pitch, span_of(dtype, hidden, T, pitch, H), static_cast<T_*>(rows)));
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
  // One launch instead of two where a CTA per token does not repeat the order too often.  One / two launches, back to back, tokens of
  // 4096, 128 experts, top-8: 16 tokens 5.1 / 7.4 us, 64 5.4 / 7.4, 128 6.9 / 7.4, 160 9.5 / 7.9, 256 10.1 / 9.4 (8 experts: 128 5.7 /
  // 7.4, 256 7.4 / 7.8; 1024 experts: 128 7.3 / 8.4, 160 10.8 / 9.1).
  if (static_cast<int64_t>(T) * K <= kChunk && T <= 128) {
    widen_copy(dtype, H, pitch, hidden, rows);
    const SortArgs s{expert_index, index_bytes == 8, static_cast<int64_t>(T) * K, E};
    const RowArgs a{T, K, H, E, nullptr, nullptr, T * K};
    return with_rows("sort_tokens", dtype, H, {{hidden, pitch}, {rows, H}}, [&](auto element, auto whole) -> int {
      using T_ = decltype(element);
      constexpr bool W = decltype(whole)::value;
      B200MOE_CUDA_OK(ensure_dynamic_smem(reinterpret_cast<const void*>(sort_few_kernel<T_, W>), kMostHist));
      B200MOE_CUDA_OK(launch_overlapped(sort_few_kernel<T_, W>, dim3(T), kSortThreads, (kSortWarps + 1) * E * sizeof(int),
                                        static_cast<cudaStream_t>(stream), s, a, static_cast<const T_*>(hidden), pitch,
                                        span_of(dtype, hidden, T, pitch, H),
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
  const RowArgs a{T, K, H, 0, row_of_pair, nullptr, T * K};
  return with_rows("unsort_rows", dtype, H, {{rows, pitch}, {out, H}}, [&](auto element, auto whole) -> int {
    using T_ = decltype(element);
    constexpr bool W = decltype(whole)::value;
    const Layout l = row_layout(T, H, kPer<T_>, 128, true);
    // Rows in flight, four / eight: 32768 tokens of 4096 bf16, top-8 356 / 347 us, of 2048 185 / 180 (fp32 687 / 690), where several
    // tokens share a CTA 111 / 118 (65536 of 512); cut rows, whose reads take three registers more each, of 2045 251 / 368; with top-2
    // (16384 of 4096) 76 / 85.
    const auto kernel = l.block.y > 1 ? (K > 4 ? unsort_rows_kernel<T_, W, true, W ? 8 : 4> : unsort_rows_kernel<T_, W, true, 4>)
                                      : (K > 4 ? unsort_rows_kernel<T_, W, false, W ? 8 : 4> : unsort_rows_kernel<T_, W, false, 4>);
    B200MOE_CUDA_OK(launch_overlapped(kernel, l.grid, l.block, 0, static_cast<cudaStream_t>(stream), a,
                                      static_cast<const T_*>(rows), pitch,
                                      span_of(dtype, rows, static_cast<int64_t>(T) * K, pitch, H), affinities,
                                      aff_dtype, static_cast<T_*>(out)));
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
  const RowArgs a{T, K, H, E, row_of_pair, expert_offsets, T * K};
  return with_rows("unsort_rows_backward", dtype, H, {{d_out, d_pitch}, {rows, pitch}, {d_rows, H}},
                   [&](auto element, auto whole) -> int {
    using T_ = decltype(element);
    constexpr bool W = decltype(whole)::value;
    // Threads of a CTA, 128 / 256: 32768 tokens, top-8, bf16 of 2048 344 / 455 us, 4096 683 / 733, 8192 1373 / 1384, 16384 (16384 tokens,
    // top-4) 742 / 726; fp32 of 2048 684 / 737, 4096 1373 / 1363, 8192 2772 / 2718.  Few tokens leave SMs idle, and the wider CTA is
    // through sooner where they do: 64 of 4096 fp32 10.4 / 9.3, bf16 8.6 / 8.4 (300 11.0 / 11.4, 600 12.3 / 14.7).
    const int threads = T >= 8 * sm_count() && H <= 128 * 8 * kPer<T_> ? 128 : 256;
    const Layout l = row_layout(T, H, kPer<T_>, threads, false);
    const bool few_tokens = T <= 2 * sm_count();  // all of them at once in the form of eight rows
    const auto pick = [&](auto brief, auto alike) {
      constexpr bool S = decltype(brief)::value, A = decltype(alike)::value;
      if (!A || K <= 2 || (!W && S)) return unsort_backward_kernel<T_, W, A, S, 2>;
      if constexpr (A && (W || !S))
        return K > 4 && (W || few_tokens) ? unsort_backward_kernel<T_, W, A, S, 8> : unsort_backward_kernel<T_, W, A, S, 4>;
      return unsort_backward_kernel<T_, W, A, S, 2>;
    };
    const auto with_length = [&](auto alike) {
      return l.block.y > 1 ? pick(std::true_type{}, alike) : pick(std::false_type{}, alike);
    };
    const bool lie_alike = d_rows == nullptr || d_affinities == nullptr ||
                           (((reinterpret_cast<uintptr_t>(rows) ^ reinterpret_cast<uintptr_t>(d_rows)) |
                             static_cast<uintptr_t>((pitch - H) * static_cast<int64_t>(sizeof(T_)))) & 15) == 0;
    const auto kernel = W || lie_alike ? with_length(std::true_type{}) : with_length(std::bool_constant<W>{});
    B200MOE_CUDA_OK(launch_overlapped(kernel, l.grid, l.block, 0, static_cast<cudaStream_t>(stream), a,
                                      static_cast<const T_*>(d_out), d_pitch, span_of(dtype, d_out, T, d_pitch, H),
                                      static_cast<const T_*>(rows), pitch, span_of(dtype, rows, static_cast<int64_t>(T) * K, pitch, H), affinities,
                                      aff_dtype, static_cast<T_*>(d_rows), d_affinities));
    B200MOE_LAUNCH_OK("unsort_backward_kernel");
    return B200MOE_OK;
  });
}
