// m = act(gate) * up with an 8-bit activation checkpoint, and its backward pass from that checkpoint.
//
// Kept of a row's gate and up (each on its own, per 32 columns): e4m3 codes of v / s and s, the smallest power of two of at
// least 2^-127 for which no finite value of the block exceeds 448 s.  Values that are not finite are kept as NaN and do not
// count for s.  A kept value is off by at most 2^-4 of itself (or 2^-10 s).  8.25 bits instead of 16 a value.
// Backward, with the kept g^ and u^: d g = d m u^ act'(g^), d u = d m act(g^); m^ = act(g^) u^ if the caller wants it (the
// weight gradient of the product behind).
#include "common.cuh"
#include "quantize_row.cuh"

namespace b200moe {
namespace {

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float rcp(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Two fp32 operations in one instruction, each rounded as the single ones are.
__device__ __forceinline__ unsigned long long& bits2(float2& v) { return reinterpret_cast<unsigned long long&>(v); }
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(bits2(r)) : "l"(bits2(a)), "l"(bits2(b)));
  return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(bits2(r)) : "l"(bits2(a)), "l"(bits2(b)));
  return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(bits2(r)) : "l"(bits2(a)), "l"(bits2(b)), "l"(bits2(c)));
  return r;
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// act(g) and act'(g) of two values in fp32.  SiLU, Swish and the tanh form of GELU are g sigma(z(g)): act' = sigma + g sigma
// (1 - sigma) z'.  The two approximations are good to 2^-22 each.
template <int ACT>
__device__ __forceinline__ void act_and_slope(float2 g, float2& act, float2& slope) {
  constexpr float kLog2e = 1.4426950408889634f;
  if constexpr (ACT == B200MOE_ACT_GELU) {
    // With a = |g| / sqrt 2 and t = 1 / (1 + 0.51 a): erfc(a) exp(a^2) = t Q(t), a least-squares fit of the relative error over
    // a in [0, 10] that is off by 1.2e-6 of itself; the exponential is what the slope needs too.  The tail keeps its relative
    // precision.  (65536 x 4096 with checkpoint: 353 us; with erfcf, exp and a division from the library 856.)  Here Q / 2.
    const float2 square = mul2(mul2(g, both(-0.5f * kLog2e)), g);
    const float2 e = make_float2(ex2(square.x), ex2(square.y));
    const float2 d = fma2(both(0.51f * 0.70710678118654752f), make_float2(fabsf(g.x), fabsf(g.y)), both(1.0f));
    const float2 t = make_float2(rcp(d.x), rcp(d.y));
    float2 q = both(4.725153e-2f);
    q = fma2(q, t, both(-1.7957276e-1f));
    q = fma2(q, t, both(1.7923014e-1f));
    q = fma2(q, t, both(2.75213645e-2f));
    q = fma2(q, t, both(1.39534905e-1f));
    q = fma2(q, t, both(1.4207582e-1f));
    q = fma2(q, t, both(1.43958775e-1f));
    const float2 tail = mul2(mul2(q, t), e);
    const float2 rest = fma2(tail, both(-1.0f), both(1.0f));
    const float2 cdf = make_float2(g.x < 0.0f ? tail.x : rest.x, g.y < 0.0f ? tail.y : rest.y);
    act = mul2(g, cdf);
    slope = fma2(mul2(g, both(0.39894228040143268f)), e, cdf);
  } else {
    float2 z, dz;  // z in powers of two
    if constexpr (ACT == B200MOE_ACT_SILU) {
      z = mul2(both(-kLog2e), g);
      dz = both(1.0f);
    } else if constexpr (ACT == B200MOE_ACT_SWISH) {
      z = mul2(both(-1.702f * kLog2e), g);
      dz = both(1.702f);
    } else {  // (1 + tanh(z / 2)) / 2 = sigma(z)
      float2 g2 = mul2(g, g);
      g2 = make_float2(fminf(g2.x, 1e30f), fminf(g2.y, 1e30f));  // keeps dz finite
      z = mul2(mul2(both(-1.5957691216057308f * kLog2e), g), fma2(both(0.044715f), g2, both(1.0f)));
      dz = fma2(both(1.5957691216057308f * 3.0f * 0.044715f), g2, both(1.5957691216057308f));
    }
    const float2 d = add2(both(1.0f), make_float2(ex2(z.x), ex2(z.y)));
    const float2 sigma = make_float2(rcp(d.x), rcp(d.y));
    act = mul2(g, sigma);
    const float2 turn = mul2(act, fma2(sigma, both(-1.0f), both(1.0f)));
    slope = fma2(turn, dz, sigma);
  }
}

// Eight values of a block that four neighbouring lanes hold: their codes and the block's scale byte.  The whole warp calls.
__device__ __forceinline__ uint2 keep8(float (&v)[8], uint32_t& scale_byte) {
  const auto largest = [&v] {
    float t = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) t = fmaxf(t, fabsf(v[j]));  // takes no notice of NaN
    t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 1));
    return fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 2));
  };
  float top = largest();
  if (__any_sync(0xffffffffu, isinf(top))) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (isinf(v[j])) v[j] = __uint_as_float(0x7fc00000u);
    top = largest();
  }
  // exponent of top / 448 = top / (1.75 * 2^8), rounded up: one more where top's mantissa is above 1.75
  scale_byte = max(static_cast<int>((__float_as_uint(top) + 0x1fffffu) >> 23) - 8, 0);
  const float f = __uint_as_float((254u - scale_byte) << 23);  // 1 / s, a normal number for every s
  float2 x[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) x[j] = mul2(make_float2(v[2 * j], v[2 * j + 1]), both(f));
  return make_uint2(pack4_e4m3(x[0].x, x[0].y, x[1].x, x[1].y), pack4_e4m3(x[2].x, x[2].y, x[3].x, x[3].y));
}

__device__ __forceinline__ void kept8(uint2 codes, uint32_t scale_byte, float (&v)[8]) {
  const float scale = __uint_as_float(scale_byte != 0 ? scale_byte << 23 : 0x400000u);
  const uint32_t w[2] = {codes.x, codes.y};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_fp8x2_storage_t two = static_cast<__nv_fp8x2_storage_t>(w[i >> 1] >> (16 * (i & 1)));
    const __half2 h = __half2(__nv_cvt_fp8x2_to_halfraw2(two, __NV_E4M3));
    const float2 f = mul2(__half22float2(h), both(scale));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
  if (scale_byte >= 247) {  // 256 * 2^120, what the largest finite values round up to, is no fp32 number
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (isinf(v[j])) v[j] = copysignf(3.402823466e38f, v[j]);
  }
}

__device__ __forceinline__ uint4 pack8_bf16(const float (&v)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&b);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// A CTA's up to 256 threads cover `width` pieces of eight columns (whole blocks of 32, so that a block's four lanes sit together)
// of 256 / width rows; blockIdx.y picks the piece range of a wide row.  Each thread has two rows in flight.
struct Shape {
  int64_t R;
  int I, blocks, width, rows, inverse;  // inverse: 2^16 / width, rounded up
};
struct Place {
  int row, c;  // row of the CTA's, first column
  bool used;
};
__device__ __forceinline__ Place place(const Shape& s) {
  const int r = (threadIdx.x * s.inverse) >> 16;
  const int c = (static_cast<int>(blockIdx.y) * s.width + static_cast<int>(threadIdx.x) - r * s.width) * 8;
  return {r, c, r < s.rows && c < s.I};
}

// Bound by the bytes it moves: 65536 x 4096, SiLU, 2.16 GB with the checkpoint in 341 us, 1.61 GB without in 249; GELU 353 and
// 245 (one value at a time, its arithmetic showed: 391 and 254).
template <int ACT, bool KEEP>
__global__ void __launch_bounds__(256) glu_kernel(Shape s, const __nv_bfloat16* gate_up, int64_t pitch, __nv_bfloat16* m,
                                                  uint8_t* codes, uint8_t* scales) {
  grid_enter(gate_up);
  const Place at = place(s);
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * s.rows * 2; base < s.R; base += static_cast<int64_t>(gridDim.x) * s.rows * 2) {
    uint4 raw[2][2] = {};
    bool inside[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int64_t row = base + i * s.rows + at.row;
      inside[i] = at.used && row < s.R;
      if (inside[i]) {
        raw[i][0] = __ldg(reinterpret_cast<const uint4*>(gate_up + row * pitch + at.c));
        raw[i][1] = __ldg(reinterpret_cast<const uint4*>(gate_up + row * pitch + s.I + at.c));
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int64_t row = base + i * s.rows + at.row;
      float g[8], u[8], out[8];
      unpack8_bf16(raw[i][0], g);
      unpack8_bf16(raw[i][1], u);
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        float2 a, slope;
        act_and_slope<ACT>(make_float2(g[j], g[j + 1]), a, slope);
        const float2 v = mul2(a, make_float2(u[j], u[j + 1]));
        out[j] = v.x;
        out[j + 1] = v.y;
      }
      if (inside[i]) *reinterpret_cast<uint4*>(m + row * s.I + at.c) = pack8_bf16(out);
      if constexpr (KEEP) {
        uint32_t sg, su;
        const uint2 cg = keep8(g, sg), cu = keep8(u, su);
        if (inside[i]) {
          *reinterpret_cast<uint2*>(codes + row * 2 * s.I + at.c) = cg;
          *reinterpret_cast<uint2*>(codes + row * 2 * s.I + s.I + at.c) = cu;
          if ((threadIdx.x & 3) == 0) {
            scales[row * 2 * s.blocks + (at.c >> 5)] = static_cast<uint8_t>(sg);
            scales[row * 2 * s.blocks + s.blocks + (at.c >> 5)] = static_cast<uint8_t>(su);
          }
        }
      }
    }
  }
}

// The same 2.16 GB in 343 us, 2.70 GB with m in 435; GELU 412 and 441.  Four CTAs per SM: with 66 to 74 registers, three, it took
// 370 and 435, with five and 51 registers 381 and 459.
template <int ACT>
__global__ void __launch_bounds__(256, 4) glu_backward_kernel(Shape s, const __nv_bfloat16* d_m, int64_t pitch, const uint8_t* codes,
                                                           const uint8_t* scales, __nv_bfloat16* d_gate_up, __nv_bfloat16* m) {
  grid_enter(d_m, codes, scales);
  const Place at = place(s);
  if (!at.used) return;
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * s.rows * 2; base < s.R; base += static_cast<int64_t>(gridDim.x) * s.rows * 2) {
    uint4 raw[2] = {};
    uint2 cg[2], cu[2];
    uint32_t sg[2], su[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int64_t row = base + i * s.rows + at.row;
      if (row < s.R) {
        if (d_gate_up != nullptr) raw[i] = __ldg(reinterpret_cast<const uint4*>(d_m + row * pitch + at.c));
        cg[i] = __ldg(reinterpret_cast<const uint2*>(codes + row * 2 * s.I + at.c));
        cu[i] = __ldg(reinterpret_cast<const uint2*>(codes + row * 2 * s.I + s.I + at.c));
        sg[i] = __ldg(scales + row * 2 * s.blocks + (at.c >> 5));
        su[i] = __ldg(scales + row * 2 * s.blocks + s.blocks + (at.c >> 5));
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int64_t row = base + i * s.rows + at.row;
      if (row >= s.R) break;
      float d[8], g[8], u[8], dg[8], du[8], out[8];
      unpack8_bf16(raw[i], d);
      kept8(cg[i], sg[i], g);
      kept8(cu[i], su[i], u);
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        const float2 up = make_float2(u[j], u[j + 1]), dm = make_float2(d[j], d[j + 1]);
        float2 a, slope;
        act_and_slope<ACT>(make_float2(g[j], g[j + 1]), a, slope);
        const float2 v = mul2(a, up), vg = mul2(mul2(dm, up), slope), vu = mul2(dm, a);
        out[j] = v.x;
        out[j + 1] = v.y;
        dg[j] = vg.x;
        dg[j + 1] = vg.y;
        du[j] = vu.x;
        du[j + 1] = vu.y;
      }
      if (d_gate_up != nullptr) {
        *reinterpret_cast<uint4*>(d_gate_up + row * 2 * s.I + at.c) = pack8_bf16(dg);
        *reinterpret_cast<uint4*>(d_gate_up + row * 2 * s.I + s.I + at.c) = pack8_bf16(du);
      }
      if (m != nullptr) *reinterpret_cast<uint4*>(m + row * s.I + at.c) = pack8_bf16(out);
    }
  }
}

template <typename F>
int with_act(int act, const F& fn) {
  using std::integral_constant;
  switch (act) {
    case B200MOE_ACT_SILU: return fn(integral_constant<int, B200MOE_ACT_SILU>{});
    case B200MOE_ACT_GELU: return fn(integral_constant<int, B200MOE_ACT_GELU>{});
    case B200MOE_ACT_GELU_TANH: return fn(integral_constant<int, B200MOE_ACT_GELU_TANH>{});
    default: return fn(integral_constant<int, B200MOE_ACT_SWISH>{});
  }
}

Shape make_shape(int64_t R, int I) {
  const int blocks = (I + 31) / 32, pieces = blocks * 4, parts = (pieces + 255) / 256;
  const int width = ((pieces + parts - 1) / parts + 3) & ~3;
  return {R, I, blocks, width, 256 / width, (65536 + width - 1) / width};
}

unsigned threads_for(const Shape& s) { return static_cast<unsigned>((s.width * s.rows + 31) & ~31); }

dim3 grid_for(const Shape& s) {
  const int64_t parts = ceil_div64(s.blocks * 4, s.width), ctas = ceil_div64(s.R, s.rows * 2);
  const int64_t most = ceil_div64(static_cast<int64_t>(sm_count()) * 32, parts);
  return dim3(static_cast<unsigned>(ctas < most ? ctas : most), static_cast<unsigned>(parts));
}

int check_glu(const char* name, int64_t R, int I, int act, const void* in, int64_t pitch, int cols) {
  B200MOE_REQUIRE(R > 0 && R <= INT32_MAX && I > 0 && I % 8 == 0 && I <= (1 << 26), B200MOE_ERR_INVALID,
                  "%s: need at least one row and an intermediate size that is a positive multiple of 8", name);
  B200MOE_REQUIRE(act >= 0 && act <= 3, B200MOE_ERR_INVALID, "%s: unknown activation %d", name, act);
  B200MOE_REQUIRE((reinterpret_cast<uintptr_t>(in) & 15) == 0 && pitch % 8 == 0 && pitch >= cols, B200MOE_ERR_INVALID,
                  "%s: rows must start on 16-byte boundaries", name);
  return B200MOE_OK;
}

}  // namespace
}  // namespace b200moe

using namespace b200moe;

extern "C" int b200moe_glu(const void* gate_up_bf16, int64_t pitch, int64_t R, int I, int act_fn, void* m_bf16,
                           uint8_t* codes, uint8_t* scales, b200moe_stream_t stream) {
  B200MOE_REQUIRE(gate_up_bf16 && m_bf16 && (codes == nullptr) == (scales == nullptr), B200MOE_ERR_INVALID,
                  "glu: null pointer argument");
  const int rc = check_glu("glu", R, I, act_fn, gate_up_bf16, pitch, 2 * I);
  if (rc != B200MOE_OK) return rc;
  B200MOE_REQUIRE((reinterpret_cast<uintptr_t>(m_bf16) & 15) == 0 && (reinterpret_cast<uintptr_t>(codes) & 15) == 0,
                  B200MOE_ERR_INVALID, "glu: m and codes must be 16-byte aligned");
  const Shape s = make_shape(R, I);
  return with_act(act_fn, [&](auto act) -> int {
    constexpr int A = decltype(act)::value;
    B200MOE_CUDA_OK(launch_overlapped(codes != nullptr ? glu_kernel<A, true> : glu_kernel<A, false>, grid_for(s), threads_for(s), 0,
                                      static_cast<cudaStream_t>(stream), s, static_cast<const __nv_bfloat16*>(gate_up_bf16), pitch,
                                      static_cast<__nv_bfloat16*>(m_bf16), codes, scales));
    B200MOE_LAUNCH_OK("glu_kernel");
    return B200MOE_OK;
  });
}

extern "C" int b200moe_glu_backward(const void* d_m_bf16, int64_t pitch, const uint8_t* codes, const uint8_t* scales,
                                    int64_t R, int I, int act_fn, void* d_gate_up_bf16, void* m_bf16,
                                    b200moe_stream_t stream) {
  B200MOE_REQUIRE(codes && scales && (d_gate_up_bf16 || m_bf16) && (d_m_bf16 || !d_gate_up_bf16), B200MOE_ERR_INVALID,
                  "glu_backward: null pointer argument");
  const int rc = check_glu("glu_backward", R, I, act_fn, d_m_bf16, d_m_bf16 ? pitch : I, I);
  if (rc != B200MOE_OK) return rc;
  B200MOE_REQUIRE(((reinterpret_cast<uintptr_t>(codes) | reinterpret_cast<uintptr_t>(d_gate_up_bf16) |
                    reinterpret_cast<uintptr_t>(m_bf16)) & 15) == 0,
                  B200MOE_ERR_INVALID, "glu_backward: codes, d_gate_up and m must be 16-byte aligned");
  const Shape s = make_shape(R, I);
  return with_act(act_fn, [&](auto act) -> int {
    constexpr int A = decltype(act)::value;
    B200MOE_CUDA_OK(launch_overlapped(glu_backward_kernel<A>, grid_for(s), threads_for(s), 0, static_cast<cudaStream_t>(stream), s,
                                      static_cast<const __nv_bfloat16*>(d_m_bf16), pitch, codes, scales,
                                      static_cast<__nv_bfloat16*>(d_gate_up_bf16),
                                      static_cast<__nv_bfloat16*>(m_bf16)));
    B200MOE_LAUNCH_OK("glu_backward_kernel");
    return B200MOE_OK;
  });
}
