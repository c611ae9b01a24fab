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

// act(g) and act'(g) in fp32.  SiLU, Swish and the tanh form of GELU are g sigma(z(g)): act' = sigma + g sigma (1 - sigma) z'.
template <int ACT>
__device__ __forceinline__ void act_and_slope(float g, float& act, float& slope) {
  if constexpr (ACT == B200MOE_ACT_GELU) {
    const float cdf = 0.5f * erfcf(-0.70710678118654752f * g);  // no cancellation for negative g
    act = g * cdf;
    slope = fmaf(g * 0.39894228040143268f, __expf(-0.5f * g * g), cdf);
  } else {
    float z, dz;
    if constexpr (ACT == B200MOE_ACT_SILU) {
      z = g;
      dz = 1.0f;
    } else if constexpr (ACT == B200MOE_ACT_SWISH) {
      z = 1.702f * g;
      dz = 1.702f;
    } else {  // (1 + tanh(z / 2)) / 2 = sigma(z)
      const float g2 = g * g;
      z = 1.5957691216057308f * g * fmaf(0.044715f, g2, 1.0f);
      dz = 1.5957691216057308f * fmaf(3.0f * 0.044715f, g2, 1.0f);
    }
    const float sigma = 1.0f / (1.0f + __expf(-z));
    act = g * sigma;
    slope = fmaf(act * (1.0f - sigma), dz, sigma);
  }
}

// The scale's exponent from the bits of the largest finite magnitude: 448 = 1.75 * 2^8.
__device__ __forceinline__ int scale_exponent(uint32_t top) {
  const int e = static_cast<int>(top >> 23) - 127 - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
  return max(e, -127);
}
__device__ __forceinline__ float power_of_two(int e) {  // e in [-149, 127]
  return e >= -126 ? __uint_as_float(static_cast<uint32_t>(e + 127) << 23) : __uint_as_float(1u << (e + 149));
}

// Eight values of a block that four neighbouring lanes hold: their codes and the block's scale byte.
__device__ __forceinline__ uint2 keep8(const float (&v)[8], int& scale_byte) {
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t b = __float_as_uint(v[j]) & 0x7fffffffu;
    top = max(top, b < 0x7f800000u ? b : 0u);
  }
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
  const int e = scale_exponent(top);
  scale_byte = e + 127;
  // v 2^-e in two exact steps: -e reaches 127 + 8
  const int n = -e, n0 = n >> 1;
  const float f0 = power_of_two(n0), f1 = power_of_two(n - n0);
  float x[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    x[j] = v[j] * f0 * f1;
    if (!(fabsf(v[j]) < INFINITY)) x[j] = __uint_as_float(0x7fc00000u);  // saturation would make 448 of an infinity
  }
  return make_uint2(pack4_e4m3(x[0], x[1], x[2], x[3]), pack4_e4m3(x[4], x[5], x[6], x[7]));
}

__device__ __forceinline__ void kept8(uint2 codes, int scale_byte, float (&v)[8]) {
  const float scale = power_of_two(scale_byte - 127);
  const uint32_t w[2] = {codes.x, codes.y};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_fp8x2_storage_t two = static_cast<__nv_fp8x2_storage_t>(w[i >> 1] >> (16 * (i & 1)));
    const __half2 h = __half2(__nv_cvt_fp8x2_to_halfraw2(two, __NV_E4M3));
    const float2 f = __half22float2(h);
    v[2 * i] = f.x * scale;
    v[2 * i + 1] = f.y * scale;
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

// Thread = eight columns of a row; rows are counted in whole blocks of 32 columns, so that a block's four lanes sit together.
__device__ __forceinline__ bool locate(int64_t i, int I, int blocks, int64_t& row, int& c) {
  row = i / (blocks * 4);
  c = static_cast<int>(i - row * (blocks * 4)) * 8;
  return c < I;
}

template <int ACT, bool KEEP>
__global__ void __launch_bounds__(256) glu_kernel(const __nv_bfloat16* gate_up, int64_t pitch, int64_t R, int I, int blocks,
                                                  __nv_bfloat16* m, uint8_t* codes, uint8_t* scales) {
  grid_enter(gate_up);
  const int64_t total = R * blocks * 4;
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * blockDim.x; base < total; base += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    int64_t row;
    int c;
    const int64_t i = base + threadIdx.x;
    const bool inside = locate(i, I, blocks, row, c) && i < total;
    float g[8] = {}, u[8] = {};
    if (inside) {
      unpack8_bf16(*reinterpret_cast<const uint4*>(gate_up + row * pitch + c), g);
      unpack8_bf16(*reinterpret_cast<const uint4*>(gate_up + row * pitch + I + c), u);
      float out[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float a, slope;
        act_and_slope<ACT>(g[j], a, slope);
        out[j] = a * u[j];
      }
      *reinterpret_cast<uint4*>(m + row * I + c) = pack8_bf16(out);
    }
    if constexpr (KEEP) {
      int sg, su;
      const uint2 cg = keep8(g, sg), cu = keep8(u, su);
      if (inside) {
        *reinterpret_cast<uint2*>(codes + row * 2 * I + c) = cg;
        *reinterpret_cast<uint2*>(codes + row * 2 * I + I + c) = cu;
        if ((threadIdx.x & 3) == 0) {
          scales[row * 2 * blocks + (c >> 5)] = static_cast<uint8_t>(sg);
          scales[row * 2 * blocks + blocks + (c >> 5)] = static_cast<uint8_t>(su);
        }
      }
    }
  }
}

template <int ACT>
__global__ void __launch_bounds__(256) glu_backward_kernel(const __nv_bfloat16* d_m, int64_t pitch, const uint8_t* codes,
                                                           const uint8_t* scales, int64_t R, int I, int blocks,
                                                           __nv_bfloat16* d_gate_up, __nv_bfloat16* m) {
  grid_enter(d_m, codes, scales);
  const int64_t total = R * blocks * 4;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < total; i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    int64_t row;
    int c;
    if (!locate(i, I, blocks, row, c)) continue;
    float d[8], g[8], u[8];
    if (d_gate_up != nullptr) unpack8_bf16(*reinterpret_cast<const uint4*>(d_m + row * pitch + c), d);
    const uint8_t* s = scales + row * 2 * blocks + (c >> 5);
    kept8(*reinterpret_cast<const uint2*>(codes + row * 2 * I + c), s[0], g);
    kept8(*reinterpret_cast<const uint2*>(codes + row * 2 * I + I + c), s[blocks], u);
    float dg[8], du[8], out[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float a, slope;
      act_and_slope<ACT>(g[j], a, slope);
      out[j] = a * u[j];
      dg[j] = d[j] * u[j] * slope;
      du[j] = d[j] * a;
    }
    if (d_gate_up != nullptr) {
      *reinterpret_cast<uint4*>(d_gate_up + row * 2 * I + c) = pack8_bf16(dg);
      *reinterpret_cast<uint4*>(d_gate_up + row * 2 * I + I + c) = pack8_bf16(du);
    }
    if (m != nullptr) *reinterpret_cast<uint4*>(m + row * I + c) = pack8_bf16(out);
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

unsigned grid_for(int64_t R, int blocks) {
  const int64_t ctas = ceil_div64(R * blocks * 4, 256), most = static_cast<int64_t>(sm_count()) * 8;
  return static_cast<unsigned>(ctas < most ? ctas : most);
}

int check_glu(const char* name, int64_t R, int I, int act, const void* in, int64_t pitch, int cols) {
  B200MOE_REQUIRE(R > 0 && R <= INT32_MAX && I > 0 && I % 8 == 0 && I <= (1 << 28), B200MOE_ERR_INVALID,
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
  const int blocks = (I + 31) / 32;
  return with_act(act_fn, [&](auto act) -> int {
    constexpr int A = decltype(act)::value;
    B200MOE_CUDA_OK(launch_overlapped(codes != nullptr ? glu_kernel<A, true> : glu_kernel<A, false>, dim3(grid_for(R, blocks)), 256,
                                      0, static_cast<cudaStream_t>(stream), static_cast<const __nv_bfloat16*>(gate_up_bf16),
                                      pitch, R, I, blocks, static_cast<__nv_bfloat16*>(m_bf16), codes, scales));
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
  const int blocks = (I + 31) / 32;
  return with_act(act_fn, [&](auto act) -> int {
    constexpr int A = decltype(act)::value;
    B200MOE_CUDA_OK(launch_overlapped(glu_backward_kernel<A>, dim3(grid_for(R, blocks)), 256, 0,
                                      static_cast<cudaStream_t>(stream), static_cast<const __nv_bfloat16*>(d_m_bf16), pitch,
                                      codes, scales, R, I, blocks, static_cast<__nv_bfloat16*>(d_gate_up_bf16),
                                      static_cast<__nv_bfloat16*>(m_bf16)));
    B200MOE_LAUNCH_OK("glu_backward_kernel");
    return B200MOE_OK;
  });
}
