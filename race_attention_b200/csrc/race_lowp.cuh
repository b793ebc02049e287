// race_lowp.cuh -- device helpers of the 8-bit operators: rows in fp32 or bf16,
// the 8-bit format and its block scales.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace race {
namespace lowp {

using bf16 = __nv_bfloat16;

constexpr int kBlock = 128;                    // elements that share a scale
constexpr float kTop = 448.f;                  // largest value of the format
constexpr float kTiny = 1.17549435e-38f;       // 2^-126: smallest scale, 1 / s stays finite

template <typename T>
__device__ __forceinline__ float to_f32(T x) {
  if constexpr (sizeof(T) == 4) return x; else return __bfloat162float(x);
}
template <typename T>
__device__ __forceinline__ T from_f32(float x) {
  if constexpr (sizeof(T) == 4) return x; else return __float2bfloat16_rn(x);
}

// Eight consecutive elements, 16-byte aligned.
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
    const float4 a = *reinterpret_cast<const float4*>(p);
    const float4 b = *reinterpret_cast<const float4*>(p + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// Magnitudes are compared as integers: the order of their bits is that of
// their values, with infinity above every number and NaN above infinity, so a
// block's maximum is NaN as soon as one element is.
__device__ __forceinline__ uint32_t mag(float x) { return __float_as_uint(x) & 0x7fffffffu; }

__device__ __forceinline__ uint32_t max_over(uint32_t a, int lanes) {
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1)
    if (o < lanes) a = max(a, __shfl_xor_sync(0xffffffffu, a, o));
  return a;
}

// s = max(amax (1/448), 2^-126); NaN stays NaN.  The product with the rounded
// reciprocal, here and of x with 1 / s below, costs one instruction where a
// division costs ten; the largest element still lands on 448, which its code
// rounds to from either side.
__device__ __forceinline__ float scale_of(uint32_t amax) {
  const float s = __uint_as_float(amax) * (1.f / kTop);
  return s < kTiny ? kTiny : s;
}

// codes of x * inv for two and for eight values, lowest address first
__device__ __forceinline__ uint32_t code2(float a, float b) {
  return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ uint2 code8(const float (&v)[8], float inv) {
  uint2 c;
  c.x = code2(v[0] * inv, v[1] * inv) | code2(v[2] * inv, v[3] * inv) << 16;
  c.y = code2(v[4] * inv, v[5] * inv) | code2(v[6] * inv, v[7] * inv) << 16;
  return c;
}

}  // namespace lowp
}  // namespace race
