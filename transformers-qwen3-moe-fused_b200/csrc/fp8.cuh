// 8-bit activations: e4m3 codes with one power of two for each 128 values of a row.
//
//   scale = the smallest power of two with max|x| <= 448 scale (at least 2^-100), code = e4m3(x / scale), nearest, ties to even
// A power of two costs e4m3 nothing (its precision does not depend on the exponent; the largest code is between 224 and 448),
// x / scale is exact, and the codes are the same whatever precision they are computed in.  A block that holds an infinity or a
// NaN gets the scale NaN: the row's results become NaN, no other row's do.
#pragma once
#include <cuda_fp8.h>

#include "common.cuh"

namespace moe {

constexpr int FP8_BLOCK = 128;  // values that share a scale along a row; weights: 128 x 128

// Largest magnitude as the bits of |x|: ordered like the values, with infinity and NaN above all numbers.
__device__ __forceinline__ uint32_t magnitude_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// The scale of a block whose largest magnitude has these bits, and its reciprocal.
__device__ __forceinline__ float fp8_block_scale(uint32_t top, float& inverse) {
  if (top >= 0x7f800000u) {
    inverse = 0.f;
    return __uint_as_float(0x7fc00000u);
  }
  // 448 = 1.75 * 2^8
  int s = (int)(top >> 23) - 127 - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
  s = s < -100 ? -100 : s;
  inverse = __uint_as_float((uint32_t)(127 - s) << 23);
  return __uint_as_float((uint32_t)(127 + s) << 23);
}

__device__ __forceinline__ uint32_t fp8_pack4(float a, float b, float c, float d) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}

__device__ __forceinline__ float fp8_value(uint8_t code) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)code, __NV_E4M3)));
}

// Activation of the gated expert MLP and its gradients, fp32 throughout: h = silu(e) g.  fp32 tensors (T) take expf and the
// IEEE division, which the framework's other SiLU kernels keep for them too.  16-bit tensors take the fast forms, off by up to
// 4 + 1.2 |e| units of 2^-24, far below half a step of a code, 2^-4 (and 0 for e below -87.3, where the sigmoid is under 2^-126).
template <typename T>
__device__ __forceinline__ float gate_sigmoid(float e) {
  if constexpr (sizeof(T) == 4) return 1.f / (1.f + expf(-e));
  return __fdividef(1.f, 1.f + __expf(-e));
}
template <typename T>
__device__ __forceinline__ float gated_silu(float e, float g) { return e * gate_sigmoid<T>(e) * g; }
template <typename T>
__device__ __forceinline__ void gated_silu_bwd(float dh, float e, float g, float& de, float& dg) {
  const float sg = gate_sigmoid<T>(e);
  dg = dh * (e * sg);
  de = dh * g * (sg * fmaf(e, 1.f - sg, 1.f));
}

}  // namespace moe
