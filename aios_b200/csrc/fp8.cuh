// 8-bit (e4m3) block quantisation shared by the row kernels and the weight
// quantiser. A block of 128 values y has
//   a = max(max |y|, 2^-100), scale = a / 448, q = e4m3(y * (448 / a)),
// 448 being the largest e4m3 value. The floor keeps the reciprocal finite for an
// all-zero block (q = 0, scale = 2^-100 / 448) and leaves every bf16 value that
// survives a product with anything of normal size unchanged. A NaN or an infinity
// in a block makes its scale NaN or infinite, so that it shows in every product
// instead of being clipped away: the maximum propagates NaN, and an infinite
// value's own q is inf * 0 = NaN.
// Rounding: one division for the reciprocal and one multiply, each to fp32 (off by
// 2^-24 of the value), ahead of the e4m3 rounding (off by 2^-4): multiplying by the
// reciprocal costs one instruction per value where a division would cost about ten.
#pragma once

#include <cuda_fp8.h>

#include "common.cuh"

namespace aiosb {

constexpr int kFp8Block = 128;
constexpr float kFp8Max = 448.0f;
constexpr float kFp8MinAmax = 0x1p-100f;

// max(a, |b|), NaN if either is.
__device__ __forceinline__ float amax_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(fabsf(b)));
  return r;
}

// Maximum over the 16 lanes of a half warp, NaN if any is; every lane gets it.
__device__ __forceinline__ float half_warp_amax(float a) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) a = amax_nan(a, __shfl_xor_sync(0xffffffffu, a, o));
  return a;
}

struct Fp8Scale {
  float scale;  // value = q * scale
  float inv;    // q = e4m3(value * inv)
};
__device__ __forceinline__ Fp8Scale fp8_scale(float amax) {
  const float a = amax_nan(amax, kFp8MinAmax);
  return {__fdiv_rn(a, kFp8Max), __fdiv_rn(kFp8Max, a)};
}

// Eight values to eight e4m3 bytes, value 0 in the lowest byte. |v * inv| exceeds
// 448 by rounding at most, which rounds back to 448, so saturation changes nothing.
__device__ __forceinline__ uint2 fp8_pack8(const float (&v)[8], float inv) {
  uint32_t h[4];
#pragma unroll
  for (int j = 0; j < 4; ++j)
    h[j] = __nv_cvt_float2_to_fp8x2(make_float2(v[2 * j] * inv, v[2 * j + 1] * inv), __NV_SATFINITE, __NV_E4M3);
  return make_uint2(h[0] | (h[1] << 16), h[2] | (h[3] << 16));
}

__device__ __forceinline__ void unpack8(const uint4& u, float (&v)[8]) {
  const uint32_t p[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    v[2 * j] = bf16_lo(p[j]);
    v[2 * j + 1] = bf16_hi(p[j]);
  }
}

}  // namespace aiosb
