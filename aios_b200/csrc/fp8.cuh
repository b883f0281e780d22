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
// max(|a|, |b|, |c|), NaN if any is (one instruction).
__device__ __forceinline__ float amax3_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float amax8_nan(const float (&v)[8]) {
  return amax_nan(amax3_nan(amax3_nan(amax3_nan(v[0], v[1], v[2]), v[3], v[4]), v[5], v[6]), v[7]);
}

struct Fp8Scale {
  float scale;  // value = q * scale
  float inv;    // q = e4m3(value * inv)
};
__device__ __forceinline__ Fp8Scale fp8_scale(float amax) {
  const float a = amax_nan(amax, kFp8MinAmax);
  return {__fdiv_rn(a, kFp8Max), __fdiv_rn(kFp8Max, a)};
}

// Scales of U blocks (1 to 4) whose lane maxima m[0..U) the 16 lanes of a half warp hold.
// The lanes share the blocks out as they reduce: each shuffle round halves the blocks that
// a lane still carries, until lane group `unit` holds block `unit` alone. That is 5 shuffles
// and one pair of divisions for four blocks instead of 16 and four pairs, and another 4 hand
// every lane every reciprocal. `unit`: the block of this lane's `scale`; `first`: whether it
// is the first lane that has it.
template <int U>
struct HalfWarpScales {
  float inv[U];
  float scale;
  int unit;
  bool first;

  __device__ __forceinline__ explicit HalfWarpScales(const float (&m)[U]) {
    const int lane = threadIdx.x & 31;
    float mine;
    int step;
    if (U == 1) {
      mine = m[0];
      step = 8;
      unit = 0;
    } else if (U == 2) {
      const bool hi = lane & 8;
      mine = amax_nan(hi ? m[U - 1] : m[0], __shfl_xor_sync(0xffffffffu, hi ? m[0] : m[U - 1], 8));
      step = 4;
      unit = hi;
    } else {
      constexpr int k1 = U > 1 ? 1 : 0, k2 = U > 2 ? 2 : 0;
      const float m3 = U > 3 ? m[U - 1] : 0.f;
      const bool hi = lane & 8, odd = lane & 4;
      const float x = amax_nan(hi ? m[k2] : m[0], __shfl_xor_sync(0xffffffffu, hi ? m[0] : m[k2], 8));
      const float y = amax_nan(hi ? m3 : m[k1], __shfl_xor_sync(0xffffffffu, hi ? m[k1] : m3, 8));
      mine = amax_nan(odd ? y : x, __shfl_xor_sync(0xffffffffu, odd ? x : y, 4));
      step = 2;
      unit = (hi ? 2 : 0) + (odd ? 1 : 0);
    }
    first = (lane & (2 * step - 1)) == 0;
#pragma unroll
    for (int o = 8; o > 0; o >>= 1)
      if (o <= step) mine = amax_nan(mine, __shfl_xor_sync(0xffffffffu, mine, o));
    const Fp8Scale f = fp8_scale(mine);
    scale = f.scale;
#pragma unroll
    for (int u = 0; u < U; ++u)
      inv[u] = U == 1 ? f.inv
                      : __shfl_sync(0xffffffffu, f.inv, (lane & 16) | (U == 2 ? u * 8 : (u >> 1) * 8 + (u & 1) * 4));
  }
};

// Eight values to eight e4m3 bytes, value 0 in the lowest byte. |v * inv| exceeds
// 448 by rounding at most, which rounds back to 448, so saturation changes nothing.
__device__ __forceinline__ uint2 fp8_pack8(const float (&v)[8], float inv) {
  uint32_t h[4];
  const float2 i2 = make_float2(inv, inv);
#pragma unroll
  for (int j = 0; j < 4; ++j)
    h[j] = __nv_cvt_float2_to_fp8x2(__fmul2_rn(make_float2(v[2 * j], v[2 * j + 1]), i2), __NV_SATFINITE, __NV_E4M3);
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
