// Shared by the 8-bit linear kernels: arguments, the tcgen05 / TMA / mbarrier pieces that
// only they use, and the epilogue's store.
#pragma once

#include <float.h>

#include "abi_util.h"
#include "fp8.cuh"

namespace aiosb {

constexpr int kBM = 128;                      // tokens per tile (UMMA M, TMEM lanes)
constexpr int kBK = kFp8Block;                // bytes of k per stage: one scale block, one swizzle row
constexpr int kMaxStages = 16;
constexpr int kMaxSplit = 8;
constexpr int kScaleGroup = 8;

struct Fp8LinearArgs {
  const float* x_scale;  // [rows, kblocks]
  const float* w_scale;  // [ceil(n / 128), kblocks]
  __nv_bfloat16* y;
  const __nv_bfloat16* residual;  // or NULL
  int64_t y_stride, residual_stride;
  int rows, n, kblocks;
  int m_tiles, n_tiles;
  int split;
  int stages;
  int scale_offset;  // of the scale products, bytes from the start of dynamic shared memory
  int a_rows;  // token rows a stage holds: rows, rounded up to the swizzle's 8, at most 128
  int stable_weight;  // AIOSB_LINEAR_STABLE_WEIGHT
  int32_t* status;
};

__device__ __forceinline__ void tc_mma_e4m3(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Instruction descriptor: fp32 accumulator, e4m3 A and B (format 0), both K-major.
__host__ __device__ constexpr uint32_t umma_idesc_e4m3(int M, int N) {
  return (1u << 4) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}

// ---- results: sums of one row to bf16; the residual is added in fp32 (one rounding).
// A thread loads all of its pieces of the residual before its first store: the output may be
// the residual's own memory, so the compiler keeps a load behind every store before it, and
// 500 x 4096 x 768 spent 3.2 us on those round trips one after another. The kernels with a
// residual are instances of their own: what they hold in registers cost the others 2%.
__device__ __forceinline__ uint4 residual8(const Fp8LinearArgs& a, int64_t row, int col) {
  return *reinterpret_cast<const uint4*>(a.residual + row * a.residual_stride + col);
}
__device__ __forceinline__ uint2 residual4(const Fp8LinearArgs& a, int64_t row, int col) {
  return *reinterpret_cast<const uint2*>(a.residual + row * a.residual_stride + col);
}
__device__ __forceinline__ uint4 pack8(const float2* v) {
  return make_uint4(pack_bf16x2(v[0].x, v[0].y), pack_bf16x2(v[1].x, v[1].y), pack_bf16x2(v[2].x, v[2].y),
                    pack_bf16x2(v[3].x, v[3].y));
}
__device__ __forceinline__ uint4 add8(const float2* v, const uint4& residual) {
  float r[8];
  unpack8(residual, r);
  return make_uint4(pack_bf16x2(v[0].x + r[0], v[0].y + r[1]), pack_bf16x2(v[1].x + r[2], v[1].y + r[3]),
                    pack_bf16x2(v[2].x + r[4], v[2].y + r[5]), pack_bf16x2(v[3].x + r[6], v[3].y + r[7]));
}
template <bool RES>
__device__ __forceinline__ void store8(const Fp8LinearArgs& a, int64_t row, int col, const float2* v,
                                       const uint4& residual) {
  *reinterpret_cast<uint4*>(a.y + row * a.y_stride + col) = RES ? add8(v, residual) : pack8(v);
}
template <bool RES>
__device__ __forceinline__ void store4(const Fp8LinearArgs& a, int64_t row, int col, float4 v, const uint2& r) {
  if (RES) {
    v.x += bf16_lo(r.x);
    v.y += bf16_hi(r.x);
    v.z += bf16_lo(r.y);
    v.w += bf16_hi(r.y);
  }
  *reinterpret_cast<uint2*>(a.y + row * a.y_stride + col) = make_uint2(pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w));
}

// Four neighbouring floats at shared-memory offset `off`, summed over the first `split`
// CTAs of the cluster in rank order. Every rank's load is issued before the first sum: one
// round trip to the peers, not one per rank.
__device__ __forceinline__ float4 sum_ranks4(uint32_t off, int split) {
  float4 part[kMaxSplit];
#pragma unroll
  for (int p = 0; p < kMaxSplit; ++p)
    if (p < split) part[p] = ld_dsmem_f4(map_shared_rank(off, (uint32_t)p));
  float4 v = part[0];
#pragma unroll
  for (int p = 1; p < kMaxSplit; ++p) {
    if (p < split) {
      v.x += part[p].x;
      v.y += part[p].y;
      v.z += part[p].z;
      v.w += part[p].w;
    }
  }
  return v;
}

// ---- scales ------------------------------------------------------------------------
// A block's product d (0, or 2^-18 to 448 * 448 * 128) counts x * w * d, with x * w formed once
// for all of its values. Where x * w overflows, or falls so low that its rounding to a subnormal
// would show (below 2^-134 it is off by more than 2^-16 of itself), the scales are applied one
// after the other instead: d * first keeps in range with the smaller one first where x * w is
// too large, with the larger one first where it is too small. (Below 2^-176 no d brings the
// product back into fp32.) A value's bits do not depend on its neighbours' scales: d * 1 is d.
// The range of the products that a lane forms, in two instructions each (a comparison of each
// product with both limits kept the scale warp behind the fold: 256 x 4096 x 4096 11.3 -> 13.1 us).
struct ScaleRange {
  float lo = 1.f, hi = 1.f;
  __device__ __forceinline__ void add(float p) {
    lo = fminf(lo, fabsf(p));
    hi = fmaxf(hi, fabsf(p));
  }
  __device__ __forceinline__ bool far() const { return lo < 0x1p-134f || hi > FLT_MAX; }
};
__device__ __forceinline__ bool splits(float x, float w) {
  const float p = fabsf(x * w), lo = fminf(fabsf(x), fabsf(w)), hi = fmaxf(fabsf(x), fabsf(w));
  // not where a scale itself is zero, infinite or NaN
  return (p > FLT_MAX && hi <= FLT_MAX) || (p < 0x1p-134f && lo * 0x1p26f * hi != 0.f);
}
__device__ __forceinline__ void split_scales(float x, float w, float* first, float* second) {
  const float p = x * w;
  const bool x_first = (fabsf(p) > FLT_MAX) == (fabsf(x) <= fabsf(w));
  const bool split = splits(x, w);
  *first = !split ? 1.f : x_first ? x : w;
  *second = !split ? p : x_first ? w : x;
}
template <int N>
__device__ __forceinline__ void scale_all(uint32_t (&d)[N], float first) {
#pragma unroll
  for (int j = 0; j < N; ++j) d[j] = __float_as_uint(__uint_as_float(d[j]) * first);
}
// Behind ScaleRange: the blocks (bits) among `count` from `kb` on whose products need split_scales
// in any of the warp's rows (kRows a lane); their factors go to store(row, block, second, first).
// Most of what leaves the range are scales of 0, which some quantisers give empty rows: those are
// told apart in registers. Factors are written from scales that are read again.
template <int kRows, typename Store>
__device__ __forceinline__ uint32_t split_group(const float (&x)[kRows][kScaleGroup], const float (&w)[kScaleGroup],
                                                const float* const (&sx)[kRows], const float* sw, int kb, int count,
                                                Store store) {
  bool any = false;
#pragma unroll
  for (int j = 0; j < kScaleGroup; ++j) {
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const float p = fabsf(x[i][j] * w[j]);
      any |= (p < 0x1p-134f || p > FLT_MAX) && fminf(fabsf(x[i][j]), fabsf(w[j])) > 0.f;
    }
  }
  uint32_t blocks = 0;
  if (!__any_sync(0xffffffffu, any)) return blocks;
#pragma unroll 1
  for (int j = 0; j < count; ++j) {
    bool split = false;
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      float first, second;
      split_scales(sx[i][kb + j], sw[kb + j], &first, &second);
      split |= splits(sx[i][kb + j], sw[kb + j]);
      store(i, j, second, first);
    }
    blocks |= (uint32_t)__any_sync(0xffffffffu, split) << j;
  }
  return blocks;
}

// ---- host side -------------------------------------------------------------------
// Tensor map of a row-major byte matrix [rows, cols] in boxes of box_rows x 128; reads
// past an edge give zeros.
int fp8_tensor_map(CUtensorMap* m, const void* base, int64_t rows, int64_t cols, int64_t row_stride,
                   uint32_t box_rows);

// Opts `kern` into `bytes` of dynamic shared memory once per device.
template <typename Kern>
int fp8_configure(Kern kern, int bytes, bool (&configured)[64]) {
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !configured[dev]) {
    const int rc =
        check_launch("linear_fp8", cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    if (rc != AIOSB_OK) return rc;
    if (dev >= 0 && dev < 64) configured[dev] = true;
  }
  return AIOSB_OK;
}

// Launches with programmatic dependent launch, in clusters of `cluster` CTAs along x.
template <typename Kern>
int fp8_launch(Kern kern, int grid, int threads, int smem, int cluster, cudaStream_t stream, const CUtensorMap& tx,
               const CUtensorMap& tw, const Fp8LinearArgs& a) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return check_launch("linear_fp8", cudaLaunchKernelEx(&cfg, kern, tx, tw, a));
}

// Many token rows: two CTAs share a 256 x 256 tile (fp8_linear_pair.cu).
int fp8_linear_pair(const void* x, int64_t x_row_stride, int64_t k, const void* w, Fp8LinearArgs a,
                    cudaStream_t stream);
// Few token rows: the weight is the M operand, `tokens` (16, 32, 64) rows to a tile; a.split
// is set (fp8_linear_few.cu).
int fp8_linear_few(int tokens, const void* x, int64_t x_row_stride, int64_t k, const void* w, Fp8LinearArgs a,
                   cudaStream_t stream);

}  // namespace aiosb
