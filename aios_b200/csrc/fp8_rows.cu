// Row kernels with 8-bit output: RMSNorm (with or without the residual's addition),
// SwiGLU and the plain quantiser of bf16 rows, plus the weight quantiser. Rows get
// one fp32 scale for each block of 128 columns, weights one for each 128 x 128
// block (fp8.cuh). All of them read each input once and write each output once, so
// HBM bounds them at size; the layouts below serve that: a lane holds 8 consecutive
// values (a 16-byte load), 16 lanes hold one block of 128, so the block's maximum is
// a few shuffles and a warp's loads and stores are whole lines.
//
// Measured (GB/s of the bytes that have to move; a copy reaches 6520): norm with residual of
// 16384 x 8192 137 us, 6850 GB/s; plain norm 79 us, 5130 GB/s (3 bytes a value where the
// residual's form moves 7, so the arithmetic shows); SwiGLU of 12001 x 10240 91 us, 6740 GB/s;
// rows of 16384 x 8192 66 us, 6110 GB/s; weight of 16384 x 8192 60.5 us, 6650 GB/s.
#include <algorithm>

#include "abi_util.h"
#include "fp8.cuh"

namespace aiosb {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ uint4 ld16(const __nv_bfloat16* p) { return *reinterpret_cast<const uint4*>(p); }

// ---- RMSNorm ------------------------------------------------------------------
struct NormArgs {
  const __nv_bfloat16* x;
  int64_t x_stride;
  const __nv_bfloat16* res;  // contiguous rows, or NULL
  __nv_bfloat16* res_out;    // may be res
  const __nv_bfloat16* w;
  int64_t rows;
  int hidden;
  float eps;
  uint8_t* q;
  float* scale;
};

// TPR threads share a row, U 16-byte units of it each (unit t + u * TPR), held in
// registers between the sum of squares and the quantised store: one pass over HBM.
// s = x [+ res] and everything after it stay in fp32 until the e4m3 rounding; only
// the stored residual is rounded to bf16, after the norm has taken the exact sum.
template <int TPR, int U, bool RES>
__global__ void __launch_bounds__(TPR == 32 ? kThreads : TPR) norm_fp8_kernel(const NormArgs a) {
  pdl_wait();
  if (threadIdx.x < 32) pdl_launch_dependents();
  __shared__ float scratch[32];
  const int64_t r = TPR == 32 ? (int64_t)blockIdx.x * (kThreads / 32) + threadIdx.x / 32 : (int64_t)blockIdx.x;
  const int t = TPR == 32 ? threadIdx.x & 31 : threadIdx.x;
  if (r >= a.rows) return;  // whole warps; with TPR > 32 the grid has no such row
  const int units = a.hidden / 8;
  const __nv_bfloat16* xr = a.x + r * a.x_stride;
  const int64_t base = r * a.hidden;
  // The weight comes with the row, so that its latency hides behind the row's (8 x 768: 2.2
  // -> 1.8 us), except with four units and no residual, where its registers cost occupancy. Late /
  // early there, us: 4096 x 1024 4.6 / 5.0, 8192 x 4096 20.6 / 21.3, 8192 x 16384 84.1 / 88.4; a
  // block to a row and few rows would gain: 2048 x 4096 7.4 / 7.3, 2048 x 8192 13.5 / 12.6, 1024 x
  // 16384 15.0 / 14.1; 16384 x 8192 78.7 / 77.9.
  constexpr bool kEarlyWeight = U < 4 || RES;
  uint4 xv[U], rv[U], wv[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int i = t + u * TPR;
    xv[u] = i < units ? ld16(xr + 8 * i) : make_uint4(0, 0, 0, 0);
    if (RES) rv[u] = i < units ? ld16(a.res + base + 8 * i) : make_uint4(0, 0, 0, 0);
    if (kEarlyWeight) wv[u] = i < units ? ld16(a.w + 8 * i) : make_uint4(0, 0, 0, 0);
  }
  float s[U][8];
  float2 ss2 = make_float2(0.f, 0.f);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int i = t + u * TPR;
    unpack8(xv[u], s[u]);
    if (RES) {
      float f[8];
      unpack8(rv[u], f);
#pragma unroll
      for (int j = 0; j < 8; ++j) s[u][j] += f[j];
      if (i < units)
        *reinterpret_cast<uint4*>(a.res_out + base + 8 * i) =
            make_uint4(pack_bf16x2(s[u][0], s[u][1]), pack_bf16x2(s[u][2], s[u][3]), pack_bf16x2(s[u][4], s[u][5]),
                       pack_bf16x2(s[u][6], s[u][7]));
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {  // packed: one instruction for two columns
      const float2 v = make_float2(s[u][2 * j], s[u][2 * j + 1]);
      ss2 = __ffma2_rn(v, v, ss2);
    }
  }
  float ss = ss2.x + ss2.y;
  ss = TPR == 32 ? warp_sum(ss) : block_sum(ss, scratch);
  const float rcp = 1.0f / sqrtf(ss / (float)a.hidden + a.eps);
  const float2 rcp2 = make_float2(rcp, rcp);
  float m[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int i = t + u * TPR;
    float g[8];
    if (!kEarlyWeight) wv[u] = i < units ? ld16(a.w + 8 * i) : make_uint4(0, 0, 0, 0);
    unpack8(wv[u], g);
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      const float2 v = __fmul2_rn(__fmul2_rn(make_float2(s[u][j], s[u][j + 1]), rcp2), make_float2(g[j], g[j + 1]));
      s[u][j] = v.x;
      s[u][j + 1] = v.y;
    }
    m[u] = amax8_nan(s[u]);
  }
  // lanes past the row's end hold zeros: 0 * rcp is NaN where the row's sum is, but they
  // share a block only with lanes of the same row, which are NaN too
  const HalfWarpScales<U> f(m);
  const int blocks = (a.hidden + kFp8Block - 1) / kFp8Block;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int i = t + u * TPR;
    if (i < units) *reinterpret_cast<uint2*>(a.q + base + 8 * i) = fp8_pack8(s[u], f.inv[u]);
  }
  const int b = ((t & ~15) + f.unit * TPR) / 16;
  if (f.first && f.unit < U && b < blocks) a.scale[r * blocks + b] = f.scale;
}

template <int TPR, int U>
cudaError_t launch_norm(const NormArgs& a, cudaStream_t s) {
  const unsigned grid = TPR == 32 ? (unsigned)((a.rows + kThreads / 32 - 1) / (kThreads / 32)) : (unsigned)a.rows;
  const dim3 block(TPR == 32 ? kThreads : TPR);
  return launch_pdl(a.res != nullptr ? norm_fp8_kernel<TPR, U, true> : norm_fp8_kernel<TPR, U, false>, dim3(grid),
                    block, 0, s, a);
}

// ---- SwiGLU and the plain quantiser ---------------------------------------------
// silu(g) * u of two columns, with the hardware exponential and reciprocal (each within a few
// units of 2^-23, the exponential's argument within 2^-24 of itself), far below the e4m3
// rounding that follows. In their flushing forms: a subnormal e^-g vanishes beside 1, and a
// subnormal reciprocal belongs to g < -87, which gives g * 0 (with their range checks, one column at
// a time, the SwiGLU of 12001 x 10240 took 102 us).
__device__ __forceinline__ float ex2_ftz(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float rcp_ftz(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float2 silu_mul2(float2 g, float2 u) {
  const float2 t = __fmul2_rn(g, make_float2(-1.4426950408889634f, -1.4426950408889634f));  // log2(e)
  const float2 d = __fadd2_rn(make_float2(1.f, 1.f), make_float2(ex2_ftz(t.x), ex2_ftz(t.y)));
  return __fmul2_rn(__fmul2_rn(g, make_float2(rcp_ftz(d.x), rcp_ftz(d.y))), u);
}

// One 16-lane group per block of 128 columns: group index = row * blocks + block.
// (rows * blocks stays below 2^31: that many blocks would be 275 G values.)
// UPT groups per thread, kThreads / 16 apart, to keep more loads in flight.
// x is not `const __restrict__`, here and in the weight's quantiser: the grid may start while
// its predecessor still writes x, and a load that is declared read-only for the grid's whole
// life need not stay behind pdl_wait().
template <bool SILU, int UPT>
__global__ void __launch_bounds__(kThreads)
    rows_fp8_kernel(const __nv_bfloat16* x, int64_t x_stride, uint32_t groups, uint32_t blocks, int cols, uint8_t* q,
                    float* scale) {
  pdl_wait();
  if (threadIdx.x < 32) pdl_launch_dependents();
  const int lane16 = threadIdx.x & 15;
  const uint32_t g0 = blockIdx.x * (uint32_t)(kThreads / 16 * UPT) + threadIdx.x / 16;
  uint4 gv[UPT], uv[UPT];
  int64_t row[UPT];
  int c[UPT];
  bool in[UPT];
#pragma unroll
  for (int k = 0; k < UPT; ++k) {
    const uint32_t g = g0 + k * (kThreads / 16);
    row[k] = g / blocks;
    c[k] = (int)(g % blocks) * kFp8Block + lane16 * 8;
    in[k] = g < groups && c[k] < cols;
    const __nv_bfloat16* p = x + row[k] * x_stride + c[k];
    gv[k] = in[k] ? ld16(p) : make_uint4(0, 0, 0, 0);
    if (SILU) uv[k] = in[k] ? ld16(p + cols) : make_uint4(0, 0, 0, 0);
  }
  float v[UPT][8], m[UPT];
#pragma unroll
  for (int k = 0; k < UPT; ++k) {
    unpack8(gv[k], v[k]);
    if (SILU) {
      float u[8];
      unpack8(uv[k], u);
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        const float2 y = silu_mul2(make_float2(v[k][j], v[k][j + 1]), make_float2(u[j], u[j + 1]));
        v[k][j] = y.x;
        v[k][j + 1] = y.y;
      }
    }
    m[k] = amax8_nan(v[k]);
  }
  const HalfWarpScales<UPT> f(m);
#pragma unroll
  for (int k = 0; k < UPT; ++k)
    if (in[k]) *reinterpret_cast<uint2*>(q + row[k] * cols + c[k]) = fp8_pack8(v[k], f.inv[k]);
  const uint32_t g = g0 + f.unit * (kThreads / 16);
  if (f.first && f.unit < UPT && g < groups) scale[g] = f.scale;
}

template <bool SILU, int UPT>
cudaError_t launch_rows_as(const __nv_bfloat16* x, int64_t x_stride, uint32_t groups, uint32_t blocks, int cols,
                           uint8_t* q, float* scale, cudaStream_t s) {
  constexpr uint32_t kPer = kThreads / 16 * UPT;
  return launch_pdl(rows_fp8_kernel<SILU, UPT>, dim3((groups + kPer - 1) / kPer), dim3(kThreads), 0, s, x, x_stride,
                    groups, blocks, cols, q, scale);
}

// Groups per thread, by the blocks of one group per thread that each SM gets: one while the SMs
// hold them all at once, then more for the loads in flight. With 1 / 2 / 4, in us:
//   SwiGLU of 1024 x 2048 (7 per SM) 3.5 / 4.0 / 4.0, 2048 x 2048 (14) 5.5 / 5.3 / 5.7,
//   2048 x 4096 (28) 9.6 / 8.7 / 8.9, 4096 x 4096 (55) 17.5 / 15.7 / 15.4, 12001 x 10240 112 / 97 / 91;
//   rows of 1024 x 2048 2.6 / 2.7 / 2.8, 2048 x 2048 4.1 / 4.1 / 3.9, 8192 x 8192 43 / 37 / 34.
template <bool SILU>
cudaError_t launch_rows(const void* x, int64_t x_stride, int64_t rows, int64_t cols, void* q, float* scale,
                        cudaStream_t s) {
  const uint32_t blocks = (uint32_t)((cols + kFp8Block - 1) / kFp8Block);
  const uint32_t groups = (uint32_t)rows * blocks;
  const uint32_t per_sm = groups / (kThreads / 16) / (uint32_t)sm_count();  // blocks of one group per thread
  auto launch = per_sm < 10 ? launch_rows_as<SILU, 1> : launch_rows_as<SILU, 4>;
  if constexpr (SILU)
    if (per_sm >= 10 && per_sm < 40) launch = launch_rows_as<SILU, 2>;
  return launch((const __nv_bfloat16*)x, x_stride, groups, blocks, (int)cols, (uint8_t*)q, scale, s);
}

// ---- weights ----------------------------------------------------------------------
// One CTA per 128 x 128 block: 16 lanes per row, 16 rows per pass, all eight passes'
// loads in flight before the block's maximum. It lets no kernel launch early: the
// linears that read the weight may be the next launch.
__global__ void __launch_bounds__(kThreads)
    weight_fp8_kernel(const __nv_bfloat16* w, int64_t w_stride, int64_t n, int64_t k, uint8_t* q, float* scale) {
  pdl_wait();
  __shared__ float part[kThreads / 32];
  constexpr int kPasses = kFp8Block / (kThreads / 16);
  const int64_t c = (int64_t)blockIdx.x * kFp8Block + (threadIdx.x & 15) * 8;
  const int64_t r0 = (int64_t)blockIdx.y * kFp8Block + threadIdx.x / 16;
  uint4 v[kPasses];
#pragma unroll
  for (int p = 0; p < kPasses; ++p) {
    const int64_t r = r0 + p * (kThreads / 16);
    v[p] = r < n && c < k ? ld16(w + r * w_stride + c) : make_uint4(0, 0, 0, 0);
  }
  float m = 0.f;
#pragma unroll
  for (int p = 0; p < kPasses; ++p) {
    float f[8];
    unpack8(v[p], f);
    m = amax_nan(m, amax8_nan(f));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = amax_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
  if ((threadIdx.x & 31) == 0) part[threadIdx.x / 32] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kThreads / 32; ++i) m = amax_nan(m, part[i]);
  const Fp8Scale f = fp8_scale(m);
#pragma unroll
  for (int p = 0; p < kPasses; ++p) {
    const int64_t r = r0 + p * (kThreads / 16);
    float u[8];
    unpack8(v[p], u);
    if (r < n && c < k) *reinterpret_cast<uint2*>(q + r * k + c) = fp8_pack8(u, f.inv);
  }
  if (threadIdx.x == 0) scale[(int64_t)blockIdx.y * gridDim.x + blockIdx.x] = f.scale;
}

constexpr int64_t kMaxHidden = 32768;  // 1024 threads x 4 units of 8

// Shared checks of the row entry points: `cols` values of a row.
int check_rows(const char* what, const void* x, int64_t rows, int64_t cols, int64_t row_values, int64_t x_row_stride,
               const void* q, const float* scale) {
  AIOSB_REQUIRE(rows >= 0 && cols > 0, AIOSB_ERR_INVALID_ARG, "%s: bad sizes", what);
  AIOSB_REQUIRE(rows < (int64_t)1 << 31 && cols < (int64_t)1 << 30 &&
                    rows * ((cols + kFp8Block - 1) / kFp8Block) < (int64_t)1 << 31,
                AIOSB_ERR_UNSUPPORTED, "%s: too many values", what);
  AIOSB_REQUIRE(cols % 16 == 0, AIOSB_ERR_UNSUPPORTED, "%s: %lld columns: must be a multiple of 16", what,
                (long long)cols);
  AIOSB_REQUIRE(x_row_stride >= row_values && x_row_stride % 8 == 0, AIOSB_ERR_INVALID_ARG,
                "%s: x row stride must cover the row and be a multiple of 8", what);
  if (rows == 0) return 1;
  AIOSB_REQUIRE(x && q && scale, AIOSB_ERR_INVALID_ARG, "%s: null pointer", what);
  AIOSB_REQUIRE(aligned16(x) && aligned16(q) && (reinterpret_cast<uintptr_t>(scale) & 3u) == 0,
                AIOSB_ERR_MISALIGNED, "%s: x and q must be 16-byte aligned", what);
  return AIOSB_OK;
}

}  // namespace
}  // namespace aiosb

using namespace aiosb;

extern "C" int aiosb_rmsnorm_fp8(const void* x, int64_t rows, int64_t hidden, int64_t x_row_stride,
                                 const void* residual, void* residual_out, const void* weight, float eps, void* q,
                                 float* scale, void* stream) {
  int rc = check_rows("rmsnorm_fp8", x, rows, hidden, hidden, x_row_stride, q, scale);
  if (rc < 0) return rc;
  AIOSB_REQUIRE(hidden <= kMaxHidden, AIOSB_ERR_UNSUPPORTED, "rmsnorm_fp8: at most %lld columns",
                (long long)kMaxHidden);
  AIOSB_REQUIRE((residual == nullptr) == (residual_out == nullptr), AIOSB_ERR_INVALID_ARG,
                "rmsnorm_fp8: residual and residual_out go together");
  if (rc == 1) return AIOSB_OK;
  AIOSB_REQUIRE(weight && aligned16(weight) && aligned16(residual) && aligned16(residual_out), AIOSB_ERR_MISALIGNED,
                "rmsnorm_fp8: weight and residual must be 16-byte aligned");
  const NormArgs a = {(const __nv_bfloat16*)x, x_row_stride, (const __nv_bfloat16*)residual,
                      (__nv_bfloat16*)residual_out, (const __nv_bfloat16*)weight, rows, (int)hidden, eps,
                      (uint8_t*)q, scale};
  cudaStream_t s = as_stream(stream);
  // The fewest threads per row that hold it in four units each: a warp needs no
  // block barrier, and more rows per SM hide the row's two dependent phases.
  const int units = (int)(hidden / 8);
  const int tpr = units <= 128 ? 32 : units <= 512 ? 128 : units <= 1024 ? 256 : units <= 2048 ? 512 : 1024;
  const int u = (units + tpr - 1) / tpr;
  cudaError_t e;
  switch (tpr * 8 + u) {
    case 32 * 8 + 1: e = launch_norm<32, 1>(a, s); break;
    case 32 * 8 + 2: e = launch_norm<32, 2>(a, s); break;
    case 32 * 8 + 3: e = launch_norm<32, 3>(a, s); break;
    case 32 * 8 + 4: e = launch_norm<32, 4>(a, s); break;
    case 128 * 8 + 2: e = launch_norm<128, 2>(a, s); break;
    case 128 * 8 + 3: e = launch_norm<128, 3>(a, s); break;
    case 128 * 8 + 4: e = launch_norm<128, 4>(a, s); break;
    case 256 * 8 + 3: e = launch_norm<256, 3>(a, s); break;
    case 256 * 8 + 4: e = launch_norm<256, 4>(a, s); break;
    case 512 * 8 + 3: e = launch_norm<512, 3>(a, s); break;
    case 512 * 8 + 4: e = launch_norm<512, 4>(a, s); break;
    case 1024 * 8 + 3: e = launch_norm<1024, 3>(a, s); break;
    default: e = launch_norm<1024, 4>(a, s); break;
  }
  return check_launch("rmsnorm_fp8", e);
}

extern "C" int aiosb_silu_mul_fp8(const void* x, int64_t rows, int64_t f, int64_t x_row_stride, void* q, float* scale,
                                  void* stream) {
  const int rc = check_rows("silu_mul_fp8", x, rows, f, 2 * f, x_row_stride, q, scale);
  if (rc != AIOSB_OK) return rc == 1 ? AIOSB_OK : rc;
  return check_launch("silu_mul_fp8", launch_rows<true>(x, x_row_stride, rows, f, q, scale, as_stream(stream)));
}

extern "C" int aiosb_quantize_fp8(const void* x, int64_t rows, int64_t cols, int64_t x_row_stride, void* q,
                                  float* scale, void* stream) {
  const int rc = check_rows("quantize_fp8", x, rows, cols, cols, x_row_stride, q, scale);
  if (rc != AIOSB_OK) return rc == 1 ? AIOSB_OK : rc;
  return check_launch("quantize_fp8", launch_rows<false>(x, x_row_stride, rows, cols, q, scale, as_stream(stream)));
}

extern "C" int aiosb_quantize_weight_fp8(const void* w, int64_t n, int64_t k, int64_t w_row_stride, void* q,
                                         float* scale, void* stream) {
  const int rc = check_rows("quantize_weight_fp8", w, n, k, k, w_row_stride, q, scale);
  if (rc != AIOSB_OK) return rc == 1 ? AIOSB_OK : rc;
  const int64_t tall = (n + kFp8Block - 1) / kFp8Block, wide = (k + kFp8Block - 1) / kFp8Block;
  AIOSB_REQUIRE(tall <= 65535, AIOSB_ERR_UNSUPPORTED, "quantize_weight_fp8: more than %lld rows",
                (long long)65535 * kFp8Block);
  return check_launch("quantize_weight_fp8",
                      launch_pdl(weight_fp8_kernel, dim3((unsigned)wide, (unsigned)tall), dim3(kThreads), 0,
                                 as_stream(stream), (const __nv_bfloat16*)w, w_row_stride, n, k, (uint8_t*)q, scale));
}
