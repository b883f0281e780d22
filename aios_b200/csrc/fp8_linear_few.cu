// The 8-bit linear for few token rows (decode): bound by the weight's bytes.
//
// The weight is the UMMA M operand (128 features per tile) and the tokens the N operand
// (16, 32 or 64 columns), so an MMA's time follows the token count: with the tokens as
// M, a decode step's MMAs would run at the speed of 128 rows. A TMEM lane is a feature,
// a column a token: the fold's scale is one product per column, the same for every lane,
// read from shared memory four at a time. Otherwise as fp8_linear.cu: a ring of TMA
// stages, four accumulators in turn, the products sx * sw formed eight blocks of k ahead
// by a warp of their own, and k split over a cluster whose partial tiles are summed in
// rank order.
//
// Measured: 1 x 8192 x 14336 21.9 us (5376 GB/s, 82% of measured HBM; 117.5 MB read, each
// weight byte once). A short k is latency: 8 x 1280 x 768 2.9 us and 8 x 768 x 2048 3.1 us in
// a chain of launches, for 0.15 and 0.24 us of bytes.
#include <algorithm>
#include <type_traits>

#include "fp8_linear.cuh"

namespace aiosb {
namespace {

template <int TN>
struct Few {
  static constexpr int kCols = TN < 32 ? TN : 32;      // tokens of one fold warp
  static constexpr int kFoldWarps = 4 * (TN / kCols);  // 4 groups of 32 TMEM lanes
  static constexpr int kThreads = (kFoldWarps + 4) * 32;
  static constexpr int kAccs = 4;
  // MMA warps, as in fp8_linear.cu: a second one gives 3% with 16 tokens (8 x 8192 x 8192 17.9 ->
  // 17.3 us) and costs 2 to 4% with 64
  static constexpr int kIssuers = TN == 16 ? 2 : 1;
  static constexpr int kTmemCols = kAccs * TN;         // 64, 128 or 256: two CTAs per SM
  static constexpr int kScaleBytes = 2 * 2 * kScaleGroup * TN * 4;
  static constexpr int kStageBytes = (kBM + TN) * kBK;
};
constexpr int kRedStride = kBM + 4;  // floats per token of the partial tile

template <int TN, bool RES>
__global__ void __launch_bounds__(Few<TN>::kThreads, 2)
    linear_fp8_few_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w,
                          const Fp8LinearArgs a) {
  using S = Few<TN>;
  constexpr int kCols = S::kCols, kFoldWarps = S::kFoldWarps, kAccs = S::kAccs;
  constexpr uint32_t kWBytes = kBM * kBK;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t full[kMaxStages], done[kMaxStages], acc_empty[kAccs], scale_full[2], scale_empty[2];
  __shared__ uint32_t tmem_slot, far_blocks[2];
  __shared__ volatile int abort_flag;
  // [2][kScaleGroup][TN], and as many first factors, written and read for far blocks only
  float* const scales = reinterpret_cast<float*>(smem_raw + a.scale_offset);
  constexpr int kFirsts = 2 * kScaleGroup * TN;

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < a.stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&done[s], 1);
    }
    for (int s = 0; s < kAccs; ++s) mbar_init(&acc_empty[s], kFoldWarps);
    for (int s = 0; s < 2; ++s) {
      mbar_init(&scale_full[s], 1);
      mbar_init(&scale_empty[s], kFoldWarps);
    }
    abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == kFoldWarps + 1) {
    tmem_alloc(&tmem_slot, S::kTmemCols);
    tmem_relinquish();
  }
  if (warp == kFoldWarps && elect_one()) {
    tma_prefetch_desc(&tm_x);
    tma_prefetch_desc(&tm_w);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;

  // m tiles are features, n tiles tokens; the token tiles of one feature tile are
  // neighbours, so that the second reads the weight from L2
  const int split = a.split, rank = blockIdx.x % split, tile = blockIdx.x / split;
  const int kb0 = (int)((int64_t)a.kblocks * rank / split), kb1 = (int)((int64_t)a.kblocks * (rank + 1) / split);
  const int f0 = tile / a.n_tiles * kBM, t0 = tile % a.n_tiles * TN;

  // The weight's first stages and scales are asked for before the dependency wait when the
  // caller vouches for them; everything else comes after it.
  if (warp != kFoldWarps && warp != kFoldWarps + 2) pdl_wait();

  if (warp == kFoldWarps) {
    // ---- TMA producer
    const int early = a.stable_weight ? min(kb1 - kb0, a.stages) : 0;
    if (early > 0 && elect_one()) {
      for (int i = 0; i < early; ++i) {
        mbar_arrive_expect_tx(&full[i], S::kStageBytes);
        tma_load_2d(smem + i * S::kStageBytes, &tm_w, &full[i], (kb0 + i) * kBK, f0);
      }
    }
    __syncwarp();
    pdl_wait();
    pdl_launch_dependents();  // after the wait: whoever follows may rely on this kernel's predecessors being done
    int s = 0, issued = 0;
    uint32_t phase = 1;
    bool ok = true;
    for (int kb = kb0; kb < kb1; ++kb) {
      ok = __all_sync(0xffffffffu, mbar_wait(&done[s], phase));
      if (!ok) break;
      if (elect_one()) {
        uint8_t* const dst = smem + s * S::kStageBytes;
        if (kb - kb0 >= early) {
          mbar_arrive_expect_tx(&full[s], S::kStageBytes);
          tma_load_2d(dst, &tm_w, &full[s], kb * kBK, f0);
        }
        tma_load_2d(dst + kWBytes, &tm_x, &full[s], kb * kBK, t0);
      }
      issued = min(issued + 1, a.stages);
      if (++s == a.stages) {
        s = 0;
        phase ^= 1;
      }
    }
    if (!ok) {  // let the copies that are still in flight land before this CTA returns
      report(a.status, AIOSB_DEV_WAIT_TIMEOUT);
      abort_flag = 1;
      for (; issued > 0; --issued) {
        if (--s < 0) {
          s = a.stages - 1;
          phase ^= 1;
        }
        mbar_wait(&full[s], phase ^ 1);
      }
    }
  } else if (warp == kFoldWarps + 1 || (S::kIssuers == 2 && warp == kFoldWarps + 3)) {
    // ---- MMA issuers, taking blocks in turn
    constexpr uint32_t idesc = umma_idesc_e4m3(kBM, TN);
    const uint64_t w_desc = umma_desc_sw128(smem_u32(smem)), x_desc = umma_desc_sw128(smem_u32(smem + kWBytes));
    int s = 0, t = 0;
    uint32_t phase = 0, acc_phase = 1;
    bool ok = true, mine = warp == kFoldWarps + 1;
    for (int kb = kb0; kb < kb1; ++kb, mine = S::kIssuers == 1 || !mine) {
      if (mine) {
        ok = __all_sync(0xffffffffu, mbar_wait(&acc_empty[t], acc_phase) && mbar_wait(&full[s], phase));
        if (!ok) break;
        tc_fence_after();
        const uint32_t off = (uint32_t)s * (S::kStageBytes >> 4);
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < kBK / 32; ++kk)
            tc_mma_e4m3(tmem + t * TN, w_desc + off + 2 * kk, x_desc + off + 2 * kk, idesc, kk != 0);
          tc_commit(&done[s]);
        }
      }
      if (++s == a.stages) {
        s = 0;
        phase ^= 1;
      }
      if (++t == kAccs) {
        t = 0;
        acc_phase ^= 1;
      }
    }
    if (!ok) {
      report(a.status, AIOSB_DEV_WAIT_TIMEOUT);
      abort_flag = 1;
    }
  } else if (warp == kFoldWarps + 2) {
    // ---- scale products, a group of blocks of k at a time; lane l has tokens l + 32 i
    constexpr int kPer = (TN + 31) / 32;
    const float* sx[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) sx[i] = a.x_scale + (int64_t)min(t0 + i * 32 + lane, a.rows - 1) * a.kblocks;
    const float* const sw = a.w_scale + (int64_t)(f0 / kFp8Block) * a.kblocks;
    int g = 0;
    uint32_t phase = 1;
    bool ok = true;
    if (!a.stable_weight) pdl_wait();
    for (int kb = kb0; kb < kb1; kb += kScaleGroup) {
      float x[kPer][kScaleGroup], w[kScaleGroup];
#pragma unroll
      for (int j = 0; j < kScaleGroup; ++j) w[j] = kb + j < kb1 ? sw[kb + j] : 1.f;
      if (a.stable_weight && kb == kb0) pdl_wait();
#pragma unroll
      for (int j = 0; j < kScaleGroup; ++j) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) x[i][j] = kb + j < kb1 ? sx[i][kb + j] : 1.f;
      }
      ok = __all_sync(0xffffffffu, mbar_wait(&scale_empty[g], phase));
      if (!ok) break;
      auto store = [&](int i, int j, float product, float first) {
        float* const at = scales + (g * kScaleGroup + j) * TN + i * 32 + lane;
        if (TN < 32 && lane >= TN) return;
        at[0] = product;
        at[kFirsts] = first;
      };
      ScaleRange range;
#pragma unroll
      for (int j = 0; j < kScaleGroup; ++j) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          const float p = x[i][j] * w[j];
          range.add(p);
          if (TN >= 32 || lane < TN) scales[(g * kScaleGroup + j) * TN + i * 32 + lane] = p;
        }
      }
      uint32_t blocks = 0;
      if (__any_sync(0xffffffffu, range.far()))
        blocks = split_group(x, w, sx, sw, kb, min(kScaleGroup, kb1 - kb), store);
      if (lane == 0) far_blocks[g] = blocks;
      __syncwarp();
      if (lane == 0) mbar_arrive(&scale_full[g]);
      g ^= 1;
      if (g == 0) phase ^= 1;
    }
    if (!ok) {
      report(a.status, AIOSB_DEV_WAIT_TIMEOUT);
      abort_flag = 1;
    }
  } else if (warp < kFoldWarps) {
    // ---- fold: acc[token] += (sx * sw)[token] * d[token] per block of k
    const int part = warp >> 2;
    const uint32_t t_lane = tmem + ((uint32_t)((warp & 3) * 32) << 16) + (uint32_t)(part * kCols);
    const float* const my_scales = scales + part * kCols;
    float2 acc[kCols / 2];
#pragma unroll
    for (int j = 0; j < kCols / 2; ++j) acc[j] = make_float2(0.f, 0.f);
    int ring = 0, t = 0, g = 0;
    uint32_t phase = 0, g_phase = 0;
    bool ok = true;
    // One block of k; `far`: the group has products of scales that split_scales divides.
    auto fold_block = [&](int in_group, auto far) {
      ok = __all_sync(0xffffffffu, mbar_wait(&done[ring], phase));
      if (!ok) return;
      tc_fence_after();
      const float* const block_scales = my_scales + (g * kScaleGroup + in_group) * TN;
      uint32_t d[kCols];
      tmem_ld(t_lane + t * TN, d);
      auto release = [&] {  // the block's values are in registers: the accumulator may be reused
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&acc_empty[t]);
      };
      if (far && ((far_blocks[g] >> in_group) & 1)) {  // a value at a time: few registers
        tmem_wait(d);
        release();
#pragma unroll
        for (int j = 0; j < kCols; ++j) {
          float& sum = j & 1 ? acc[j / 2].y : acc[j / 2].x;
          sum = fmaf(block_scales[j], __uint_as_float(d[j]) * block_scales[kFirsts + j], sum);
        }
      } else {
        float4 s[kCols / 4];
#pragma unroll
        for (int j = 0; j < kCols / 4; ++j) s[j] = *reinterpret_cast<const float4*>(block_scales + 4 * j);
        tmem_wait(d);
        release();
#pragma unroll
        for (int j = 0; j < kCols / 4; ++j) {
          acc[2 * j] = __ffma2_rn(make_float2(s[j].x, s[j].y),
                                  make_float2(__uint_as_float(d[4 * j]), __uint_as_float(d[4 * j + 1])), acc[2 * j]);
          acc[2 * j + 1] =
              __ffma2_rn(make_float2(s[j].z, s[j].w),
                         make_float2(__uint_as_float(d[4 * j + 2]), __uint_as_float(d[4 * j + 3])), acc[2 * j + 1]);
        }
      }
      if (++ring == a.stages) {
        ring = 0;
        phase ^= 1;
      }
      if (++t == kAccs) t = 0;
    };
    for (int kb = kb0; kb < kb1 && ok; kb += kScaleGroup) {
      const int count = min(kScaleGroup, kb1 - kb);
      ok = __all_sync(0xffffffffu, mbar_wait(&scale_full[g], g_phase));
      if (ok && far_blocks[g] == 0) {
#pragma unroll 1
        for (int j = 0; j < count && ok; ++j) fold_block(j, std::false_type());
      } else {
#pragma unroll 1
        for (int j = 0; j < count && ok; ++j) fold_block(j, std::true_type());
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&scale_empty[g]);
      g ^= 1;
      if (g == 0) g_phase ^= 1;
    }
    if (ok) {
      // every MMA of this CTA has read its operands: the partial tile takes their place
      float* const red = reinterpret_cast<float*>(smem) + part * kCols * kRedStride + (warp & 3) * 32 + lane;
#pragma unroll
      for (int j = 0; j < kCols / 2; ++j) {
        red[(2 * j) * kRedStride] = acc[j].x;
        red[(2 * j + 1) * kRedStride] = acc[j].y;
      }
    } else {
      report(a.status, AIOSB_DEV_WAIT_TIMEOUT);
      abort_flag = 1;
    }
  }

  __syncwarp();
  __syncthreads();
  const int live = min(a.rows - t0, TN);
  if (split == 1) {
    const float* const red = reinterpret_cast<const float*>(smem);
    constexpr int kUnits = (TN * (kBM / 8) + S::kThreads - 1) / S::kThreads;  // of a thread, at most
    uint4 res[kUnits];
    if (RES) {
#pragma unroll
      for (int i = 0; i < kUnits; ++i) {
        const int u = threadIdx.x + i * S::kThreads, r = u / (kBM / 8), c = u % (kBM / 8) * 8;
        if (r < live && f0 + c < a.n) res[i] = residual8(a, t0 + r, f0 + c);
      }
    }
    if (!abort_flag) {
#pragma unroll
      for (int i = 0; i < kUnits; ++i) {
        const int u = threadIdx.x + i * S::kThreads, r = u / (kBM / 8), c = u % (kBM / 8) * 8;
        if (r >= live || f0 + c >= a.n) continue;
        const float4 lo = *reinterpret_cast<const float4*>(red + r * kRedStride + c);
        const float4 hi = *reinterpret_cast<const float4*>(red + r * kRedStride + c + 4);
        const float2 v[4] = {{lo.x, lo.y}, {lo.z, lo.w}, {hi.x, hi.y}, {hi.z, hi.w}};
        store8<RES>(a, t0 + r, f0 + c, v, res[i]);
      }
    }
  } else {
    // Rank r sums and stores every split-th token: a warp reads whole lines of its peers'
    // partial tiles (16-byte pieces of many tokens took four times as long).
    constexpr int kUnits = (TN / 2 * (kBM / 4) + S::kThreads - 1) / S::kThreads;
    const int units = (live - rank + split - 1) / split * (kBM / 4);
    uint2 res[kUnits];
    if (RES) {
#pragma unroll
      for (int i = 0; i < kUnits; ++i) {
        const int u = threadIdx.x + i * S::kThreads, r = u / (kBM / 4) * split + rank, c = u % (kBM / 4) * 4;
        if (u < units && f0 + c < a.n) res[i] = residual4(a, t0 + r, f0 + c);
      }
    }
    cluster_sync();
    if (!abort_flag) {
      const uint32_t base = smem_u32(smem);
#pragma unroll
      for (int i = 0; i < kUnits; ++i) {
        const int u = threadIdx.x + i * S::kThreads, r = u / (kBM / 4) * split + rank, c = u % (kBM / 4) * 4;
        if (u < units && f0 + c < a.n)
          store4<RES>(a, t0 + r, f0 + c, sum_ranks4(base + (uint32_t)(r * kRedStride + c) * 4, split), res[i]);
      }
    }
    cluster_sync();  // peers may still read this CTA's partial tile
  }
  if (warp == kFoldWarps + 1) {
    tc_fence_after();
    tmem_dealloc(tmem, S::kTmemCols);
  }
}

template <int TN, bool RES>
int launch_few(const void* x, int64_t x_row_stride, int64_t k, const void* w, Fp8LinearArgs a, cudaStream_t stream) {
  using S = Few<TN>;
  constexpr int kBudget = 111 * 1024;  // two CTAs per SM
  auto kern = linear_fp8_few_kernel<TN, RES>;
  static bool configured[64] = {false};
  int rc = fp8_configure(kern, kBudget, configured);
  if (rc != AIOSB_OK) return rc;
  a.m_tiles = (a.n + kBM - 1) / kBM;
  a.n_tiles = (a.rows + TN - 1) / TN;
  const int tiles = a.m_tiles * a.n_tiles;
  const int per_cta = (a.kblocks + a.split - 1) / a.split;
  a.stages = std::max(S::kAccs, std::min({(kBudget - 1024 - S::kScaleBytes) / S::kStageBytes, kMaxStages, per_cta}));
  const int body = std::max(a.stages * S::kStageBytes, TN * kRedStride * 4);
  a.scale_offset = body + 1024;
  CUtensorMap tx, tw;
  rc = fp8_tensor_map(&tx, x, a.rows, k, x_row_stride, TN);
  if (rc == AIOSB_OK) rc = fp8_tensor_map(&tw, w, a.n, k, k, kBM);
  if (rc != AIOSB_OK) return rc;
  return fp8_launch(kern, tiles * a.split, S::kThreads, body + 1024 + S::kScaleBytes, a.split, stream, tx, tw, a);
}

template <bool RES>
int launch_tokens(int tokens, const void* x, int64_t x_row_stride, int64_t k, const void* w, const Fp8LinearArgs& a,
                  cudaStream_t stream) {
  if (tokens == 16) return launch_few<16, RES>(x, x_row_stride, k, w, a, stream);
  if (tokens == 32) return launch_few<32, RES>(x, x_row_stride, k, w, a, stream);
  return launch_few<64, RES>(x, x_row_stride, k, w, a, stream);
}

}  // namespace

int fp8_linear_few(int tokens, const void* x, int64_t x_row_stride, int64_t k, const void* w, Fp8LinearArgs a,
                   cudaStream_t stream) {
  return a.residual != nullptr ? launch_tokens<true>(tokens, x, x_row_stride, k, w, a, stream)
                               : launch_tokens<false>(tokens, x, x_row_stride, k, w, a, stream);
}

}  // namespace aiosb
