// The 8-bit linear for many token rows: bound by the tensor cores.
//
// Two CTAs of a cluster (two SMs) share one 256-token x 256-feature tile
// (cta_group::2): each stages its own 128 token rows and one half of the weight rows,
// so a block of k costs 32 KB of L2 reads per SM where a CTA alone with a 128 x 256 tile
// reads 48 KB, which is what bounded that form. The even CTA issues every MMA; each CTA
// holds the accumulators of its own tokens (lane = token) and folds them as in
// fp8_linear.cu, 8 warps of 128 columns each. The grid is one pair per two SMs and walks
// the tiles.
//
// An accumulator is busy from its first MMA to the last read of its fold, commit and
// barrier latencies included, and tensor memory holds two of 256 columns: taken whole,
// they left the tensor cores waiting half of the time. So a block's product is formed as
// two halves of 128 features, each with two accumulators and its own 4 fold warps: while
// one half is read the other half's MMAs run.
//
// Finished rows go through shared memory (one 256-byte row piece per lane in, whole lines
// out); a residual is fetched into the same place by asynchronous copies issued at the
// tile's start.
//
// Measured: 2048 x 4096 x 4096 35-36 us (1910-1960 TFLOP/s; its 128 tiles fill 1.7 of 2 rounds of
// 74 pairs), 8192^3 469-485 us (2270-2345 TFLOP/s) in a short burst and 515 us under sustained load,
// where the board's power limit sets the pace: the SM clock drops to 1.4-1.7 GHz. The
// tensor pipe is active 51% of the SM cycles at 2048 x 4096 x 4096 and L2 at 26% of its
// throughput: what is left there are the half-empty second round and the prologue. Tried
// without gain: two issuing warps, six stages, an undivided 256-column product, TMA stores.
#include <algorithm>
#include <type_traits>

#include "fp8_linear.cuh"

namespace aiosb {
namespace {

constexpr int kBN = 256;           // features per pair tile
constexpr int kCols = 128;         // columns of one fold warp
constexpr int kFoldWarps = 8;      // 4 groups of 32 TMEM lanes x 2 halves of the features
constexpr int kThreads = (kFoldWarps + 4) * 32;
constexpr int kAccs = 2;           // of each 128-feature half: all of tensor memory
constexpr int kHalf = kBN / 2;     // features of a half; each CTA stages 64 weight rows of it
constexpr uint32_t kHalfBytes = kHalf / 2 * kBK;
constexpr int kPairStages = 4;
constexpr int kWBlocks = kBN / kFp8Block;
constexpr uint32_t kABytes = kBM * kBK, kBBytes = kBN / 2 * kBK, kStageBytes = kABytes + kBBytes;
constexpr uint32_t kScaleOffset = kPairStages * kStageBytes;
constexpr uint32_t kScaleBytes = 2 * kScaleGroup * kWBlocks * kBM * 4;
constexpr uint32_t kOutOffset = kScaleOffset + kScaleBytes;
constexpr uint32_t kOutWarpBytes = 32 * kCols * 2;
constexpr uint32_t kSmemBytes = kOutOffset + kFoldWarps * kOutWarpBytes + 1024;

// TMA load of this CTA's tile whose bytes are counted on the mbarrier at a cluster
// address, here the even CTA's. Point to point: no multicast.
__device__ __forceinline__ void tma_load_2d_pair(void* dst, const CUtensorMap* map, uint32_t bar_cluster, int32_t x,
                                                 int32_t y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], "
      "[%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar_cluster), "r"(x), "r"(y)
      : "memory");
}
__device__ __forceinline__ void tc_mma_e4m3_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                                 uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Arrives on the barrier at this offset in both CTAs once the MMAs issued so far are done.
__device__ __forceinline__ void tc_commit_pair(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_u32(bar)),
      "h"((uint16_t)3)
      : "memory");
}
// Arrives on the even CTA's barrier. Nothing but finished tensor-memory loads is ordered
// by it, so it carries no cluster-wide fence (with .release.cluster the fence took 1400
// clocks per block).
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar_cluster) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar_cluster) : "memory");
}

__global__ void __launch_bounds__(kThreads, 1)
    linear_fp8_pair_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w,
                           const Fp8LinearArgs a) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  // full, acc_empty: the even CTA's are used; the others each CTA's own. done[h][s]: half h
  // of the block in stage s is in TMEM; with h = 1 the stage's operands are read, too
  __shared__ uint64_t full[kPairStages], done[2][kPairStages], acc_empty[2 * kAccs], scale_full[2], scale_empty[2];
  __shared__ uint32_t tmem_slot, far_blocks[2][kWBlocks];
  float* const scales = reinterpret_cast<float*>(smem + kScaleOffset);

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  if (threadIdx.x == 0) {
    for (int s = 0; s < kPairStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&done[0][s], 1);
      mbar_init(&done[1][s], 1);
    }
    for (int s = 0; s < 2 * kAccs; ++s) mbar_init(&acc_empty[s], kFoldWarps);  // half of the warps, of two CTAs
    for (int s = 0; s < 2; ++s) {
      mbar_init(&scale_full[s], 1);
      mbar_init(&scale_empty[s], kFoldWarps);
    }
    fence_mbar_init();
  }
  if (warp == kFoldWarps + 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)),
                 "r"(kAccs * kBN)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  if (warp == kFoldWarps && elect_one()) {
    tma_prefetch_desc(&tm_x);
    tma_prefetch_desc(&tm_w);
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // the barriers of both CTAs are initialised
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  pdl_wait();
  // after the wait: whoever follows may rely on this kernel's predecessors being done
  if (warp == kFoldWarps) pdl_launch_dependents();

  const int tiles = a.m_tiles * a.n_tiles;  // pair tiles
  const int first = blockIdx.x / 2, step = gridDim.x / 2;
  const int kblocks = a.kblocks;
  // Tiles in groups of 8 feature tiles, tokens inside: the pairs that run together read
  // few distinct rows of either operand.
  auto place = [&](int tile, int* m0, int* n0) {
    const int per = 8 * a.m_tiles, group = tile / per, rest = tile % per;
    const int width = min(8, a.n_tiles - group * 8);
    *n0 = (group * 8 + rest % width) * kBN;
    *m0 = rest / width * 2 * kBM + (int)rank * kBM;
  };
  bool ok = true;

  if (warp == kFoldWarps) {
    // ---- TMA producer: this CTA's tokens and its half of the weight rows
    int s = 0, issued = 0;
    uint32_t phase = 1;
    for (int tile = first; tile < tiles && ok; tile += step) {
      int m0, n0;
      place(tile, &m0, &n0);
      for (int kb = 0; kb < kblocks; ++kb) {
        ok = __all_sync(0xffffffffu, mbar_wait(&done[1][s], phase));
        if (!ok) break;
        if (elect_one()) {
          uint8_t* const dst = smem + s * kStageBytes;
          const uint32_t bar = map_shared_rank(smem_u32(&full[s]), 0);
          if (rank == 0) mbar_arrive_expect_tx(&full[s], 2 * kStageBytes);
          tma_load_2d_pair(dst, &tm_x, bar, kb * kBK, m0);
          tma_load_2d_pair(dst + kABytes, &tm_w, bar, kb * kBK, n0 + (int)rank * (kHalf / 2));
          tma_load_2d_pair(dst + kABytes + kHalfBytes, &tm_w, bar, kb * kBK, n0 + kHalf + (int)rank * (kHalf / 2));
        }
        issued = min(issued + 1, kPairStages);
        if (++s == kPairStages) {
          s = 0;
          phase ^= 1;
        }
      }
    }
    if (!ok && rank == 0) {  // let the pair's copies that are still in flight land before either CTA returns
      for (; issued > 0; --issued) {
        if (--s < 0) {
          s = kPairStages - 1;
          phase ^= 1;
        }
        mbar_wait(&full[s], phase ^ 1);
      }
    }
  } else if (warp == kFoldWarps + 1) {
    // ---- MMA issuer (even CTA). A half's accumulator waits for the folds of both CTAs, so
    // neither falls a whole ring of stages behind the done[] phases.
    if (rank == 0) {
      constexpr uint32_t idesc = umma_idesc_e4m3(2 * kBM, kHalf);
      const uint64_t a_desc = umma_desc_sw128(smem_u32(smem)), b_desc = umma_desc_sw128(smem_u32(smem + kABytes));
      int s = 0, t = 0;
      uint32_t phase = 0, acc_phase = 1;
      for (int tile = first; tile < tiles && ok; tile += step) {
        for (int kb = 0; kb < kblocks && ok; ++kb) {
          ok = __all_sync(0xffffffffu, mbar_wait(&full[s], phase));
          if (!ok) break;
          const uint32_t off = (uint32_t)s * (kStageBytes >> 4);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            ok = ok && __all_sync(0xffffffffu, mbar_wait(&acc_empty[2 * t + h], acc_phase));
            if (!ok) break;
            tc_fence_after();
            if (elect_one()) {
#pragma unroll
              for (int kk = 0; kk < kBK / 32; ++kk)
                tc_mma_e4m3_pair(tmem + (2 * t + h) * kHalf, a_desc + off + 2 * kk,
                                 b_desc + off + h * (kHalfBytes >> 4) + 2 * kk, idesc, kk != 0);
              tc_commit_pair(&done[h][s]);
            }
          }
          if (++s == kPairStages) {
            s = 0;
            phase ^= 1;
          }
          if (++t == kAccs) {
            t = 0;
            acc_phase ^= 1;
          }
        }
      }
    }
  } else if (warp == kFoldWarps + 2) {
    // ---- scale products of this CTA's tokens; lane l has rows l + 32 i
    int g = 0;
    uint32_t phase = 1;
    for (int tile = first; tile < tiles && ok; tile += step) {
      int m0, n0;
      place(tile, &m0, &n0);
      const float *sx[4], *sw[kWBlocks];
#pragma unroll
      for (int i = 0; i < 4; ++i) sx[i] = a.x_scale + (int64_t)min(m0 + i * 32 + lane, a.rows - 1) * kblocks;
#pragma unroll
      for (int b = 0; b < kWBlocks; ++b)
        sw[b] = a.w_scale + (int64_t)(min(n0 + b * kFp8Block, a.n - 1) / kFp8Block) * kblocks;
      for (int kb = 0; kb < kblocks; kb += kScaleGroup) {
        float x[4][kScaleGroup], w[kWBlocks][kScaleGroup];
#pragma unroll
        for (int j = 0; j < kScaleGroup; ++j) {
          const bool in = kb + j < kblocks;
#pragma unroll
          for (int i = 0; i < 4; ++i) x[i][j] = in ? sx[i][kb + j] : 1.f;
#pragma unroll
          for (int b = 0; b < kWBlocks; ++b) w[b][j] = in ? sw[b][kb + j] : 1.f;
        }
        ok = __all_sync(0xffffffffu, mbar_wait(&scale_empty[g], phase));
        if (!ok) break;
        ScaleRange range;
#pragma unroll
        for (int j = 0; j < kScaleGroup; ++j) {
#pragma unroll
          for (int b = 0; b < kWBlocks; ++b) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float p = x[i][j] * w[b][j];
              range.add(p);
              scales[((g * kScaleGroup + j) * kWBlocks + b) * kBM + i * 32 + lane] = p;
            }
          }
        }
        const bool any_far = __any_sync(0xffffffffu, range.far());
#pragma unroll
        for (int b = 0; b < kWBlocks; ++b) {
          uint32_t blocks = 0;
          if (any_far)
            blocks = split_group(x, w[b], sx, sw[b], kb, min(kScaleGroup, kblocks - kb),
                                 [&](int i, int j, float product, float) {
                                   scales[((g * kScaleGroup + j) * kWBlocks + b) * kBM + i * 32 + lane] = product;
                                 });
          if (lane == 0) far_blocks[g][b] = blocks;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&scale_full[g]);
        g ^= 1;
        if (g == 0) phase ^= 1;
      }
    }
  } else if (warp < kFoldWarps) {
    // ---- fold and store
    const int half = warp >> 2, lane_group = warp & 3;
    const uint32_t t_lane = tmem + ((uint32_t)(lane_group * 32) << 16) + (uint32_t)(half * kHalf);
    const float* const my_scales = scales + half * kBM + lane_group * 32 + lane;
    uint8_t* const out = smem + kOutOffset + warp * kOutWarpBytes;
    const uint32_t acc_bar = map_shared_rank(smem_u32(&acc_empty[half]), 0);
    int ring = 0, t = 0, g = 0;
    uint32_t phase = 0, g_phase = 0;
    for (int tile = first; tile < tiles && ok; tile += step) {
      int m0, n0;
      place(tile, &m0, &n0);
      const int r0 = m0 + lane_group * 32, c0 = n0 + half * kCols;
      // 16-byte piece `chunk` of row `row` of this warp's 32 x 128 outputs, the pieces of a
      // row permuted by the row so that both directions are free of bank conflicts
      const int chunk = lane & 15;
      const bool col_in = c0 + chunk * 8 < a.n;
      if (a.residual != nullptr) {
        __syncwarp();  // the previous tile's rows have been read out
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int row = i * 2 + (lane >> 4);
          if (col_in && r0 + row < a.rows)
            cp_async16(out + row * 256 + ((chunk ^ (row & 7)) << 4),
                       a.residual + (int64_t)(r0 + row) * a.residual_stride + c0 + chunk * 8);
        }
      }
      float2 acc[kCols / 2];
#pragma unroll
      for (int j = 0; j < kCols / 2; ++j) acc[j] = make_float2(0.f, 0.f);
      // One block of k; `far`: the group has products of scales that split_scales divides.
      auto fold_block = [&](int kb, int in_group, auto far) {
        ok = __all_sync(0xffffffffu, mbar_wait(&done[half][ring], phase));
        if (!ok) return;
        tc_fence_after();
        const float s1 = my_scales[(g * kScaleGroup + in_group) * kWBlocks * kBM];
        const float2 s = make_float2(s1, s1);
        float first = 1.f;
        if (far && ((far_blocks[g][half] >> in_group) & 1)) {
          float second;
          split_scales(a.x_scale[(int64_t)min(r0 + lane, a.rows - 1) * kblocks + kb],
                       a.w_scale[(int64_t)(min(c0, a.n - 1) / kFp8Block) * kblocks + kb], &first, &second);
        }
        // the next columns are on their way while kWide are folded; the rare form takes fewer at a
        // time, for its registers
        constexpr int kWide = decltype(far)::value ? 16 : 32;
        uint32_t d[2][kWide];
        tmem_ld(t_lane + t * kBN, d[0]);
        tmem_wait(d[0]);
#pragma unroll
        for (int c = 0; c < kCols / kWide; ++c) {
          if (c + 1 < kCols / kWide) {
            tmem_ld(t_lane + t * kBN + (c + 1) * kWide, d[(c + 1) & 1]);
          } else {  // this block's values are in registers: the accumulator may be reused
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(acc_bar + t * 16);
          }
          if (far) scale_all(d[c & 1], first);
#pragma unroll
          for (int j = 0; j < kWide / 2; ++j)
            acc[c * (kWide / 2) + j] = __ffma2_rn(
                s, make_float2(__uint_as_float(d[c & 1][2 * j]), __uint_as_float(d[c & 1][2 * j + 1])),
                acc[c * (kWide / 2) + j]);
          if (c + 1 < kCols / kWide) tmem_wait(d[(c + 1) & 1]);
        }
        if (++ring == kPairStages) {
          ring = 0;
          phase ^= 1;
        }
        t ^= 1;
      };
      for (int kb = 0; kb < kblocks && ok; kb += kScaleGroup) {
        const int count = min(kScaleGroup, kblocks - kb);
        ok = __all_sync(0xffffffffu, mbar_wait(&scale_full[g], g_phase));
        if (ok && far_blocks[g][half] == 0) {
#pragma unroll 1
          for (int j = 0; j < count && ok; ++j) fold_block(kb + j, j, std::false_type());
        } else {
#pragma unroll 1
          for (int j = 0; j < count && ok; ++j) fold_block(kb + j, j, std::true_type());
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&scale_empty[g]);
        g ^= 1;
        if (g == 0) g_phase ^= 1;
      }
      if (a.residual != nullptr) cp_async_wait_all();  // also where a wait ran out: nothing stays in flight
      if (!ok) break;
      __syncwarp();
#pragma unroll
      for (int c = 0; c < 16; ++c) {
        uint4* const at = reinterpret_cast<uint4*>(out + lane * 256 + ((c ^ (lane & 7)) << 4));
        float v[8] = {acc[4 * c].x,     acc[4 * c].y,     acc[4 * c + 1].x, acc[4 * c + 1].y,
                      acc[4 * c + 2].x, acc[4 * c + 2].y, acc[4 * c + 3].x, acc[4 * c + 3].y};
        if (a.residual != nullptr) {
          float r[8];
          unpack8(*at, r);
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] += r[j];
        }
        *at = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                         pack_bf16x2(v[6], v[7]));
      }
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int row = i * 2 + (lane >> 4);
        if (col_in && r0 + row < a.rows)
          *reinterpret_cast<uint4*>(a.y + (int64_t)(r0 + row) * a.y_stride + c0 + chunk * 8) =
              *reinterpret_cast<const uint4*>(out + row * 256 + ((chunk ^ (row & 7)) << 4));
      }
      __syncwarp();
    }
  }
  if (!ok) report(a.status, AIOSB_DEV_WAIT_TIMEOUT);

  __syncwarp();
  __syncthreads();
  tc_fence_before();
  cluster_sync();  // nothing of the pair is in flight any more: barriers, operands, accumulators
  if (warp == kFoldWarps + 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kAccs * kBN));
  }
}

}  // namespace

int fp8_linear_pair(const void* x, int64_t x_row_stride, int64_t k, const void* w, Fp8LinearArgs a,
                    cudaStream_t stream) {
  static bool configured[64] = {false};
  int rc = fp8_configure(linear_fp8_pair_kernel, (int)kSmemBytes, configured);
  if (rc != AIOSB_OK) return rc;
  a.m_tiles = (a.rows + 2 * kBM - 1) / (2 * kBM);
  a.n_tiles = (a.n + kBN - 1) / kBN;
  CUtensorMap tx, tw;
  rc = fp8_tensor_map(&tx, x, a.rows, k, x_row_stride, kBM);
  if (rc == AIOSB_OK) rc = fp8_tensor_map(&tw, w, a.n, k, k, kHalf / 2);
  if (rc != AIOSB_OK) return rc;
  const int pairs = std::min(a.m_tiles * a.n_tiles, std::max(1, sm_count() / 2));
  return fp8_launch(linear_fp8_pair_kernel, 2 * pairs, kThreads, (int)kSmemBytes, 2, stream, tx, tw, a);
}

}  // namespace aiosb
