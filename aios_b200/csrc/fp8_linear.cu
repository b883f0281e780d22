// Linear with 8-bit operands: y[t, c] = [residual +] sum_b sx[t, b] sw[c / 128, b]
// sum_{k in block b} xq[t, k] wq[c, k] on e4m3 values with one fp32 scale for each
// 128 columns of an x row and for each 128 x 128 block of the weight.
//
// The tensor cores (tcgen05 kind::f8f6f4) form the sum over one 128-wide block of k
// at a time; its two scales belong to no operand, so each block's product is read
// from tensor memory and folded into fp32 registers as acc += (sx * sw) * d. x is the
// M operand: a TMEM lane is a token, its scale one register of the thread that reads
// the lane, and the weight's scale is uniform over the columns of a warp, so the fold
// costs one FMA per value. Four TMEM accumulators take turns: the tensor cores work
// on the next blocks while the warps fold one.
//
// Per CTA: the first 8 warps fold (warp w: lanes 32 (w % 4).., columns w / 4). Of the four
// warps after them one loads tiles by TMA into a ring of stages, two issue the MMAs in turn,
// and one forms the products sx * sw eight blocks of k at a time (in fp32; split_scales has
// those that fp32 does not hold) and hands them over in shared memory: read by the folding
// threads themselves, each row's scale is a cache line of its own, and fetching 32 lines per
// warp and block took as long as the MMAs.
// Few rows leave few tiles: then a cluster of up to 8 CTAs splits the blocks of k and
// the partial tiles are summed in rank order through distributed shared memory, so
// results do not depend on scheduling.
//
// These 128 x 128 tiles serve tens to hundreds of rows; fp8_linear_few.cu has the shape for fewer,
// fp8_linear_pair.cu for more, and choose() below picks. Measured: 77 x 10000 x 5008 16.8-17.9 us
// (its bytes take 8.0: 79 tiles leave half of the SMs idle, and a fold warp's wait, TMEM loads
// and FMAs take 460 clocks per block of k in the others; with k = 5120, rows on 128-byte lines,
// 14.2), 500 x 4096 x 768 6.0 us, 256 x 4096 x 4096 11.2 us, 512 x 8192 x 8192 35-40 us (1700-1970
// TFLOP/s, two rounds). Loading the next block's columns behind the last FMAs brought 2% at
// 77 x 10000 x 10240 and nothing elsewhere.
#include <string.h>

#include <algorithm>
#include <mutex>
#include <type_traits>

#include "fp8_linear.cuh"

namespace aiosb {
namespace {

constexpr int kBN = 128;                         // features per tile
constexpr int kCols = 64;                        // columns of one fold warp
constexpr int kFoldWarps = 4 * (kBN / kCols);    // 4 groups of 32 TMEM lanes
constexpr int kThreads = (kFoldWarps + 4) * 32;
constexpr int kAccs = 4;                         // TMEM accumulators in turn: all of tensor memory
// scale products: two groups of kScaleGroup blocks of k, 128 rows each
constexpr int kScaleBytes = 2 * kScaleGroup * kBM * 4;
// A bf16 tile of staging, at the price of a stage: the residual comes into it while the products
// are formed, and rows leave it in whole lines. With a row to a lane, 16 bytes at a time: 500 x
// 4096 x 768 6.6 -> 6.0 us, with a residual 8.6 -> 6.8; 128 x 10240 x 768 7.6 -> 6.1, with a residual
// 9.8 -> 6.8. (Tiles of 64 features, two CTAs to an SM, have no room for it and lost to these.)
constexpr int kPieces = kCols / 8;               // 16-byte pieces of a fold warp's row
constexpr int kOutWarpBytes = 32 * kCols * 2;
constexpr int kRedStride = kBN + 4;              // floats per row of the partial tile: free of bank conflicts

template <bool RES>
__global__ void __launch_bounds__(kThreads, 1)
    linear_fp8_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w,
                      const Fp8LinearArgs a) {
  constexpr uint32_t kBBytes = kBN * kBK;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t full[kMaxStages], done[kMaxStages], acc_empty[kAccs], scale_full[2], scale_empty[2];
  __shared__ uint32_t tmem_slot, far_blocks[2];
  __shared__ volatile int abort_flag;

  // the shuffle tells the compiler that the warp index, and every branch on it, is uniform
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t a_bytes = (uint32_t)a.a_rows * kBK;
  uint8_t* const smem_a = smem;
  uint8_t* const smem_b = smem + (uint32_t)a.stages * a_bytes;
  float* const scales = reinterpret_cast<float*>(smem_raw + a.scale_offset);
  // fold warps whose lanes hold tokens (a tile of fewer than 128 rows is the only m tile)
  const int lane_groups = (a.a_rows + 31) / 32;
  const bool folds = warp < kFoldWarps && (warp & 3) < lane_groups;

  if (threadIdx.x == 0) {
    for (int s = 0; s < a.stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&done[s], 1);
    }
    for (int s = 0; s < kAccs; ++s) mbar_init(&acc_empty[s], (uint32_t)lane_groups * (kBN / kCols));
    for (int s = 0; s < 2; ++s) {
      mbar_init(&scale_full[s], 1);
      mbar_init(&scale_empty[s], (uint32_t)lane_groups * (kBN / kCols));
    }
    abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == kFoldWarps + 1) {
    tmem_alloc(&tmem_slot, kAccs * kBN);
    tmem_relinquish();
  }
  if (threadIdx.x == kFoldWarps * 32) {
    tma_prefetch_desc(&tm_x);
    tma_prefetch_desc(&tm_w);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  pdl_wait();
  // after the wait: whoever follows may rely on this kernel's predecessors being done
  if (warp == kFoldWarps) pdl_launch_dependents();

  const int split = a.split;
  const int rank = blockIdx.x % split;
  const int kb0 = (int)((int64_t)a.kblocks * rank / split), kb1 = (int)((int64_t)a.kblocks * (rank + 1) / split);
  const int tiles = a.m_tiles * a.n_tiles;
  const int step = gridDim.x / split;

  // The two single-thread loops below pace everything, once per block of k: ring
  // positions and phases are counters (a division by the stage count costs more than
  // the MMAs of a narrow tile), descriptors are one addition, and a wait that runs out
  // ends its own role only (the other roles' waits then run out too).
  if (warp == kFoldWarps) {
    // ---- TMA producer
    int s = 0, issued = 0;
    uint32_t phase = 1;
    bool ok = true;
    for (int tile = blockIdx.x / split; tile < tiles && ok; tile += step) {
      const int m0 = tile % a.m_tiles * kBM, n0 = tile / a.m_tiles * kBN;
      for (int kb = kb0; kb < kb1; ++kb) {
        ok = __all_sync(0xffffffffu, mbar_wait(&done[s], phase));
        if (!ok) break;
        if (elect_one()) {
          mbar_arrive_expect_tx(&full[s], a_bytes + kBBytes);
          tma_load_2d(smem_b + s * kBBytes, &tm_w, &full[s], kb * kBK, n0);
          tma_load_2d(smem_a + s * a_bytes, &tm_x, &full[s], kb * kBK, m0);
        }
        issued = min(issued + 1, a.stages);
        if (++s == a.stages) {
          s = 0;
          phase ^= 1;
        }
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
  } else if (warp == kFoldWarps + 1 || warp == kFoldWarps + 3) {
    // ---- MMA issuers, two warps that take blocks in turn: a wait that is over and the issue
    // behind it take about 500 clocks of a warp, the MMAs of a block 256 (77 x 10000 x 10240 with
    // one warp 27.3 us, with two 23.9). With fewer than 128 rows staged the A operand's unused rows are
    // whatever follows the slot in shared memory (inside the allocation): a row of A
    // reaches its own TMEM lane only, and those lanes are not read.
    // One commit per block serves two readers of done[]: the producer (the stage's
    // operands are read) and the fold (the product is in TMEM). The fold cannot fall a
    // whole ring behind, because stages >= kAccs and an accumulator waits for its fold;
    // for the same reason one issuer is never more than kAccs blocks ahead of the other.
    constexpr uint32_t idesc = umma_idesc_e4m3(kBM, kBN);
    const uint64_t a_desc = umma_desc_sw128(smem_u32(smem_a)), b_desc = umma_desc_sw128(smem_u32(smem_b));
    int s = 0, t = 0;
    uint32_t phase = 0, acc_phase = 1;
    bool ok = true, mine = warp == kFoldWarps + 1;
    for (int tile = blockIdx.x / split; tile < tiles && ok; tile += step) {
      for (int kb = kb0; kb < kb1; ++kb, mine = !mine) {
        if (mine) {
          ok = __all_sync(0xffffffffu, mbar_wait(&acc_empty[t], acc_phase) && mbar_wait(&full[s], phase));
          if (!ok) break;
          tc_fence_after();
          const uint64_t da = a_desc + (uint32_t)s * (a_bytes >> 4), db = b_desc + (uint32_t)s * (kBBytes >> 4);
          if (elect_one()) {
#pragma unroll
            for (int kk = 0; kk < kBK / 32; ++kk)
              tc_mma_e4m3(tmem + t * kBN, da + 2 * kk, db + 2 * kk, idesc, kk != 0);
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
    }
    if (!ok) {
      report(a.status, AIOSB_DEV_WAIT_TIMEOUT);
      abort_flag = 1;
    }
  } else if (warp == kFoldWarps + 2) {
    // ---- scale products, a group of blocks of k at a time; lane l has rows l + 32 i
    int g = 0;
    uint32_t phase = 1;
    bool ok = true;
    for (int tile = blockIdx.x / split; tile < tiles && ok; tile += step) {
      const int m0 = tile % a.m_tiles * kBM, n0 = tile / a.m_tiles * kBN;
      const float *sx[4], *const sw = a.w_scale + (int64_t)(min(n0, a.n - 1) / kFp8Block) * a.kblocks;
#pragma unroll
      for (int i = 0; i < 4; ++i) sx[i] = a.x_scale + (int64_t)min(m0 + i * 32 + lane, a.rows - 1) * a.kblocks;
      for (int kb = kb0; kb < kb1; kb += kScaleGroup) {
        ok = mbar_wait(&scale_empty[g], phase);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        // every load of the group in flight before the first product
        float x[4][kScaleGroup], w[kScaleGroup];
#pragma unroll
        for (int j = 0; j < kScaleGroup; ++j) {
          const bool in = kb + j < kb1;
#pragma unroll
          for (int i = 0; i < 4; ++i) x[i][j] = in && i < lane_groups ? sx[i][kb + j] : 1.f;
          w[j] = in ? sw[kb + j] : 1.f;
        }
        auto store = [&](int i, int j, float product, float) {
          if (i < lane_groups) scales[(g * kScaleGroup + j) * kBM + i * 32 + lane] = product;
        };
        ScaleRange range;
#pragma unroll
        for (int j = 0; j < kScaleGroup; ++j) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float p = x[i][j] * w[j];
            range.add(p);
            store(i, j, p, 1.f);
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
    }
    if (!ok) {
      report(a.status, AIOSB_DEV_WAIT_TIMEOUT);
      abort_flag = 1;
    }
  } else if (folds) {
    // ---- fold: acc += (sx * sw) * d per block of k
    const int part = warp >> 2;  // columns [part * kCols, +kCols) of the tile
    const int tile_row = (warp & 3) * 32 + lane;
    const uint32_t t_lane = tmem + ((uint32_t)((warp & 3) * 32) << 16) + (uint32_t)(part * kCols);
    const float* const my_scales = scales + tile_row;
    int ring = 0, t = 0, g = 0;
    uint32_t phase = 0, g_phase = 0;
    bool ok = true;
    for (int tile = blockIdx.x / split; tile < tiles && ok; tile += step) {
      const int64_t row = (int64_t)(tile % a.m_tiles) * kBM + tile_row;
      const int c0 = tile / a.m_tiles * kBN + part * kCols;
      // 16-byte piece `piece` of a row of this warp's 32 x kCols outputs; in the staging the
      // pieces of a row are permuted by the row, so that both directions are free of conflicts
      const int piece = lane & (kPieces - 1);
      const int64_t row0 = row - lane;
      uint8_t* const out = smem_raw + a.scale_offset + kScaleBytes + warp * kOutWarpBytes;
      if (RES && split == 1) {  // the residual comes while the products are formed
        __syncwarp();  // the previous tile's rows have been read out
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
          const int r = i * (32 / kPieces) + lane / kPieces;
          if (row0 + r < a.rows && c0 + 8 * piece < a.n)
            cp_async16(out + r * (kCols * 2) + ((piece ^ (r & 7)) << 4),
                       a.residual + (row0 + r) * a.residual_stride + c0 + 8 * piece);
        }
      }
      float2 acc[kCols / 2];  // pairs of neighbouring columns: one packed FMA each
#pragma unroll
      for (int j = 0; j < kCols / 2; ++j) acc[j] = make_float2(0.f, 0.f);
      // One block of k; `far`: the group has products of scales that split_scales divides.
      auto fold_block = [&](int kb, int in_group, auto far) {
        ok = __all_sync(0xffffffffu, mbar_wait(&done[ring], phase));
        if (!ok) return;
        tc_fence_after();
        const float s1 = my_scales[(g * kScaleGroup + in_group) * kBM];
        const float2 s = make_float2(s1, s1);
        uint32_t d[kCols / 32][32];
#pragma unroll
        for (int l = 0; l < kCols / 32; ++l) tmem_ld(t_lane + t * kBN + l * 32, d[l]);
#pragma unroll
        for (int l = 0; l < kCols / 32; ++l) tmem_wait(d[l]);
        // this block's values are in registers: the accumulator may be reused
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&acc_empty[t]);
        if (far && ((far_blocks[g] >> in_group) & 1)) {
          float first, second;
          split_scales(a.x_scale[min(row, (int64_t)a.rows - 1) * a.kblocks + kb],
                       a.w_scale[(int64_t)(min(c0, a.n - 1) / kFp8Block) * a.kblocks + kb], &first, &second);
#pragma unroll
          for (int l = 0; l < kCols / 32; ++l) scale_all(d[l], first);
        }
#pragma unroll
        for (int j = 0; j < kCols / 2; ++j)
          acc[j] = __ffma2_rn(s,
                              make_float2(__uint_as_float(d[j / 16][2 * j % 32]),
                                          __uint_as_float(d[j / 16][2 * j % 32 + 1])),
                              acc[j]);
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
          for (int j = 0; j < count && ok; ++j) fold_block(kb + j, j, std::false_type());
        } else {
#pragma unroll 1
          for (int j = 0; j < count && ok; ++j) fold_block(kb + j, j, std::true_type());
        }
        if (!ok) {
          report(a.status, AIOSB_DEV_WAIT_TIMEOUT);
          abort_flag = 1;
          break;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&scale_empty[g]);
        g ^= 1;
        if (g == 0) g_phase ^= 1;
      }
      if (RES) cp_async_wait_all();  // also where a wait ran out: nothing stays in flight
      if (!ok) break;
      if (split == 1) {
        __syncwarp();  // copies of every lane have landed, and the previous tile's rows are out
#pragma unroll
        for (int j = 0; j < kPieces; ++j) {
          uint4* const at = reinterpret_cast<uint4*>(out + lane * (kCols * 2) + ((j ^ (lane & 7)) << 4));
          *at = RES ? add8(acc + 4 * j, *at) : pack8(acc + 4 * j);
        }
        __syncwarp();
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
          const int r = i * (32 / kPieces) + lane / kPieces;
          if (row0 + r < a.rows && c0 + 8 * piece < a.n)
            *reinterpret_cast<uint4*>(a.y + (row0 + r) * a.y_stride + c0 + 8 * piece) =
                *reinterpret_cast<const uint4*>(out + r * (kCols * 2) + ((piece ^ (r & 7)) << 4));
        }
      } else if (tile_row < a.a_rows) {
        // every MMA of this CTA has read its operands: the partial tile takes their place
        float* red = reinterpret_cast<float*>(smem) + tile_row * kRedStride + part * kCols;
#pragma unroll
        for (int j = 0; j < kCols / 2; j += 2)
          *reinterpret_cast<float4*>(red + 2 * j) = make_float4(acc[j].x, acc[j].y, acc[j + 1].x, acc[j + 1].y);
      }
    }
  }

  __syncwarp();
  __syncthreads();
  if (split > 1) {
    // Rank r sums and stores every split-th row: a warp reads whole lines of its peers'
    // partial tiles (16-byte pieces of many rows took four times as long).
    constexpr int kUnits = (kBM / 2 * (kBN / 4) + kThreads - 1) / kThreads;  // of a thread, at most
    const int tile = blockIdx.x / split;
    const int m0 = tile % a.m_tiles * kBM, n0 = tile / a.m_tiles * kBN;
    const int units = (min(a.rows - m0, kBM) - rank + split - 1) / split * (kBN / 4);
    uint2 res[kUnits];
    if (RES) {
#pragma unroll
      for (int i = 0; i < kUnits; ++i) {
        const int u = threadIdx.x + i * kThreads, r = u / (kBN / 4) * split + rank, c = u % (kBN / 4) * 4;
        if (u < units && n0 + c < a.n) res[i] = residual4(a, m0 + r, n0 + c);
      }
    }
    cluster_sync();
    if (!abort_flag) {
      const uint32_t base = smem_u32(smem);
#pragma unroll
      for (int i = 0; i < kUnits; ++i) {
        const int u = threadIdx.x + i * kThreads, r = u / (kBN / 4) * split + rank, c = u % (kBN / 4) * 4;
        if (u < units && n0 + c < a.n)
          store4<RES>(a, m0 + r, n0 + c, sum_ranks4(base + (uint32_t)(r * kRedStride + c) * 4, split), res[i]);
      }
    }
    cluster_sync();  // peers may still read this CTA's partial tile
  }
  if (warp == kFoldWarps + 1) {
    tc_fence_after();
    tmem_dealloc(tmem, kAccs * kBN);
  }
}

// ---- host side -------------------------------------------------------------------
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(p);
  });
  return fn;
}

}  // namespace

int fp8_tensor_map(CUtensorMap* m, const void* base, int64_t rows, int64_t cols, int64_t row_stride,
                   uint32_t box_rows) {
  EncodeTiledFn fn = encode_fn();
  if (fn == nullptr) return set_error(AIOSB_ERR_LAUNCH, "cuTensorMapEncodeTiled unavailable");
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)row_stride};
  const cuuint32_t box[2] = {(cuuint32_t)kBK, box_rows};
  const cuuint32_t estr[2] = {1, 1};
  CUresult r = fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return set_error(AIOSB_ERR_LAUNCH, "cuTensorMapEncodeTiled failed (%d)", (int)r);
  return AIOSB_OK;
}

namespace {

template <bool RES>
int launch(const CUtensorMap& tx, const CUtensorMap& tw, Fp8LinearArgs a, cudaStream_t stream) {
  constexpr int kBudget = 224 * 1024;  // one CTA per SM
  auto kern = linear_fp8_kernel<RES>;
  static bool configured[64] = {false};
  const int rc = fp8_configure(kern, kBudget, configured);
  if (rc != AIOSB_OK) return rc;
  const int stage_bytes = a.a_rows * kBK + kBN * kBK;
  const int out_bytes = a.split == 1 ? kFoldWarps * kOutWarpBytes : 0;
  const int tiles = a.m_tiles * a.n_tiles, slots = sm_count();
  const int per_cta = (a.kblocks + a.split - 1) / a.split * (a.split > 1 ? 1 : (tiles + slots - 1) / slots);
  a.stages =
      std::max(kAccs, std::min({(kBudget - 1024 - kScaleBytes - out_bytes) / stage_bytes, kMaxStages, per_cta}));
  // at least the partial tile, and 16 KB past the last A slot (the B slots have that)
  const int body = std::max(a.stages * stage_bytes, a.split > 1 ? a.a_rows * kRedStride * 4 : 0);
  a.scale_offset = body + 1024;
  return fp8_launch(kern, a.split > 1 ? tiles * a.split : std::min(tiles, slots), kThreads,
                    body + 1024 + kScaleBytes + out_bytes, a.split, stream, tx, tw, a);
}

// ---- choice of the kernel ----------------------------------------------------------
// Which tile, and how many ways k is split, by an estimate of the time of each: a start,
// a time per 128-wide block of k (more where two CTAs share an SM, and where the grid
// needs several rounds), and the cluster's cost where k is split. The figures were fitted
// to a sweep on a B200 of 272 sizes (8 to 2500 rows, 16 weights). Some of both sides, in us:
//   1 x 768 x 2048:     16-token tiles split in 8 3.1, in 4 3.5, whole 4.8
//   512 x 768 x 768:    32-token tiles 3.5, 64-token 4.1
//   128 x 768 x 2048:   32-token tiles split in 4 4.5, whole 5.8; 64-token in 4 5.3
//   128 x 10240 x 768:  128 x 128 tiles 6.1, 64-token tiles 6.6, the pair 8.0
//   77 x 10000 x 5008:  128 x 128 tiles 16.9, 64-token 26.2
//   300 x 1536 x 8960:  64-token tiles split in 4 14.3; 128 x 128 in 2 14.9, in 4 20.6
//   256 x 4096 x 4096:  128 x 128 tiles in 2 11.2, whole 12.6
//   512 x 4096 x 4096:  128 x 128 tiles 12.4, the pair 17.9
//   1024 x 4096 x 4096: the pair 19.1, 128 x 128 tiles 23.9
enum Kind { kFew, kTile, kPair };
struct ShapeCost {
  Kind kind;
  int rows, cols;              // tokens and features of a tile
  int per_sm;                  // CTAs an SM holds (the pair: half of one)
  float start, start_per_row;  // us
  float block, block_shared, block_rounds;
};
constexpr ShapeCost kShapes[] = {
    {kFew, 16, 128, 2, 2.38f, 0.f, 0.201f, 0.308f, 0.303f},
    {kFew, 32, 128, 2, 2.81f, 0.f, 0.238f, 0.344f, 0.396f},
    {kFew, 64, 128, 2, 2.82f, 0.f, 0.292f, 0.477f, 0.60f},
    {kTile, 128, 128, 1, 2.68f, 0.0059f, 0.286f, 0.286f, 0.355f},
    {kPair, 256, 256, 0, 5.19f, 0.f, 0.407f, 0.407f, 0.517f},
};
struct Choice {
  const ShapeCost* shape;
  int split;
};

Choice choose(int64_t rows, int64_t n, int kblocks, int sms) {
  const float weight_us = (float)n * (float)kblocks * kBK / 6.38e6f + 2.95f;  // the weight's bytes from HBM
  Choice best = {&kShapes[0], 1};
  float best_us = 1e30f;
  for (const ShapeCost& c : kShapes) {
    if (c.kind == kFew && c.rows == 16 && rows > 16) continue;  // half of a 32-token tile at the same cost
    const int64_t tiles = ((rows + c.rows - 1) / c.rows) * ((n + c.cols - 1) / c.cols);
    const float live = (float)std::min<int64_t>(rows, c.rows);
    for (int split = 1; split <= kMaxSplit && split <= kblocks; split *= 2) {
      if (split > 1 && (c.kind == kPair || tiles * split > 2 * sms)) break;
      // a cluster stays inside one group of SMs: those of 4 reach 132 of 148 SMs, of 8 120
      const int reach = std::max(1, split == 8 ? sms * 120 / 148 : split == 4 ? sms * 132 / 148 : sms);
      const int64_t ctas = tiles * split, slots = c.per_sm > 0 ? (int64_t)reach * c.per_sm : std::max(1, sms / 2);
      const float rounds = (float)((ctas + slots - 1) / slots);
      const bool crowded = c.per_sm == 2 && ctas > reach;
      const float block = rounds > 1.f ? c.block_rounds : crowded ? c.block_shared : c.block;
      float us = c.start + c.start_per_row * live + (crowded ? 1.1f : 0.f) +
                 rounds * ((float)((kblocks + split - 1) / split) * block + 0.54f) - 0.54f;
      if (split > 1) us += 1.32f + 0.0036f * live * (float)split;
      us = std::max(us, weight_us) + 0.1f * us;
      if (us < best_us) {
        best_us = us;
        best = {&c, split};
      }
    }
  }
  return best;
}

int check_sizes(int64_t rows, int64_t n, int64_t k) {
  AIOSB_REQUIRE(rows >= 0 && k > 0 && n > 0, AIOSB_ERR_INVALID_ARG, "linear_fp8: bad sizes");
  AIOSB_REQUIRE(n % 8 == 0, AIOSB_ERR_UNSUPPORTED, "linear_fp8: n=%lld must be a multiple of 8", (long long)n);
  AIOSB_REQUIRE(k % 16 == 0, AIOSB_ERR_UNSUPPORTED, "linear_fp8: k=%lld must be a multiple of 16", (long long)k);
  constexpr int64_t kMost = (int64_t)1 << 30;
  AIOSB_REQUIRE(rows <= kMost && n <= kMost && k <= kMost && (rows / kBM + 1) * (n / 64 + 1) < kMost,
                AIOSB_ERR_UNSUPPORTED, "linear_fp8: too large");
  return AIOSB_OK;
}

}  // namespace
}  // namespace aiosb

using namespace aiosb;

extern "C" int aiosb_linear_fp8(const void* x, int64_t x_row_stride, const float* x_scale, int64_t rows, int64_t k,
                                const void* w, const float* w_scale, int64_t n, void* y, int64_t y_row_stride,
                                int epilogue, const void* residual, int64_t residual_stride, int32_t* status,
                                void* stream) {
  const int sizes = check_sizes(rows, n, k);
  if (sizes != AIOSB_OK) return sizes;
  const int stable_weight = (epilogue & AIOSB_LINEAR_STABLE_WEIGHT) != 0;
  epilogue &= ~AIOSB_LINEAR_STABLE_WEIGHT;
  AIOSB_REQUIRE(epilogue == AIOSB_EPI_STORE || epilogue == AIOSB_EPI_ADD, AIOSB_ERR_INVALID_ARG,
                "linear_fp8: unknown epilogue %d (store or add)", epilogue);
  AIOSB_REQUIRE(epilogue != AIOSB_EPI_ADD ||
                    (residual != nullptr && aligned16(residual) && residual_stride >= n && residual_stride % 8 == 0),
                AIOSB_ERR_INVALID_ARG, "linear_fp8: the add epilogue needs an aligned residual [rows, >= n]");
  AIOSB_REQUIRE(x_row_stride >= k && x_row_stride % 16 == 0, AIOSB_ERR_INVALID_ARG,
                "linear_fp8: x row stride must cover the row and be a multiple of 16");
  AIOSB_REQUIRE(y_row_stride >= n && y_row_stride % 8 == 0, AIOSB_ERR_INVALID_ARG,
                "linear_fp8: y row stride must cover the output and be a multiple of 8");
  if (rows == 0) return AIOSB_OK;
  AIOSB_REQUIRE(x && x_scale && w && w_scale && y, AIOSB_ERR_INVALID_ARG, "linear_fp8: null pointer");
  AIOSB_REQUIRE(aligned16(x) && aligned16(w) && aligned16(y) && (reinterpret_cast<uintptr_t>(x_scale) & 3u) == 0 &&
                    (reinterpret_cast<uintptr_t>(w_scale) & 3u) == 0,
                AIOSB_ERR_MISALIGNED, "linear_fp8: x, w and y must be 16-byte aligned");
  Fp8LinearArgs a;
  memset(&a, 0, sizeof(a));
  a.x_scale = x_scale;
  a.w_scale = w_scale;
  a.y = (__nv_bfloat16*)y;
  a.y_stride = y_row_stride;
  a.residual = epilogue == AIOSB_EPI_ADD ? (const __nv_bfloat16*)residual : nullptr;
  a.residual_stride = residual_stride;
  a.rows = (int)rows;
  a.n = (int)n;
  a.kblocks = (int)((k + kBK - 1) / kBK);
  a.m_tiles = (int)((rows + kBM - 1) / kBM);
  a.a_rows = (int)std::min<int64_t>(kBM, (rows + 7) / 8 * 8);
  a.split = 1;
  a.stable_weight = stable_weight;
  a.status = status;
  const Choice c = choose(rows, n, a.kblocks, sm_count());
  cudaStream_t s = as_stream(stream);
  a.split = c.split;
  if (c.shape->kind == kFew) return fp8_linear_few(c.shape->rows, x, x_row_stride, k, w, a, s);
  if (c.shape->kind == kPair) return fp8_linear_pair(x, x_row_stride, k, w, a, s);
  a.n_tiles = (int)((n + kBN - 1) / kBN);
  CUtensorMap tx, tw;
  int rc = fp8_tensor_map(&tx, x, rows, k, x_row_stride, (uint32_t)a.a_rows);
  if (rc == AIOSB_OK) rc = fp8_tensor_map(&tw, w, n, k, k, kBN);
  if (rc != AIOSB_OK) return rc;
  return a.residual != nullptr ? launch<true>(tx, tw, a, s) : launch<false>(tx, tw, a, s);
}

extern "C" int aiosb_linear_fp8_plan(int64_t rows, int64_t n, int64_t k, int64_t sms, int32_t* plan) {
  const int sizes = check_sizes(rows, n, k);
  if (sizes != AIOSB_OK) return sizes;
  AIOSB_REQUIRE(rows > 0 && sms >= 0 && sms <= 65536 && plan != nullptr, AIOSB_ERR_INVALID_ARG,
                "linear_fp8_plan: no rows, bad SM count or null pointer");
  const Choice c = choose(rows, n, (int)((k + kBK - 1) / kBK), sms > 0 ? (int)sms : sm_count());
  plan[0] = c.shape->rows;
  plan[1] = c.shape->cols;
  plan[2] = c.split;
  return AIOSB_OK;
}
