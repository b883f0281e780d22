// Attention of drafted trees, the keys of all requests dealt evenly over the SMs.
//
// A unit is up to 256 rows ((node, query head) pairs) of one KV head of one request; its keys are
// chunks of 128. The units' chunks laid end to end, each weighed by what it costs, are cut into one
// range per CTA, so that a CTA takes pieces of units, whatever the requests' lengths. A piece that is a
// whole unit is written as it is; the pieces of a cut unit leave their rows' maximum, sum and
// unnormalised output in fp32 in the work area, and a second kernel joins them in the order of the keys.
//
// In a CTA: four warps walk the CTA's pieces and gather their keys and values into a ring of 128-key
// blocks with cp.async (the slots of neighbouring keys are anywhere, so there is no box for TMA to
// fetch); two warps issue the MMAs, one for each of two streams; and two groups of four warps hold the
// streams' softmax. With more than 128 rows the streams are the two halves of the rows, both on every
// chunk; with fewer they are the even and the odd chunks of the same rows, each with its own maximum,
// sum and output, joined at the end. S = Q K^T goes from shared memory into TMEM, 64 keys at a time into
// two buffers, so that a stream's next scores are formed while it takes the present exponentials. A
// thread owns a row (a TMEM lane), takes its maximum and exponentials, and writes the weights back over
// S as bf16 A operands of O += P V (V as it lies, the keys as its k: an MN-major B operand), one of their
// upper and one of their lower halves, which together fill S's place (split_bf16x2). Up to 32
// rows go on mma.sync instead, with no TMEM round trip (few_rows below).
// A row's output is rescaled only where its maximum has grown by more than 2^8 over the one that its
// exponentials refer to: any reference gives the same quotient.
//
// What bounds it, with more than 128 rows: a step of 64 keys takes about 2560 clocks, of which the
// exponentials of 256 rows are 1024 (16 a clock) and the products 1880 (1370 without the weights' lower
// halves). Without those a step took 2100: 131071 keys, 64 nodes, 32/8 heads of 128 150 us, 182 with them
// (164 without their products, 169 without their arithmetic; the upper halves' products begun ahead of the
// lower ones 196). 32 requests x 16384 keys with the same trees: 705 to 835 us alone, 845 in a row of calls
// under the power limit; one product of each kind at the dense rate would take 328. With few rows: the
// gather (64 x 8192 keys, 5 nodes, 12/4 heads of 64: 125 us, 4.3 TB/s). With little work: the start and end
// of a unit, some 10000 clocks (16 x 1900 keys 17.8 us).
#include <algorithm>

#include "tree.cuh"

namespace aiosb {
namespace {

constexpr int kTile = 128;      // rows of a tile: UMMA M, TMEM lanes
constexpr int kUnitRows = 256;  // two tiles
constexpr int kFewRows = 32;    // up to here on mma.sync
constexpr int kKeys = 128;      // keys of a chunk: a block of keys and one of values
constexpr int kStep = 64;       // keys of a softmax step, half a chunk
constexpr int kSoftWarps = 8;
constexpr int kLoadWarps = 4;
constexpr int kMmaWarp = kSoftWarps + kLoadWarps;
constexpr int kThreads = (kMmaWarp + 4) * 32;  // whole groups of four warps: two idle
// Registers of a thread, by role: 2 x 176 + 96 + 64 = 4 x 128, what the block is launched with.
constexpr int kSoftRegs = 176, kLoadRegs = 96, kMmaRegs = 64;
static_assert(2 * kSoftRegs + kLoadRegs + kMmaRegs <= 65536 / kThreads * 4, "more registers than the block has");
constexpr int kAtomBytes = kKeys * 128;  // 128 rows of 64 values, 128-byte swizzled
// Weights of the cut: a chunk of a unit of up to 128 rows, of a wider one, a unit's start and end, and the least range
// that is worth a CTA (above kWideCost, so that every range inside a unit has a chunk's start). Fitted, with one product
// of the weights: 41 ragged requests of up to 264 rows 105 us with chunks and units of equal weight, 100 with 2, 4, 5,
// 6, 87 with these; 16 x 1900 keys 20.7, 18.2 and 18.3, and 23 with a least range of 8.
constexpr int kChunkCost = 2, kWideCost = 4, kUnitCost = 12, kMinShare = 5;
constexpr int kPieceSlots = 8;
constexpr int kMaxGrid = 256;            // ranges: the join holds a weight for each of a unit's pieces and 32 rows
constexpr int kBadSlots = 8;
constexpr float kRescaleAt = 8.f;

template <int D>
struct Shape {
  static constexpr int kAtoms = (D + 63) / 64;
  static constexpr int kBlockBytes = kAtoms * kAtomBytes;  // a block of keys or values; also a tile of Q
  static constexpr int kStages = kAtoms == 1 ? 10 : 5;
  static constexpr int kBlocks = (2 + kStages) * kBlockBytes;  // two tiles of Q, the ring
};

// ---- the cut --------------------------------------------------------------------------------
struct Cut {
  int64_t total;  // weight of all units
  int ctas;       // ranges in use
  __device__ __forceinline__ int64_t begin(int c) const { return total * c / ctas; }
  // the range that holds position p
  __device__ __forceinline__ int owner(int64_t p) const { return (int)(((p + 1) * ctas - 1) / total); }
};

struct Piece {
  TreeRequest t;
  int h;
  int row0, rows;  // rows of the unit, in the request's (node, head) pairs
  int c0, c1, chunks;
  int64_t last_at;  // position of the unit's last chunk
  __device__ __forceinline__ bool whole() const { return c0 == 0 && c1 == chunks; }
  __device__ __forceinline__ bool pair() const { return rows > kTile; }
  __device__ __forceinline__ bool few() const { return rows <= kFewRows; }
};

// x / group for the rows of a tree (below 2^17): (x + 1/2) / group is 1/128 or more away from a whole number, and
// fp32 is off by 2^-23 of it.
__device__ __forceinline__ int node_of(int x, float inv_group) { return (int)(((float)x + 0.5f) * inv_group); }

// Of a request, for each KV head: `full` units of 256 rows, and one of the rest.
struct Units {
  int chunks, full, rest;  // rest: rows of the last unit, 0 if there is none
  int64_t wide, last;      // weights of a unit of 256 rows and of the last one
  __device__ __forceinline__ Units() {}
  __device__ __forceinline__ Units(const TreeAttnArgs& a, const TreeRequest& t) {
    const int rows = t.nodes * a.group;
    chunks = max(1, (t.keys + kKeys - 1) / kKeys);
    full = rows / kUnitRows;
    rest = rows - full * kUnitRows;
    wide = (int64_t)chunks * kWideCost + kUnitCost;
    last = rest > 0 ? (int64_t)chunks * (rest > kTile ? kWideCost : kChunkCost) + kUnitCost : 0;
  }
  __device__ __forceinline__ int64_t head() const { return full * wide + last; }
};

// The pieces of a range, in order. The gathering warps walk them, ahead of the others, and the first one of them hands
// them on (sh.pieces).
struct Pieces {
  int64_t pos, end, base;
  int r;
  TreeRequest t;
  Units u;
  int64_t span;

  __device__ __forceinline__ void take(const TreeAttnArgs& a, const TreeRequest& request) {
    t = request;
    u = Units(a, t);
    span = u.head() * a.hkv;
  }
  __device__ __forceinline__ bool next(const TreeAttnArgs& a, Piece& p) {
    while (pos < end) {
      while (pos >= base + span) {
        base += span;
        ++r;
        take(a, tree_request(a, r, false));
      }
      // (64-bit divisions only for what no memory holds)
      const int64_t off = pos - base, per_head = u.head();
      const bool small = span >> 32 == 0;
      const int h = (int)(small ? (uint32_t)off / (uint32_t)per_head : off / per_head);
      const int64_t in_head = off - h * per_head;
      const int block = min(u.full, (int)(small ? (uint32_t)in_head / (uint32_t)u.wide : in_head / u.wide));
      const bool is_last = block == u.full;
      const int cost = is_last && u.rest <= kTile ? kChunkCost : kWideCost;
      const int64_t at = base + h * per_head + block * u.wide, stop = min(end, at + (is_last ? u.last : u.wide));
      // chunk i starts at at + kUnitCost + i * cost, and belongs to the range with its start
      const int64_t from = pos - at - kUnitCost, to = stop - at - kUnitCost;
      p.c0 = from <= 0 ? 0 : (int)((from + cost - 1) / cost);
      p.c1 = to <= 0 ? 0 : (int)((to + cost - 1) / cost);
      pos = stop;
      if (p.c1 <= p.c0) continue;
      p.t = t;
      p.h = h;
      p.row0 = block * kUnitRows;
      p.rows = is_last ? u.rest : kUnitRows;
      p.chunks = u.chunks;
      p.last_at = at + kUnitCost + (int64_t)(u.chunks - 1) * cost;
      return true;
    }
    return false;
  }
};

// ---- work area ------------------------------------------------------------------------------
// Per range a descriptor of the cut unit that starts in it, then two slots of partial rows: slot 2c holds
// the piece that goes on from the range before, slot 2c + 1 the one that starts here.
struct __align__(16) Join {
  int start, row0, rows, h;  // rows 0: nothing to join
  int last;                  // the range with the unit's end
  int pad[3];
};
template <int D>
__host__ __device__ constexpr size_t slot_floats(int unit_rows) {
  return (size_t)unit_rows * (D + 2);
}
__device__ __forceinline__ float* slot_at(const TreeAttnArgs& a, int grid, size_t floats, int slot) {
  return reinterpret_cast<float*>(reinterpret_cast<Join*>(a.work) + grid) + floats * slot;
}

// ---- tcgen05 pieces of this kernel ----------------------------------------------------------
// D(tmem) (+)= A(tmem) * B(smem desc)
__device__ __forceinline__ void tc_mma_bf16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                               uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
          taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st2(uint32_t taddr, uint32_t x, uint32_t y) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x2.b32 [%0], {%1,%2};" ::"r"(taddr), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ void tmem_ld2(uint32_t taddr, float2& v) {
  uint32_t x, y;
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x2.b32 {%0,%1}, [%2];" : "=r"(x), "=r"(y) : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" : "+r"(x), "+r"(y)::"memory");
  v = make_float2(__uint_as_float(x), __uint_as_float(y));
}
__device__ __forceinline__ void mbar_arrive_count(uint64_t* bar, uint32_t count) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ float max3(float x, float y, float z) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(z));
  return r;
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// MN-major B operand (values as they lie: a key to a 128-byte row of 64 columns): 8 keys 1024 bytes apart
// along k, the next 64 columns an atom away.
__device__ __forceinline__ uint64_t umma_desc_mn(uint32_t smem_addr) {
  uint64_t d = 0;
  d |= (uint64_t)((smem_addr >> 4) & 0x3FFFu);
  d |= (uint64_t)(kAtomBytes >> 4) << 16;
  d |= (uint64_t)(1024u >> 4) << 32;
  d |= (uint64_t)1u << 46;
  d |= (uint64_t)2u << 61;
  return d;
}
constexpr uint32_t kBMajorMn = 1u << 16;  // instruction descriptor: B is MN-major

__device__ __forceinline__ void cp_async16_or_zero(uint32_t dst, const void* src, bool in) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0)
               : "memory");
}

// Bits of the 32 keys from kb on that a node with mask words `bits` sees.
__device__ __forceinline__ uint32_t seen32(const int32_t* bits, int words, int kb, int cached, int keys) {
  if (kb >= keys) return 0;
  const int o = kb - cached;
  uint32_t m;
  if (o <= -32) {
    m = 0xFFFFFFFFu;
  } else if (o < 0) {
    const uint32_t w = keys > cached ? (uint32_t)bits[0] : 0u;
    m = (w << -o) | ((1u << -o) - 1u);
  } else {
    const int i = o >> 5;
    const uint32_t w0 = i < words ? (uint32_t)bits[i] : 0u, w1 = i + 1 < words ? (uint32_t)bits[i + 1] : 0u;
    m = __funnelshift_r(w0, w1, o & 31);
  }
  const int left = keys - kb;
  return left >= 32 ? m : m & ((1u << left) - 1u);
}

// One step of a row: its 64 scores at t_s to weights over them, 32 columns of upper halves and 32 of lower ones; the
// row's reference and sum, and its output at t_o where the reference moves (behind `settled`: the products so far are
// in it). `seen`: bits of the keys, if some are hidden. False: a wait ran out.
template <int D, bool MASKED, typename Settled>
__device__ __forceinline__ bool soft_step(uint32_t t_s, uint32_t t_o, const uint32_t (&seen)[2], float scale, bool fresh,
                                          float& ref, float& sum, Settled settled) {
  bool ok = true;
  uint32_t v[2][32];
#pragma unroll
  for (int j = 0; j < 2; ++j) tmem_ld(t_s + j * 32, v[j]);
#pragma unroll
  for (int j = 0; j < 2; ++j) tmem_wait(v[j]);
  if (MASKED) {
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 32; ++e)
        if (!((seen[j] >> e) & 1)) v[j][e] = 0xFF800000u;  // -inf
  }
  float top[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t* const u = v[j / 2] + j % 2 * 16;
    top[j] = fmaxf(__uint_as_float(u[0]), __uint_as_float(u[15]));
#pragma unroll
    for (int e = 1; e < 15; e += 2) top[j] = max3(top[j], __uint_as_float(u[e]), __uint_as_float(u[e + 1]));
  }
  const float most = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * scale;
  const bool grows = most > ref + kRescaleAt;
  if (__any_sync(0xffffffffu, grows)) {
    const float corr = grows ? exp2_fast(ref - most) : 1.f;
    if (!fresh) {
      ok = settled();
      if (ok) {
#pragma unroll 1
        for (int j = 0; j < D / 16; ++j) {
          uint32_t o[16];
          tmem_ld(t_o + j * 16, o);
          tmem_wait(o);
#pragma unroll
          for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * corr);
          tmem_st16(t_o + j * 16, o);
        }
      }
    }
    sum *= corr;
    if (grows) ref = most;
  }
  const float minus = ref == -INFINITY ? 0.f : -ref;  // nothing seen yet: any finite reference will do
  const float2 m2 = make_float2(minus, minus), s2 = make_float2(scale, scale);
  float2 part[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    uint32_t w[2][16];
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      float2 x = __ffma2_rn(make_float2(__uint_as_float(v[j][2 * e]), __uint_as_float(v[j][2 * e + 1])), s2, m2);
      x = make_float2(exp2_fast(x.x), exp2_fast(x.y));
      part[e & 1] = __fadd2_rn(part[e & 1], x);
      split_bf16x2(x, w[0][e], w[1][e]);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) tmem_st16(t_s + i * (kStep / 2) + j * 16, w[i]);  // over columns that have been read
  }
  sum += (part[0].x + part[0].y) + (part[1].x + part[1].y);
  tmem_wait_st();
  return ok;
}

struct Shared {
  uint64_t full[10], empty[10];
  uint64_t s_full[2][2], p_full[2][2], pv_done[2], q_full, piece_done, met, drained, piece_ready[kPieceSlots], piece_read[kPieceSlots];
  uint32_t tmem_slot;
  volatile int abort_flag;
  int r0;
  int64_t pos, end, base;  // this CTA's range, and where the first request of it starts
  TreeRequest first;
  Piece pieces[kPieceSlots];  // rows 0: no more
  Cut cut;
  float2 few_state[kSoftWarps][16];  // (reference, sum) of the warps' rows, in a piece of few rows
  uint32_t bad[kBadSlots][AIOSB_TREE_MAX_NODES / 32];  // per piece: tree keys whose V holds an infinity or a NaN
};

template <int D>
constexpr int kSmem = Shape<D>::kBlocks + (int)sizeof(Shared);
static_assert(kSmem<128> <= 232448 && kSmem<96> <= 232448 && kSmem<64> <= 232448, "shared memory of a CTA");

template <int D>
__global__ void __launch_bounds__(kThreads, 1) attn_tree_split_kernel(const TreeAttnArgs a, int unit_rows) {
  using S = Shape<D>;
  // No static shared memory: the blocks start where dynamic shared memory does, on 1024 bytes.
  extern __shared__ __align__(1024) uint8_t smem[];
  Shared& sh = *reinterpret_cast<Shared*>(smem + S::kBlocks);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t q_smem = smem_u32(smem), ring = q_smem + 2 * S::kBlockBytes;

  if (threadIdx.x == 0) {
    for (int i = 0; i < S::kStages; ++i) {
      mbar_init(&sh.full[i], kLoadWarps * 32);
      mbar_init(&sh.empty[i], kSoftWarps);
    }
    for (int i = 0; i < 2; ++i) {
      for (int b = 0; b < 2; ++b) {
        mbar_init(&sh.s_full[i][b], 1);
        mbar_init(&sh.p_full[i][b], 4);
      }
      mbar_init(&sh.pv_done[i], 1);
    }
    mbar_init(&sh.q_full, kSoftWarps);
    mbar_init(&sh.piece_done, 2);
    mbar_init(&sh.met, kSoftWarps);
    mbar_init(&sh.drained, 2);
    for (int i = 0; i < kPieceSlots; ++i) {
      mbar_init(&sh.piece_ready[i], 1);
      mbar_init(&sh.piece_read[i], kSoftWarps + 2);
    }
    sh.abort_flag = 0;
    fence_mbar_init();
  }
  for (int i = threadIdx.x; i < kBadSlots * (AIOSB_TREE_MAX_NODES / 32); i += kThreads)
    (&sh.bad[0][0])[i] = 0;
  if (warp == kMmaWarp) {
    tmem_alloc(&sh.tmem_slot, 512);
    tmem_relinquish();
  }
  pdl_wait();
  if (warp == 0) {  // the weight of all units, and where this CTA's range starts
    TreeRequest t;  // of the last request that this lane looked at
    auto weight_of = [&](int r, bool tell) {
      if (r >= a.requests) return (int64_t)0;
      t = tree_request(a, r, tell);
      return Units(a, t).head() * a.hkv;
    };
    const int64_t first = weight_of(lane, blockIdx.x == 0);
    int64_t total = first;
    for (int r = 32 + lane; r - lane < a.requests; r += 32) total += weight_of(r, blockIdx.x == 0);
#pragma unroll 1
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    Cut cut;
    cut.total = total;
    cut.ctas = (int)max((int64_t)1, min((int64_t)gridDim.x, total / kMinShare));
    const bool used = (int)blockIdx.x < cut.ctas && total > 0;
    const int64_t pos = used ? cut.begin(blockIdx.x) : 0, end = used ? cut.begin(blockIdx.x + 1) : 0;
    int64_t base = 0;
    int found = 0;
    for (int r0 = 0; used; r0 += 32) {
      const int64_t w = a.requests <= 32 ? first : weight_of(r0 + lane, false);
      int64_t upto = w;
#pragma unroll 1
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, base + upto > pos);
      if (hit) {
        const int l = __ffs(hit) - 1;
        found = r0 + l;
        base += __shfl_sync(0xffffffffu, upto - w, l);
        if (lane == l) sh.first = t;
        break;
      }
      base += __shfl_sync(0xffffffffu, upto, 31);
    }
    if (lane == 0) {
      sh.cut = cut;
      sh.r0 = found;
      sh.pos = pos;
      sh.end = end;
      sh.base = base;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_launch_dependents();
  const uint32_t tmem = sh.tmem_slot;
  const int me = blockIdx.x;
  const float inv_group = 1.f / (float)a.group;

  Piece p = {};
  uint32_t piece_number = 0;
  auto next_piece = [&](bool& ok) {
    const uint32_t slot = piece_number % kPieceSlots;
    ok = __all_sync(0xffffffffu, mbar_wait(&sh.piece_ready[slot], (piece_number / kPieceSlots) & 1));
    if (!ok) return false;
    ++piece_number;
    p = sh.pieces[slot];
    __syncwarp();
    if (lane == 0) mbar_arrive(&sh.piece_read[slot]);
    return p.rows > 0;
  };

  if (warp >= kSoftWarps && warp < kMmaWarp) {
    // ---- gather
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kLoadRegs));
    const int lw = warp - kSoftWarps;
    const int64_t slot_bytes = (int64_t)a.hkv * D * 2;
    int stage = 0;
    uint32_t phase = 1;
    bool ok = true;
    int turn = 0;
    // Slots of this lane's key in eight chunks: four from `window` on, and the four behind them. They are asked
    // for four to eight chunks ahead: a page table's line comes from DRAM, which takes as long as a chunk.
    int window = 0, here[4], ahead[4];
    auto ask = [&](int chunk, int (&out)[4]) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int key = (chunk + j) * kKeys + lw * 32 + lane;
        out[j] = key < min(p.t.keys, p.c1 * kKeys) ? a.page_table[p.t.table + key] : 0;
      }
    };
    auto load = [&](bool values, int chunk) {
      if (values && chunk >= window + 4) {
        window += 4;
#pragma unroll
        for (int j = 0; j < 4; ++j) here[j] = ahead[j];
        ask(window + 4, ahead);
      }
      const int at = chunk - window;
      int slot = at < 4 ? here[0] : ahead[0];
#pragma unroll
      for (int j = 1; j < 4; ++j)
        if ((at & 3) == j) slot = at < 4 ? here[j] : ahead[j];
      ok = __all_sync(0xffffffffu, mbar_wait(&sh.empty[stage], phase));
      if (!ok) return;
      const int k0 = chunk * kKeys + lw * 32;
      if (slot < 0 || slot >= a.num_slots) {
        if (!values) report(a.status, AIOSB_DEV_SLOT_RANGE);
        slot = 0;
      }
      const char* const src =
          reinterpret_cast<const char*>(values ? a.v_cache : a.k_cache) + (int64_t)p.h * D * 2;
      const uint32_t dst = ring + stage * S::kBlockBytes + lw * 32 * 128;
      constexpr int kCols = D / 8;  // 16-byte pieces of a key
      int slots[kCols];  // every exchange before the first copy: one after another they take as long as the copies
#pragma unroll
      for (int i = 0; i < kCols; ++i) slots[i] = __shfl_sync(0xffffffffu, slot, (i * 32 + lane) / kCols);
#pragma unroll
      for (int i = 0; i < kCols; ++i) {
        const int at = i * 32 + lane, row = at / kCols, c = at % kCols;
        cp_async16_or_zero(dst + (c >> 3) * kAtomBytes + row * 128 + (((c & 7) ^ (row & 7)) << 4),
                           src + slots[i] * slot_bytes + c * 16, k0 + row < p.t.keys);
      }
      if (values && k0 + 32 > p.t.cached && k0 < p.t.keys) {
        // a key that a node does not see gets weight 0, and 0 * inf is NaN: infinities and NaN of the tree's
        // keys leave V here, and reach the nodes that see them at the end
        cp_async_wait_all();
        __syncwarp();
        const int key = k0 + lane;
        bool bad = false;
        if (key >= p.t.cached && key < p.t.keys) {
#pragma unroll 4
          for (int c = 0; c < kCols; ++c) {
            const uint32_t at = dst + (c >> 3) * kAtomBytes + lane * 128 + (((c & 7) ^ (lane & 7)) << 4);
            uint4 v;
            asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];"
                         : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                         : "r"(at)
                         : "memory");
            if (finite_bf16x2(v.x) && finite_bf16x2(v.y) && finite_bf16x2(v.z) && finite_bf16x2(v.w)) continue;
            bad = true;
            asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(drop_nonfinite_bf16x2(v.x)),
                         "r"(drop_nonfinite_bf16x2(v.y)), "r"(drop_nonfinite_bf16x2(v.z)),
                         "r"(drop_nonfinite_bf16x2(v.w))
                         : "memory");
          }
          const int j = key - p.t.cached;
          if (bad) atomicOr(&sh.bad[turn][j >> 5], 1u << (j & 31));
        }
        fence_proxy_async_shared();
        mbar_arrive(&sh.full[stage]);
      } else {
        // this thread arrives when its copies so far have landed
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&sh.full[stage]))
                     : "memory");
      }
      if (++stage == S::kStages) {
        stage = 0;
        phase ^= 1;
      }
    };
    Pieces it;
    it.pos = sh.pos;
    it.end = sh.end;
    it.base = sh.base;
    it.r = sh.r0;
    if (it.pos < it.end) it.take(a, sh.first);
    auto hand_on = [&] {
      if (lw != 0) return;
      const uint32_t slot = piece_number % kPieceSlots;
      // its last piece has been read by all
      ok = __all_sync(0xffffffffu, mbar_wait(&sh.piece_read[slot], ((piece_number / kPieceSlots) & 1) ^ 1));
      if (!ok) return;
      ++piece_number;
      if (lane == 0) sh.pieces[slot] = p;
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.piece_ready[slot]);
    };
    // block order of a piece: the order in which the MMAs want them
    while (ok && it.next(a, p)) {
      hand_on();
      if (!ok) break;
      window = p.c0;
      ask(window, here);
      ask(window + 4, ahead);
      if (p.pair() || p.few()) {
        for (int c = p.c0; c < p.c1 && ok; ++c) {
          load(false, c);
          if (ok) load(true, c);
        }
      } else {
        load(false, p.c0);
        if (ok && p.c0 + 1 < p.c1) load(false, p.c0 + 1);
        for (int c = p.c0; c < p.c1 && ok; ++c) {
          load(true, c);
          if (ok && c + 2 < p.c1) load(false, c + 2);
        }
      }
      turn = (turn + 1) % kBadSlots;
    }
    if (ok) {
      p.rows = 0;
      hand_on();
    }
    cp_async_wait_all();
    if (!ok) {
      report(a.status, AIOSB_DEV_WAIT_TIMEOUT);
      sh.abort_flag = 1;
    }
  } else if (warp >= kMmaWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kMmaRegs));
    if (warp < kMmaWarp + 2) {
    // ---- MMAs of stream s: O += P V of its last step, then S of the step after next, so that scores are there when
    // the softmax comes to them. A warp for each stream: a wait that is over and the issue behind it take some
    // hundred clocks of a warp, in which the other's MMAs run.
    constexpr uint32_t idesc_s = umma_idesc_bf16(kTile, kStep), idesc_o = umma_idesc_bf16(kTile, D) | kBMajorMn;
    const int s = warp - kMmaWarp;
    uint32_t base = 0, q_phase = 0, steps = 0;  // of the stream, in all pieces so far
    bool ok = true;
    while (ok && next_piece(ok)) {
      const int n = p.c1 - p.c0;
      if (p.few()) {
        base += 2 * n;
        continue;
      }
      const bool pair = p.pair();
      // blocks of chunk i's keys and values, as the gathering warps order them
      auto k_block = [&](int i) { return base + (pair ? 2 * i : i < 2 ? i : 2 * i - 1); };
      auto v_block = [&](int i) { return base + (pair ? 2 * i + 1 : i == n - 1 ? 2 * n - 1 : 2 * i + 2); };
      auto wait_block = [&](uint32_t b) { return mbar_wait(&sh.full[b % S::kStages], (b / S::kStages) & 1); };
      // a block is free when both streams are through with it, or the only one that uses it
      auto release = [&](uint32_t stage) {
        // (eight arrivals: in a piece of few rows the softmax warps read the blocks)
        tc_commit(&sh.empty[stage]);
        mbar_arrive_count(&sh.empty[stage], pair ? kSoftWarps / 2 - 1 : kSoftWarps - 1);
      };
      // step h is half h & 1 of this chunk of the piece
      auto chunk_of = [&](int h) { return pair ? h >> 1 : 2 * (h >> 1) + s; };
      const uint64_t q_desc = umma_desc_sw128(q_smem + (pair ? s : 0) * S::kBlockBytes);
      auto score = [&](int h) {  // S of step h; the elected lane
        const uint32_t stage = k_block(chunk_of(h)) % S::kStages, buffer = (steps + h) & 1;
        const uint64_t kd = umma_desc_sw128(ring + stage * S::kBlockBytes + (h & 1) * (kStep * 128));
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint32_t off = ((k >> 2) * kAtomBytes + (k & 3) * 32) >> 4;
          tc_mma_bf16(tmem + s * 128 + buffer * kStep, q_desc + off, kd + off, idesc_s, k > 0);
        }
        tc_commit(&sh.s_full[s][buffer]);
        if (h & 1) release(stage);
      };
      ok = __all_sync(0xffffffffu, mbar_wait(&sh.q_full, q_phase));
      q_phase ^= 1;
      if (!ok) break;
      tc_fence_after();  // the softmax warps have read the last piece's scores' place
      if (chunk_of(0) < n) {
        ok = __all_sync(0xffffffffu, wait_block(k_block(chunk_of(0))));
        if (ok && elect_one()) {
          fence_proxy_async_shared();  // the copies went through the generic proxy, the MMAs read through the other
          score(0);
          score(1);
        }
        __syncwarp();
      }
      int h = 0;
      for (; ok && chunk_of(h) < n; ++h) {
        const int next = chunk_of(h + 2);
        const uint32_t buffer = (steps + h) & 1, vb = v_block(chunk_of(h));
        // the blocks first: they are there before the weights, as a rule
        ok = wait_block(vb) && (next >= n || wait_block(k_block(next))) &&
             mbar_wait(&sh.p_full[s][buffer], ((steps + h) >> 1) & 1);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          fence_proxy_async_shared();
          const uint32_t stage = vb % S::kStages;
          const uint32_t v = ring + stage * S::kBlockBytes + (h & 1) * (kStep * 128);
#pragma unroll
          for (int k = 0; k < kStep / 16; ++k)
#pragma unroll
            for (int i = 0; i < 2; ++i)  // the weights' upper and lower halves
              tc_mma_bf16_ts(tmem + 256 + s * 128, tmem + s * 128 + buffer * kStep + i * (kStep / 2) + k * 8,
                             umma_desc_mn(v + k * 2048), idesc_o, h > 0 || k > 0 || i > 0);
          tc_commit(&sh.pv_done[s]);
          if (h & 1) release(stage);
          if (next < n) score(h + 2);
        }
        __syncwarp();
      }
      if (!ok) break;
      if (elect_one()) tc_commit(&sh.piece_done);
      __syncwarp();
      base += 2 * n;
      steps += h;
    }
    if (!ok) {
      report(a.status, AIOSB_DEV_WAIT_TIMEOUT);
      sh.abort_flag = 1;
    }
    }
  } else {
    // ---- softmax of stream s; a thread owns row `row` of the stream's tile
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftRegs));
    const int s = warp >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t t_lane = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t t_o = t_lane + 256 + s * 128;
    uint32_t step = 0, base = 0, done_phase = 0, met_phase = 0;  // steps of this stream and blocks, in all pieces so far
    int turn = 0, partial_of = -1;
    bool ok = true;
    Join join = {};
    // all softmax warps
    auto meet = [&] {
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.met);
      const bool all = __all_sync(0xffffffffu, mbar_wait(&sh.met, met_phase));
      met_phase ^= 1;
      return all;
    };
    auto start_join = [&] {
      partial_of = 1;
      join.start = p.t.start;
      join.row0 = p.row0;
      join.rows = p.rows;
      join.h = p.h;
      if (threadIdx.x == 0) join.last = sh.cut.owner(p.last_at);
    };
    // Up to 32 rows: 16 to a warp on mma.sync, each warp with its share of every chunk's keys and its own maximum,
    // sum and output, joined at the end. The tensor pipe is idle here, but a TMEM round trip per step (scores out,
    // weights back) took longer than the chunk's bytes: 64 x 8192 keys, 15 rows 148 -> 134 us.
    auto few_rows = [&](auto load_q) {
      const int tiles = p.rows > 16 ? 2 : 1, tile = warp & (tiles - 1), part = warp / tiles;
      if (s == 0) load_q(0, 16 * tiles);
      if (!meet()) return false;
      const int row[2] = {tile * 16 + lane / 4, tile * 16 + lane / 4 + 8};
      const int32_t* bits[2];
#pragma unroll
      for (int i = 0; i < 2; ++i)
        bits[i] = a.mask + (int64_t)(p.t.start + node_of(p.row0 + min(row[i], p.rows - 1), inv_group)) * a.words;
      float o[D / 8][4];
#pragma unroll
      for (int n = 0; n < D / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][e] = 0.f;
      float ref[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};
      const bool works = tile * 16 < p.rows;
      // 16-byte piece `col` of row `r` of a block or of Q
      auto piece_at = [](uint32_t block, int r, int col) {
        return block + (col >> 3) * kAtomBytes + r * 128 + (((col & 7) ^ (r & 7)) << 4);
      };
      for (int c = p.c0; c < p.c1; ++c) {
        const uint32_t kb = base + 2 * (c - p.c0), vb = kb + 1;
        const uint32_t ks = kb % S::kStages, vs = vb % S::kStages;
        const uint32_t k_mem = ring + ks * S::kBlockBytes, v_mem = ring + vs * S::kBlockBytes;
        if (!__all_sync(0xffffffffu, mbar_wait(&sh.full[ks], (kb / S::kStages) & 1))) return false;
        uint32_t w[2][2][4];  // weights as A operands, 16 keys each: upper and lower halves
        if (works) {
          float x[2][2][4];  // scores: 16 keys, 8 keys, the accumulator's values
#pragma unroll
          for (int g = 0; g < 2; ++g) {
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
              for (int e = 0; e < 4; ++e) x[g][n][e] = g < tiles ? 0.f : -INFINITY;
            if (g >= tiles) continue;
            const int key = (part * tiles + g) * 16;
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {
              uint32_t q[4], b[4];
              ldmatrix4(q, piece_at(q_smem, tile * 16 + (lane & 15), 2 * k + (lane >> 4)));
              ldmatrix4(b, piece_at(k_mem, key + (lane & 7) + (lane & 16 ? 8 : 0), 2 * k + (lane & 8 ? 1 : 0)));
              mma_16816(x[g][0], q, b[0], b[1]);
              mma_16816(x[g][1], q, b[2], b[3]);
            }
            if ((c + 1) * kKeys > p.t.cached) {
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                const uint32_t seen =
                    seen32(bits[i], a.words, c * kKeys + key, p.t.cached, p.t.keys) >> (2 * (lane & 3));
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  if (!((seen >> ((e >> 1) * 8 + (e & 1))) & 1)) x[g][e >> 1][2 * i + (e & 1)] = -INFINITY;
              }
            }
          }
          float most[2];
          bool grows[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            most[i] = -INFINITY;
#pragma unroll
            for (int g = 0; g < 2; ++g)
#pragma unroll
              for (int n = 0; n < 2; ++n) most[i] = max3(most[i], x[g][n][2 * i], x[g][n][2 * i + 1]);
            most[i] = fmaxf(most[i], __shfl_xor_sync(0xffffffffu, most[i], 1));
            most[i] = fmaxf(most[i], __shfl_xor_sync(0xffffffffu, most[i], 2)) * a.scale_log2;
            grows[i] = most[i] > ref[i] + kRescaleAt;
          }
          if (__any_sync(0xffffffffu, grows[0] || grows[1])) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const float corr = grows[i] ? exp2_fast(ref[i] - most[i]) : 1.f;
              if (grows[i]) ref[i] = most[i];
              sum[i] *= corr;
#pragma unroll
              for (int n = 0; n < D / 8; ++n) {
                o[n][2 * i] *= corr;
                o[n][2 * i + 1] *= corr;
              }
            }
          }
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            if (g >= tiles) continue;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const float minus = ref[i] == -INFINITY ? 0.f : -ref[i];
#pragma unroll
              for (int n = 0; n < 2; ++n) {
                const float y = exp2_fast(fmaf(x[g][n][2 * i], a.scale_log2, minus)),
                            z = exp2_fast(fmaf(x[g][n][2 * i + 1], a.scale_log2, minus));
                sum[i] += y + z;
                split_bf16x2(make_float2(y, z), w[g][0][2 * n + i], w[g][1][2 * n + i]);
              }
            }
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.empty[ks]);
        if (!__all_sync(0xffffffffu, mbar_wait(&sh.full[vs], (vb / S::kStages) & 1))) return false;
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          if (g >= tiles || !works) continue;
          const int key = (part * tiles + g) * 16;
#pragma unroll
          for (int n = 0; n < D / 16; ++n) {
            uint32_t b[4];
            ldmatrix4_trans(b, piece_at(v_mem, key + (lane & 15), 2 * n + (lane >> 4)));
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              mma_16816(o[2 * n], w[g][i], b[0], b[1]);
              mma_16816(o[2 * n + 1], w[g][i], b[2], b[3]);
            }
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.empty[vs]);
      }
      // ---- the warps' outputs, in Q's place: a row's columns are turned by 8 a row against bank conflicts
      if (!meet()) return false;
      float* const all = reinterpret_cast<float*>(smem);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 1);
        sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 2);
        const int r = lane / 4 + 8 * i;
        if ((lane & 3) == 0) sh.few_state[warp][r] = make_float2(ref[i], sum[i]);
#pragma unroll
        for (int n = 0; n < D / 8; ++n)
          *reinterpret_cast<float2*>(all + (warp * 16 + r) * D + (n * 8 + r * 8) % D + (lane & 3) * 2) =
              make_float2(o[n][2 * i], o[n][2 * i + 1]);
      }
      if (!meet()) return false;
      const bool whole = p.whole();
      float* const slot = whole ? nullptr
                                : slot_at(a, gridDim.x, slot_floats<D>(unit_rows), p.c0 == 0 ? 2 * me + 1 : 2 * me);
      if (!whole && p.c0 == 0) start_join();
      uint32_t any_bad = 0;
      if (p.c1 * kKeys > p.t.cached)
        for (int i = 0; i < a.words; ++i) any_bad |= sh.bad[turn][i];
      for (int i = threadIdx.x; i < p.rows * (D / 4); i += kSoftWarps * 32) {
        const int my = i / (D / 4), c4 = i % (D / 4), my_tile = my / 16, r = my & 15;
        float m = -INFINITY, l = 0.f;
        for (int q = 0; q < kSoftWarps / tiles; ++q) m = fmaxf(m, sh.few_state[q * tiles + my_tile][r].x);
        const float from = m == -INFINITY ? 0.f : m;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int q = 0; q < kSoftWarps / tiles; ++q) {
          const int from_warp = q * tiles + my_tile;
          const float2 st = sh.few_state[from_warp][r];
          const float f = exp2_fast(st.x - from);
          const float4 y = *reinterpret_cast<const float4*>(all + (from_warp * 16 + r) * D + (c4 * 4 + r * 8) % D);
          l = fmaf(st.y, f, l);
          v.x = fmaf(y.x, f, v.x);
          v.y = fmaf(y.y, f, v.y);
          v.z = fmaf(y.z, f, v.z);
          v.w = fmaf(y.w, f, v.w);
        }
        const int g = p.row0 + my, node = node_of(g, inv_group);
        if (any_bad) {
          const int32_t* const own = a.mask + (int64_t)(p.t.start + node) * a.words;
#pragma unroll 1
          for (int j = 0; j < a.words; ++j) {
            for (uint32_t hit = sh.bad[turn][j] & (uint32_t)own[j]; hit; hit &= hit - 1) {
              const int key = p.t.cached + j * 32 + __ffs(hit) - 1;
              const __nv_bfloat16* x = a.v_cache + (tree_slot(a, a.page_table[p.t.table + key]) * a.hkv + p.h) * D + c4 * 4;
              float* const e = &v.x;
              for (int z = 0; z < 4; ++z) {
                const float y = bf16_to_f(x[z]);
                if (!(fabsf(y) < INFINITY)) e[z] += y;
              }
            }
          }
        }
        if (whole) {
          const float inv = m == -INFINITY && l == 0.f ? 0.f : 1.f / l;
          __nv_bfloat16* const dst = a.out + (int64_t)(p.t.start + node) * a.out_stride +
                                     (int64_t)(p.h * a.group + g - node * a.group) * D;
          reinterpret_cast<uint2*>(dst)[c4] =
              make_uint2(pack_bf16x2(v.x * inv, v.y * inv), pack_bf16x2(v.z * inv, v.w * inv));
        } else {
          if (c4 == 0) reinterpret_cast<float2*>(slot)[my] = make_float2(m, l);
          reinterpret_cast<float4*>(slot + 2 * unit_rows)[(size_t)c4 * unit_rows + my] = v;
        }
      }
      // before Q of the next piece
      if (!meet()) return false;
      if (warp == 0) sh.bad[(turn + kBadSlots - 1) % kBadSlots][lane] = 0;
      return true;
    };
    while (ok && next_piece(ok)) {
      const bool pair = p.pair();
      // `tile` of Q's `count` rows, by 128 threads
      auto load_q = [&](int tile, int count) {
        const int wt = threadIdx.x & 127;
        constexpr int kCols = D / 8;
        const uint32_t dst = q_smem + tile * S::kBlockBytes;
#pragma unroll 4
        for (int i = 0; i * 128 < count * kCols; ++i) {
          const int at = i * 128 + wt, rr = at / kCols, c = at % kCols;
          const int g = min(p.row0 + tile * kTile + rr, p.row0 + p.rows - 1), node = node_of(g, inv_group);
          cp_async16_or_zero(dst + (c >> 3) * kAtomBytes + rr * 128 + (((c & 7) ^ (rr & 7)) << 4),
                             a.q + (int64_t)(p.t.start + node) * a.q_stride +
                                 (int64_t)(p.h * a.group + g - node * a.group) * D + c * 8,
                             tile * kTile + rr < p.rows);
        }
        cp_async_wait_all();
      };
      if (p.few()) {
        ok = few_rows(load_q);
        base += 2 * (p.c1 - p.c0);
        turn = (turn + 1) % kBadSlots;
        continue;
      }
      // this group's tile (the second group's is not used by a narrow unit)
      if (s == 0 || pair) {
        load_q(s, kTile);
        fence_proxy_async_shared();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.q_full);

      const int my_row = (pair ? s * kTile : 0) + row;  // of the unit
      const int rows_here = p.rows - (pair ? s * kTile : 0);
      const bool warp_works = (warp & 3) * 32 < rows_here;
      const int pair_row = p.row0 + min(my_row, p.rows - 1);
      const int node = p.t.start + node_of(pair_row, inv_group);
      const int32_t* const bits = a.mask + (int64_t)node * a.words;
      float ref = -INFINITY, sum = 0.f;
      bool fresh = true;  // no output of this piece yet
      for (int c = p.c0 + (pair ? 0 : s); c < p.c1 && ok; c += pair ? 1 : 2) {
#pragma unroll 1
        for (int half = 0; half < 2; ++half, ++step) {
          const uint32_t buffer = step & 1, t_s = t_lane + s * 128 + buffer * kStep;
          ok = __all_sync(0xffffffffu, mbar_wait(&sh.s_full[s][buffer], (step >> 1) & 1));
          if (!ok) break;
          tc_fence_after();
          if (warp_works) {
            const int k0 = c * kKeys + half * kStep;
            auto settled = [&] {  // the products of the steps before this one are in the output
              const bool there = __all_sync(0xffffffffu, mbar_wait(&sh.pv_done[s], (step - 1) & 1));
              tc_fence_after();
              return there;
            };
            if (k0 + kStep > p.t.cached) {
              const uint32_t seen[2] = {seen32(bits, a.words, k0, p.t.cached, p.t.keys),
                                        seen32(bits, a.words, k0 + 32, p.t.cached, p.t.keys)};
              ok = soft_step<D, true>(t_s, t_o, seen, a.scale_log2, fresh, ref, sum, settled);
            } else {
              const uint32_t all[2] = {};
              ok = soft_step<D, false>(t_s, t_o, all, a.scale_log2, fresh, ref, sum, settled);
            }
            if (!ok) break;  // the output is still at the old reference: nothing may follow it
          }
          fresh = false;
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh.p_full[s][buffer]);
        }
      }
      if (!ok) break;
      ok = __all_sync(0xffffffffu, mbar_wait(&sh.piece_done, done_phase));
      done_phase ^= 1;
      if (!ok) break;
      tc_fence_after();

      // ---- a narrow unit's streams are joined here: each group writes half of the columns
      float weight[2] = {1.f, 0.f};
      float m_all = ref, l_all = sum;
      const bool both = !pair && p.c1 - p.c0 > 1;  // streams of a narrow unit that have seen keys
      if (!pair) {
        // through TMEM, where S was: the two warps with this row reach the same lane
        tmem_st2(t_lane + s * 128, __float_as_uint(ref), __float_as_uint(sum));
        tmem_wait_st();
        tc_fence_before();
        ok = meet();
        if (!ok) break;
        tc_fence_after();
        float2 x, y;
        tmem_ld2(t_lane, x);
        tmem_ld2(t_lane + 128, y);
        m_all = fmaxf(x.x, both ? y.x : -INFINITY);
        const float m = m_all == -INFINITY ? 0.f : m_all;
        weight[0] = exp2_fast(x.x - m);
        weight[1] = both ? exp2_fast(y.x - m) : 0.f;
        l_all = x.y * weight[0] + (both ? y.y * weight[1] : 0.f);
      }
      const bool whole = p.whole();
      const bool none = m_all == -INFINITY && l_all == 0.f;  // the row sees none of these keys
      const float inv = !whole ? 1.f : none ? 0.f : 1.f / l_all;
      const int slot = p.c0 == 0 ? 2 * me + 1 : 2 * me;
      float* const part = whole ? nullptr : slot_at(a, gridDim.x, slot_floats<D>(unit_rows), slot);
      const bool row_works = my_row < p.rows;
      if (!whole && row_works && (pair || s == 0))
        reinterpret_cast<float2*>(part)[my_row] = make_float2(m_all, l_all);
      if (!whole && p.c0 == 0) start_join();
      uint32_t any_bad = 0;
      if (p.c1 * kKeys > p.t.cached)
        for (int w = 0; w < a.words; ++w) any_bad |= sh.bad[turn][w];
      if (warp_works) {
        __nv_bfloat16* const dst = a.out + (int64_t)node * a.out_stride +
                                   (int64_t)(p.h * a.group + pair_row - (node - p.t.start) * a.group) * D;
        const int j0 = pair ? 0 : s * (D / 32), j1 = pair ? D / 16 : (s + 1) * (D / 32);  // of 16 columns each
#pragma unroll 1
        for (int j = j0; j < j1; ++j) {
          uint32_t v[16];
          float o[16];
          tmem_ld(t_lane + 256 + (pair ? s * 128 : 0) + j * 16, v);
          tmem_wait(v);
#pragma unroll
          for (int e = 0; e < 16; ++e) o[e] = __uint_as_float(v[e]) * weight[0];
          if (both) {
            tmem_ld(t_lane + 384 + j * 16, v);
            tmem_wait(v);
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = fmaf(__uint_as_float(v[e]), weight[1], o[e]);
          }
          if (!row_works) continue;
          if (any_bad) {
#pragma unroll 1
            for (int w = 0; w < a.words; ++w) {
              for (uint32_t hit = sh.bad[turn][w] & (uint32_t)bits[w]; hit; hit &= hit - 1) {
                const int key = p.t.cached + w * 32 + __ffs(hit) - 1;
                const __nv_bfloat16* x =
                    a.v_cache + (tree_slot(a, a.page_table[p.t.table + key]) * a.hkv + p.h) * D + j * 16;
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                  const float y = bf16_to_f(x[e]);
                  if (!(fabsf(y) < INFINITY)) o[e] += y;
                }
              }
            }
          }
          if (whole) {
            uint4 u[2];
            uint32_t* const w = reinterpret_cast<uint32_t*>(u);
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = pack_bf16x2(o[2 * e] * inv, o[2 * e + 1] * inv);
            reinterpret_cast<uint4*>(dst + j * 16)[0] = u[0];
            reinterpret_cast<uint4*>(dst + j * 16)[1] = u[1];
          } else {  // a column of float4 for each row, so that neighbouring rows lie side by side
            float4* const f = reinterpret_cast<float4*>(part + 2 * unit_rows) + my_row;
#pragma unroll
            for (int e = 0; e < 4; ++e)
              f[(size_t)(j * 4 + e) * unit_rows] = make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
          }
        }
      }
      // every warp has started on this piece, so all are through with the one before it
      if (warp == 0) sh.bad[(turn + kBadSlots - 1) % kBadSlots][lane] = 0;
      turn = (turn + 1) % kBadSlots;
      base += 2 * (p.c1 - p.c0);
      tc_fence_before();
    }
    if (!ok) {
      report(a.status, AIOSB_DEV_WAIT_TIMEOUT);
      sh.abort_flag = 1;
    }
    if (threadIdx.x == 0) {
      if (partial_of < 0) join.rows = 0;
      reinterpret_cast<Join*>(a.work)[me] = join;
    }
  }

  tc_fence_before();
  __syncthreads();
  if (sh.abort_flag && warp >= kMmaWarp && warp < kMmaWarp + 2) {  // MMAs may still run: their end is waited for
    if (elect_one()) tc_commit(&sh.drained);
    __syncwarp();
    mbar_wait(&sh.drained, 0);
  }
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Joins the pieces of the unit that starts in range blockIdx.x and goes on behind it. A CTA takes 32 rows and D / 4
// columns: first every piece's maxima and sums, then the pieces' outputs, four loads in flight to a thread. It adds
// 4.5 us to 16 x 1900 keys (12.6 without it), two of them for a grid that finds little to do, and 11 to 41 ragged
// requests, whose 33 MB of pieces are read again. More columns to a CTA, and the first two pieces loaded at once with
// the record, took as long or longer.
constexpr int kJoinRows = 32, kJoinParts = 4;

template <int D>
__global__ void __launch_bounds__(256) attn_tree_join_kernel(const TreeAttnArgs a, int grid, int unit_rows) {
  extern __shared__ float weight[];  // [pieces, rows]
  pdl_enter();
  const Join j = reinterpret_cast<const Join*>(a.work)[blockIdx.x];
  const int r = threadIdx.x & 31, sub = threadIdx.x >> 5, row = blockIdx.y * kJoinRows + r;
  if ((int)blockIdx.y * kJoinRows >= j.rows) return;
  const size_t floats = slot_floats<D>(unit_rows);
  const int first = blockIdx.x, pieces = j.last - first + 1;
  auto slot = [&](int i) { return slot_at(a, grid, floats, i == 0 ? 2 * first + 1 : 2 * (first + i)); };
  const bool in = row < j.rows;
  __shared__ float top[8][kJoinRows], total[8][kJoinRows];
  float m = -INFINITY;
#pragma unroll 4
  for (int i = sub; i < pieces; i += 8) m = fmaxf(m, in ? reinterpret_cast<const float2*>(slot(i))[row].x : -INFINITY);
  top[sub][r] = m;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 8; ++k) m = fmaxf(m, top[k][r]);
  const float ref = m == -INFINITY ? 0.f : m;
  float l = 0.f;
#pragma unroll 4
  for (int i = sub; i < pieces; i += 8) {
    const float2 x = in ? reinterpret_cast<const float2*>(slot(i))[row] : make_float2(-INFINITY, 0.f);
    const float w = exp2_fast(x.x - ref);
    weight[i * kJoinRows + r] = w;
    l = fmaf(x.y, w, l);
  }
  total[sub][r] = l;
  __syncthreads();
  if (!in) return;
  l = 0.f;
#pragma unroll
  for (int k = 0; k < 8; ++k) l += total[k][r];
  // D / 16 columns of float4 a CTA: the first D / 16 groups of threads take one each
  if (sub >= D / 4 / kJoinParts) return;
  const int c = blockIdx.z * (D / 4 / kJoinParts) + sub;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int i = 0; i < pieces; ++i) {
    const float4 v = reinterpret_cast<const float4*>(slot(i) + 2 * unit_rows)[(size_t)c * unit_rows + row];
    const float w = weight[i * kJoinRows + r];
    o.x = fmaf(v.x, w, o.x);
    o.y = fmaf(v.y, w, o.y);
    o.z = fmaf(v.z, w, o.z);
    o.w = fmaf(v.w, w, o.w);
  }
  const float inv = m == -INFINITY && l == 0.f ? 0.f : 1.f / l;
  const int g = j.row0 + row;
  __nv_bfloat16* const dst = a.out + (int64_t)(j.start + g / a.group) * a.out_stride +
                             (int64_t)(j.h * a.group + g % a.group) * D;
  reinterpret_cast<uint2*>(dst)[c] = make_uint2(pack_bf16x2(o.x * inv, o.y * inv), pack_bf16x2(o.z * inv, o.w * inv));
}

template <int D>
cudaError_t launch(const TreeAttnArgs& a, int grid, int unit_rows, cudaStream_t stream) {
  const auto kernel = attn_tree_split_kernel<D>;
  static bool configured[64] = {false};
  cudaError_t e = allow_shared(kernel, kSmem<D>, configured);
  if (e != cudaSuccess) return e;
  e = launch_pdl(kernel, dim3((unsigned)grid), dim3(kThreads), kSmem<D>, stream, a, unit_rows);
  if (e != cudaSuccess) return e;
  return launch_pdl(attn_tree_join_kernel<D>,
                    dim3((unsigned)grid, (unsigned)((unit_rows + kJoinRows - 1) / kJoinRows), kJoinParts), dim3(256),
                    (size_t)grid * kJoinRows * sizeof(float), stream, a, grid, unit_rows);
}

}  // namespace

int tree_split_grid() { return std::min(sm_count(), kMaxGrid); }

int tree_split_unit_rows(int64_t max_rows) {
  return (int)std::min<int64_t>(kUnitRows, (max_rows + 31) / 32 * 32);
}

int64_t tree_split_work_bytes(int grid, int unit_rows, int d) {
  return (int64_t)grid * (sizeof(Join) + 2 * sizeof(float) * (int64_t)unit_rows * (d + 2));
}

cudaError_t launch_tree_split(const TreeAttnArgs& a, int d, int grid, int unit_rows, cudaStream_t stream) {
  if (d == 64) return launch<64>(a, grid, unit_rows, stream);
  if (d == 96) return launch<96>(a, grid, unit_rows, stream);
  return launch<128>(a, grid, unit_rows, stream);
}

}  // namespace aiosb
