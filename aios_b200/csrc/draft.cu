// Drafted token trees around the forward: the ancestors' bits and positions of the nodes, and the
// verification of a tree against the target model's distributions.
#include <math_constants.h>

#include <algorithm>
#include <type_traits>

#include "abi_util.h"
#include "common.cuh"

namespace aiosb {
namespace {

// ---- ancestors' bits -------------------------------------------------------------------------
constexpr int kTreeThreads = 256;

// A CTA per tree, by doubling: with every node's bits of its 2^k nearest ancestors (itself among them) and its 2^k-th
// ancestor known, the ancestor's bits or-ed into its own are those of 2^(k + 1). So a chain of 256 takes eight rounds,
// where a walk from each node to its root takes 256 dependent loads (63 us, so 10; 256 mixed trees of up to 256 nodes 6.4).
// Bits may be or-ed while their owner adds to them: what it adds are ancestors as well. The ancestors' numbers have
// two buffers.
__global__ void __launch_bounds__(kTreeThreads)
    draft_tree_kernel(const int32_t* parents, const int32_t* tree_start, int tokens, int words,
                      const int32_t* cached_lens, int32_t* mask, int32_t* positions, int32_t* status) {
  extern __shared__ uint32_t bits[];  // [words, 32 * words]: a word of all nodes side by side
  __shared__ int16_t up[2][AIOSB_TREE_MAX_NODES], depth[2][AIOSB_TREE_MAX_NODES];
  const int r = blockIdx.x, most = 32 * words;
  pdl_enter();
  const int s = tree_start[r], e = tree_start[r + 1];
  const int base = cached_lens != nullptr ? cached_lens[r] : 0;
  const int start = min(max(s, 0), tokens), all = min(max(e, start), tokens) - start, n = min(all, most);
  if (threadIdx.x == 0 && (s < 0 || e < s || e > tokens || all > n)) report(status, AIOSB_DEV_TREE_RANGE);
  int open = 0;
  for (int i = threadIdx.x; i < n; i += kTreeThreads) {
    int p = parents[start + i];
    if (p < -1 || p >= i) {
      report(status, AIOSB_DEV_TREE_RANGE);
      p = -1;
    }
    up[0][i] = (int16_t)p;
    depth[0][i] = p >= 0;
    for (int w = 0; w < words; ++w) bits[w * most + i] = w == i >> 5 ? 1u << (i & 31) : 0u;
    open |= p >= 0;
  }
  int now = 0;
  while (__syncthreads_or(open)) {
    open = 0;
    for (int i = threadIdx.x; i < n; i += kTreeThreads) {
      const int a = up[now][i], d = depth[now][i];
      int next = -1, far = d;
      if (a >= 0) {
        next = up[now][a];
        far += depth[now][a];
        for (int w = 0; w <= a >> 5; ++w) bits[w * most + i] |= bits[w * most + a];  // ancestors' numbers are lower
      }
      up[now ^ 1][i] = (int16_t)next;
      depth[now ^ 1][i] = (int16_t)far;
      open |= next >= 0;
    }
    now ^= 1;
  }
  for (int i = threadIdx.x; i < n * words; i += kTreeThreads)
    mask[(int64_t)start * words + i] = (int32_t)bits[i % words * most + i / words];
  for (int i = threadIdx.x; i < n; i += kTreeThreads) positions[start + i] = base + depth[now][i];
  // nodes behind those that the words hold (reported above): nothing known
  for (int i = n + threadIdx.x; i < all; i += kTreeThreads) {
    for (int w = 0; w < words; ++w) mask[(int64_t)(start + i) * words + w] = 0;
    positions[start + i] = base;
  }
}

// ---- verification ----------------------------------------------------------------------------
constexpr int kVerifyThreads = 512;
constexpr int kVerifyWarps = kVerifyThreads / 32;
constexpr int kMaxRanks = 16;
constexpr int kGreedyRanks = 8;
constexpr int kBlockIds = 256;  // ids that a warp takes at a time, eight to a lane

struct VerifyArgs {
  const void* logits;
  int64_t logits_stride;
  int tokens, vocab;
  const int64_t* draft_tokens;
  const int32_t* parents;
  const int32_t* tree_start;
  const float* accept_u;
  const float* sample_u;
  double inv_temperature;
  const float* probs;
  int64_t probs_stride;
  int32_t* accepted;
  int64_t* next_token;
  int32_t* order;
  int32_t* status;
  int ranks;  // CTAs of a cluster: they share a request's vocabulary
  int run;    // places of a warp, a multiple of kRunIds
};

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ double warp_sum_f64(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float load_logit(const __nv_bfloat16* p) { return bf16_to_f(*p); }
__device__ __forceinline__ float load_logit(const float* p) { return *p; }

// A row of logits in groups of eight places that lie on 16 bytes: place p holds id p - shift, and the first group's
// first `shift` places and those from `end` on hold none. 16-byte loads reach up to 15 bytes over a row's ends, but
// never a 16-byte piece without any of the row.
template <typename T>
struct Places {
  const T* base;
  int shift, end;
  __device__ __forceinline__ Places(const T* row, int vocab) {
    shift = (int)((reinterpret_cast<uintptr_t>(row) & 15u) / sizeof(T));
    base = row - shift;
    end = vocab + shift;
  }
  __device__ __forceinline__ void load(int p, float (&x)[8]) const {
    if (p < end) {
      pieces(base, p, x);
    }
    if (p < shift || p + 8 > end) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (p + j < shift || p + j >= end) x[j] = -INFINITY;
    }
  }
  __device__ __forceinline__ void pieces(const __nv_bfloat16* from, int p, float (&x)[8]) const {
    const uint4 u = *reinterpret_cast<const uint4*>(from + p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[2 * j] = bf16_lo(w[j]);
      x[2 * j + 1] = bf16_hi(w[j]);
    }
  }
  __device__ __forceinline__ void pieces(const float* from, int p, float (&x)[8]) const {
    const float4 a = *reinterpret_cast<const float4*>(from + p);
    float4 b = make_float4(0.f, 0.f, 0.f, 0.f);
    if (p + 4 < end) b = *reinterpret_cast<const float4*>(from + p + 4);
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  }
};
// The eight values of `row` from index i on (0 outside of it), by 16-byte loads as above. The row's own place on 16
// bytes is the same for every i that is a multiple of eight apart.
__device__ __forceinline__ void load_probs(const float* row, int i, int vocab, float (&x)[8]) {
  const int over = (int)((reinterpret_cast<uintptr_t>(row + i) & 15u) / 4);
  float y[12];
#pragma unroll
  for (int g = 0; g < 3; ++g) {
    const int at = i - over + 4 * g;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if ((g < 2 || over > 0) && at + 3 >= 0 && at < vocab) v = *reinterpret_cast<const float4*>(row + at);
    y[4 * g] = v.x, y[4 * g + 1] = v.y, y[4 * g + 2] = v.z, y[4 * g + 3] = v.w;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] = over == 0 ? y[j] : over == 1 ? y[j + 1] : over == 2 ? y[j + 2] : y[j + 3];
  if (i < 0 || i + 8 > vocab) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (i + j < 0 || i + j >= vocab) x[j] = 0.f;
  }
}

// An fp32 value's bits as an fp64 one: the conversion instruction runs at an eighth of the fp64 rate. 0 and subnormals
// come out as values of 2^-127 or so, infinities and NaN as ones of 2^128.
__device__ __forceinline__ double widen(float x) {
  const uint32_t u = __float_as_uint(x);
  return __hiloint2double((int)((((u >> 3) & 0x0FFFFFFFu) + 0x38000000u) | (u & 0x80000000u)), (int)(u << 29));
}

__device__ __forceinline__ double positive(double x) {  // max(x, 0) of a number
  const int keep = ~(__double2hiint(x) >> 31);
  return __hiloint2double(__double2hiint(x) & keep, __double2loint(x) & keep);
}
// A probability times 2^-896 in fp64: its bits where an fp64 value has them, exact for 0 and subnormals too. nan becomes
// NaN where a value is infinite or NaN.
__device__ __forceinline__ double probability(float x, float& nan) {
  nan = fmaf(x, 0.f, nan);
  const uint32_t u = __float_as_uint(x);
  return __hiloint2double((int)((u >> 3 & 0x0FFFFFFFu) | (u & 0x80000000u)), (int)(u << 29));
}
// max(r - q, 0) for q as above. r comes rounded: a product's rest beside q would be left over where both are the same.
__device__ __forceinline__ double less(double r, double q) { return positive(fma(q, -0x1p896, r)); }

// 2^(i / 16) for the exponential below: sixteen doubles are all of the banks once, so that no two lanes' entries
// conflict (a table of 128 cost as much as the arithmetic).
constexpr int kExpTable = 16;
// e^((x - m) / T) in fp64 for x <= m: (x - m) / (T ln 2) = (k + f) / 16 with |f| <= 1/2, 2^(k / 16) from the table and
// k's upper bits, and 2^(f / 16) by its series to the sixth power (table-driven exponentials: P. T. P. Tang, ACM TOMS
// 15, 1989), whose rest is 2^-51. Twelve fp64 instructions, where the general function takes some thirty. Off by 2^-50,
// and by 2^-51 of (x - m) / T for the rounding of what it is taken of.
// scale: 16 / (T ln 2); base: m * scale (its rounding is a factor of the weights over it). Below m - 600 T, and for x
// of -inf, it is 0: a masked token adds nothing to any sum, so that a sum is above 0 exactly where one of its tokens is.
constexpr uint32_t kFar = 0xC0CB0D00u;  // upper half of -13850
// 2^(t / 16). FAR false: t is above -13850, or the result is not used.
template <bool FAR = true>
__device__ __forceinline__ double exp_table(double t, const double* table) {
  const double magic = 6755399441055744.0;  // 1.5 * 2^52: the sum's low bits are round(t)
  const double s = t + magic, f = t - (s - magic);
  const int k = __double2loint(s);
  constexpr double c = 0.043321698784996581;  // ln 2 / 16
  double p = fma(f, c * c * c * c * c * c / 720, c * c * c * c * c / 120);
  p = fma(f, p, c * c * c * c / 24);
  p = fma(f, p, c * c * c / 6);
  p = fma(f, p, c * c / 2);
  p = fma(f, p, c);
  const double b = table[k & (kExpTable - 1)];
  const double r = fma(b, f * p, b);
  if (FAR && (uint32_t)__double2hiint(t) >= kFar) return 0.0;
  return __hiloint2double(__double2hiint(r) + ((k >> 4) << 20), __double2loint(r));
}
template <bool FAR = true>
__device__ __forceinline__ double exp_table(float x, double scale, double base, const double* table) {
  return exp_table<FAR>(fma(widen(x), scale, -base), table);
}

// Values that the CTAs of a cluster hand to one another; the buffers take turns, so that one barrier an exchange is
// enough: a CTA writes a buffer again only behind the next barrier, which all have reached after reading it.
struct Exchange {
  double sum[2][kMaxRanks];
  float top[2][kMaxRanks];
  int arg[2][kMaxRanks];
};
__device__ __forceinline__ void hand_out(Exchange& e, int turn, int rank, int to, double sum, float top, int arg) {
  const uint32_t s = map_shared_rank(smem_u32(&e.sum[turn][rank]), to),
                 t = map_shared_rank(smem_u32(&e.top[turn][rank]), to),
                 a = map_shared_rank(smem_u32(&e.arg[turn][rank]), to);
  asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(s), "d"(sum) : "memory");
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(t), "f"(top) : "memory");
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(a), "r"(arg) : "memory");
}

// A request's tree in shared memory, and the path through it.
struct Walk {
  int16_t up[AIOSB_TREE_MAX_NODES];
  int16_t path[AIOSB_TREE_MAX_NODES];
  int16_t child[AIOSB_TREE_MAX_NODES];  // the current node's children
  uint32_t on_path[AIOSB_TREE_MAX_NODES / 32];
  int children;
};
__device__ __forceinline__ void list_children(Walk& w, int cur, int n) {  // one warp
  const int lane = threadIdx.x & 31;
  int count = 0;
  for (int j0 = (cur + 1) & ~31; j0 < n; j0 += 32) {
    const int j = j0 + lane;
    const bool is = j > cur && j < n && w.up[j] == cur;
    const unsigned some = __ballot_sync(0xffffffffu, is);
    if (is) w.child[count + __popc(some & ((1u << lane) - 1))] = (int16_t)j;
    count += __popc(some);
  }
  if (lane == 0) w.children = count;
}
// Bit i of `repeated`: a child before child i has its token. One warp, behind list_children.
__device__ __forceinline__ void mark_repeated(const Walk& w, const int32_t* child_x, uint32_t* repeated) {
  const int lane = threadIdx.x & 31, n = w.children;
  for (int i0 = 0; i0 < n; i0 += 32) {
    const int x = i0 + lane < n ? child_x[i0 + lane] : -2 - lane;
    bool again = (__match_any_sync(0xffffffffu, x) & ((1u << lane) - 1)) != 0;
    for (int j = 0; j < i0; ++j) again |= child_x[j] == x;
    const unsigned some = __ballot_sync(0xffffffffu, again);
    if (lane == 0) repeated[i0 >> 5] = some;
  }
}
// Writes the path, then the other nodes; one warp.
__device__ __forceinline__ void write_order(const Walk& w, int depth, int n, int all, int32_t* order) {
  const int lane = threadIdx.x & 31;
  for (int i = lane; i <= depth; i += 32) order[i] = w.path[i];
  int at = depth + 1;
  for (int j0 = 0; j0 < all; j0 += 32) {
    const int j = j0 + lane;
    const bool rest = j < all && !(j < n && ((w.on_path[j >> 5] >> (j & 31)) & 1));
    const unsigned some = __ballot_sync(0xffffffffu, rest);
    if (rest) order[at + __popc(some & ((1u << lane) - 1))] = j;
    at += __popc(some);
  }
}

// Of node i; -1 for what is not the number of a node before it.
__device__ __forceinline__ int16_t parent_of(const VerifyArgs& a, int start, int i, bool tell) {
  const int p = a.parents[start + i];
  if (p >= -1 && p < i) return (int16_t)p;
  if (tell) report(a.status, AIOSB_DEV_TREE_RANGE);
  return -1;
}

struct TreeRows {
  int start, n, all;
};
// Request r's rows; false: it has none, and its outputs are written.
__device__ __forceinline__ bool tree_rows(const VerifyArgs& a, int r, bool first, TreeRows& t) {
  const int s = a.tree_start[r], e = a.tree_start[r + 1];
  t.start = min(max(s, 0), a.tokens);
  t.all = min(max(e, t.start), a.tokens) - t.start;
  t.n = min(t.all, AIOSB_TREE_MAX_NODES);
  if (first && (s < 0 || e < s || e > a.tokens || t.all > t.n)) report(a.status, AIOSB_DEV_TREE_RANGE);
  if (t.n == 0 && first) {
    a.accepted[r] = 0;
    a.next_token[r] = -1;
  }
  return t.n > 0;
}

// Greedy: a node's argmax decides. A cluster per request; each warp looks through every (ranks x warps)th block. Bound
// by the latency of the visited nodes, one after another (a row's loads, the exchange): 24 trees of 13 at 50021 fp32
// ids 17.4 us. Four blocks in flight in place of two took 20 to 30% longer: the registers.
template <typename T>
__global__ void __launch_bounds__(kVerifyThreads, 1) verify_greedy_kernel(const VerifyArgs a) {
  __shared__ Walk walk;
  __shared__ Exchange ex;
  __shared__ float warp_top[kVerifyWarps];
  __shared__ int warp_arg[kVerifyWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int ranks = a.ranks, rank = (int)cluster_ctarank(), r = blockIdx.x / ranks;
  pdl_enter();
  TreeRows t;
  if (!tree_rows(a, r, rank == 0 && threadIdx.x == 0, t)) return;  // the whole cluster leaves
  for (int i = threadIdx.x; i < t.n; i += kVerifyThreads) walk.up[i] = parent_of(a, t.start, i, rank == 0);
  if (threadIdx.x < AIOSB_TREE_MAX_NODES / 32) walk.on_path[threadIdx.x] = threadIdx.x == 0 ? 1u : 0u;
  if (threadIdx.x == 0) walk.path[0] = 0;
  cluster_sync();  // every CTA runs: its shared memory may be written

  int cur = 0, depth = 0, turn = 0;
  int64_t token = -1;
  for (;;) {
    const T* const row = reinterpret_cast<const T*>(a.logits) + (int64_t)(t.start + cur) * a.logits_stride;
    const Places<T> places(row, a.vocab);
    float top = -INFINITY;
    int arg = INT32_MAX;
    // ids ascend within a lane, so that the first of equal ones stays
#pragma unroll 2
    for (int p = (rank * kVerifyWarps + warp) * kBlockIds + lane * 8; p < places.end;
         p += ranks * kVerifyWarps * kBlockIds) {
      float x[8];
      places.load(p, x);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (x[j] > top) arg = p + j - places.shift;
        top = max_nan(top, x[j]);
      }
    }
    auto join = [&](float x, int b) {
      arg = x > top ? b : x == top ? min(arg, b) : arg;
      top = max_nan(top, x);
    };
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) join(__shfl_xor_sync(0xffffffffu, top, o), __shfl_xor_sync(0xffffffffu, arg, o));
    if (lane == 0) {
      warp_top[warp] = top;
      warp_arg[warp] = arg;
    }
    __syncthreads();
    if (warp == 0) {
      top = lane < kVerifyWarps ? warp_top[lane] : -INFINITY;
      arg = lane < kVerifyWarps ? warp_arg[lane] : INT32_MAX;
#pragma unroll
      for (int o = kVerifyWarps / 2; o > 0; o >>= 1)
        join(__shfl_xor_sync(0xffffffffu, top, o), __shfl_xor_sync(0xffffffffu, arg, o));
      if (lane < ranks) hand_out(ex, turn, rank, lane, 0.0, top, arg);
      list_children(walk, cur, t.n);
    }
    cluster_sync();
    top = ex.top[turn][0];
    arg = ex.arg[turn][0];
    for (int c = 1; c < ranks; ++c) join(ex.top[turn][c], ex.arg[turn][c]);
    turn ^= 1;
    if (!(top > -INFINITY)) {  // NaN, or -inf only
      if (rank == 0 && threadIdx.x == 0) report(a.status, AIOSB_DEV_NO_DISTRIBUTION);
      break;
    }
    int found = INT32_MAX;
    for (int i = threadIdx.x & 31; i < walk.children; i += 32) {
      const int64_t x = a.draft_tokens[t.start + walk.child[i]];
      if (x < 0 || x >= a.vocab) {
        if (rank == 0) report(a.status, AIOSB_DEV_TOKEN_RANGE);
      } else if (x == arg) {
        found = min(found, walk.child[i]);
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) found = min(found, __shfl_xor_sync(0xffffffffu, found, o));
    if (found == INT32_MAX) {
      token = arg;
      break;
    }
    cur = found;
    ++depth;
    __syncthreads();  // the children have been read
    if (threadIdx.x == 0) {
      walk.path[depth] = (int16_t)cur;
      walk.on_path[cur >> 5] |= 1u << (cur & 31);
    }
  }
  if (rank != 0 || warp != 0) return;
  __syncwarp();
  if (lane == 0) {
    a.accepted[r] = depth;
    a.next_token[r] = token;
  }
  write_order(walk, depth, t.n, t.all, a.order + t.start);
}

// Sampling. A cluster per request walks its tree from the root. The vocabulary is cut into one run of ids per warp
// of the cluster, in ascending order, and a node's weights r stay in shared memory in fp64 while its children are
// tried, so that a row is read once. (Without probabilities the proposals are taken out of it and stand beside it: a
// rejection changes no other weight.) A pass leaves each warp the sum of its run and each CTA the sum of its warps';
// a token is found by these sums from the outside in. Sums are taken in a fixed order, in fp64: what is accepted or
// drawn hangs on comparisons of them.
// Bound by the latency of the visited nodes: some 7000 clocks each for the row's loads, twelve fp64 instructions to an
// exponential, and the cluster's exchange; with many requests by the fp64 pipes and the passes over shared memory. A
// chain of 5 at 16384 ids with probabilities 14.1 us, 16 trees of 26 at 32001 ids without 18.4, 64 trees of 24 with
// them at 131072 ids 135 (with one CTA to an SM it was 196 to 128).
// A warp's run of a row is a multiple of this; a row comes as fp32 into the first half of its groups' places.
constexpr int kRunIds = 64;

template <typename T, bool PROBS>
__global__ void __launch_bounds__(kVerifyThreads, 2) verify_kernel(const VerifyArgs a) {
  extern __shared__ __align__(16) double weights[];
  __shared__ Walk walk;
  __shared__ Exchange ex;
  __shared__ double table[kExpTable];
  __shared__ double child_r[AIOSB_TREE_MAX_NODES];  // the children's r, and what they were drawn with
  __shared__ float child_q[AIOSB_TREE_MAX_NODES], node_u[AIOSB_TREE_MAX_NODES];
  __shared__ int32_t node_x[AIOSB_TREE_MAX_NODES];  // the nodes' tokens; -1: none of the vocabulary
  __shared__ int32_t child_x[AIOSB_TREE_MAX_NODES];
  __shared__ double warp_sum_of[kVerifyWarps];
  __shared__ float warp_top[kVerifyWarps];
  __shared__ double factor[kMaxRanks];  // of the ranks' weights: they are stored over the rank's own maximum
  __shared__ double all_weights;
  // without probabilities: the children's repeated tokens, the child that is accepted (-1: none), and the only token
  // that is left (-1: there are others)
  __shared__ uint32_t repeated[AIOSB_TREE_MAX_NODES / 32];
  __shared__ int accepted_child, only_token;

  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int ranks = a.ranks, rank = (int)cluster_ctarank(), r = blockIdx.x / ranks;
  if (threadIdx.x < kExpTable) table[threadIdx.x] = exp2((double)threadIdx.x / kExpTable);
  pdl_enter();
  TreeRows t;
  const bool first = rank == 0 && threadIdx.x == 0;
  if (!tree_rows(a, r, first, t)) return;  // the whole cluster leaves
  for (int i = threadIdx.x; i < t.n; i += kVerifyThreads) {
    const int64_t x = a.draft_tokens[t.start + i];
    walk.up[i] = parent_of(a, t.start, i, rank == 0);
    node_x[i] = x >= 0 && x < a.vocab ? (int32_t)x : -1;
    node_u[i] = a.accept_u[t.start + i];
  }
  if (threadIdx.x < AIOSB_TREE_MAX_NODES / 32) walk.on_path[threadIdx.x] = threadIdx.x == 0 ? 1u : 0u;
  if (threadIdx.x == 0) walk.path[0] = 0;
  cluster_sync();  // every CTA runs: its shared memory may be written

  const double scale = a.inv_temperature * (1.4426950408889634 * kExpTable);
  // places of the row (Places), not ids
  const int per_rank = a.run * kVerifyWarps, rank_lo = rank * per_rank, lo = rank_lo + warp * a.run;
  // Groups of eight, a lane each; their 16-byte pieces change places from one pair of groups to the next, so that
  // eight lanes' pieces lie on different banks (runs are multiples of 64, so a lane's groups all have its order).
  auto group_of = [&](int p) { return weights + (p - rank_lo); };
  const int swap = (lane >> 1) & 3;
  auto load_group = [&](const double* g, double (&w)[8]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const double2 d = reinterpret_cast<const double2*>(g)[j ^ swap];
      w[2 * j] = d.x;
      w[2 * j + 1] = d.y;
    }
  };
  auto store_group = [&](double* g, const double (&w)[8]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) reinterpret_cast<double2*>(g)[j ^ swap] = make_double2(w[2 * j], w[2 * j + 1]);
  };

  int turn = 0, cur = 0, depth = 0, last_turn = 0;
  // The sums of the warps' runs within the CTA, then of the CTAs (ex.sum, in rank order); `top` goes along.
  auto exchange = [&](double mine, float top) {
    mine = warp_sum_f64(mine);
    __syncthreads();
    if (lane == 0) warp_sum_of[warp] = mine;
    __syncthreads();
    if (warp == 0) {
      double v = warp_sum_of[lane & (kVerifyWarps - 1)];
#pragma unroll
      for (int o = kVerifyWarps / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
      if (lane < ranks) hand_out(ex, turn, rank, lane, v, top, 0);
    }
    cluster_sync();
    last_turn = turn;
    turn ^= 1;
  };
  auto total_sum = [&] {
    double v = 0;
    for (int c = 0; c < ranks; ++c) v += ex.sum[last_turn][c];
    return v;
  };

  for (;;) {
    const T* const row = reinterpret_cast<const T*>(a.logits) + (int64_t)(t.start + cur) * a.logits_stride;
    const float* const q = PROBS ? a.probs + (int64_t)(t.start + cur) * a.probs_stride : nullptr;
    const Places<T> places(row, a.vocab);
    const int shift = places.shift;
    const int hi = max(lo, min(lo + a.run, places.end));  // of this warp: [lo, hi), the last group in full
    // the children; their logits and probabilities are asked for ahead of the row's, a lane each
    float child_l = -INFINITY, child_p = 0.f;
    if (warp == 0) {
      list_children(walk, cur, t.n);
      __syncwarp();
      if (lane < walk.children) {
        const int x = node_x[walk.child[lane]];
        if (x >= 0) {
          child_l = load_logit(row + x);
          if (PROBS) child_p = q[x];
        }
      }
      for (int i = lane; i < walk.children; i += 32) child_x[i] = node_x[walk.child[i]];
      __syncwarp();
      if (!PROBS) mark_repeated(walk, child_x, repeated);
    }
    // ---- the row, as it is, to its place; its maximum
    float top = -INFINITY, low = INFINITY;
#pragma unroll 2
    for (int p = lo + lane * 8; p < hi; p += kBlockIds) {
      float x[8];
      places.load(p, x);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        top = max_nan(top, x[j]);
        low = fminf(low, x[j]);
      }
      float4* const g = reinterpret_cast<float4*>(group_of(p));
      g[swap] = make_float4(x[0], x[1], x[2], x[3]);
      g[1 ^ swap] = make_float4(x[4], x[5], x[6], x[7]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (lane == 0) warp_top[warp] = top;
    if (warp == 0) {
      for (int i = lane; i < walk.children; i += 32) {
        const int x = child_x[i];
        if (x < 0 && rank == 0) report(a.status, AIOSB_DEV_TOKEN_RANGE);
        if (i >= 32) {
          child_l = x >= 0 ? load_logit(row + x) : -INFINITY;
          if (PROBS) child_p = x >= 0 ? q[x] : 0.f;
        }
        *reinterpret_cast<float*>(&child_r[i]) = child_l;
        if (PROBS) child_q[i] = child_p;
      }
    }
    __syncthreads();
    top = lane < kVerifyWarps ? warp_top[lane] : -INFINITY;
#pragma unroll
    for (int o = kVerifyWarps / 2; o > 0; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
    top = __shfl_sync(0xffffffffu, top, 0);
    const int children = walk.children;
    if (!PROBS) {  // proposals stand beside the others' weights (below): out of the row, whose values are still fp32
      for (int i = lane; i < children; i += 32) {
        const int x = child_x[i], place = x + shift;
        if (x >= 0 && place >= lo && place < hi) {
          const int at = place - rank_lo;
          reinterpret_cast<float*>(weights)[(at & ~7) * 2 + ((((at >> 4) & 3) ^ ((at >> 2) & 1)) << 2) + (at & 3)] =
              -INFINITY;
          low = -INFINITY;
        }
      }
      __syncwarp();
    }
    // ---- weights over this CTA's maximum (one that is NaN or +inf ends the walk below; -inf leaves nothing)
    double part = 0;
    const double mine = widen(top > -INFINITY ? top : 0.f) * scale;
    auto weigh = [&](auto any) {
#pragma unroll 1
      for (int v = lo + lane * 8; v < hi; v += kBlockIds) {
        double* const g = group_of(v);
        const float4 x0 = reinterpret_cast<const float4*>(g)[swap], x1 = reinterpret_cast<const float4*>(g)[1 ^ swap];
        const float x[8] = {x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w};
        double e[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) e[j] = exp_table<any.value>(x[j], scale, mine, table);
        if (v < shift || v + 8 > places.end) {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (v + j < shift || v + j >= places.end) e[j] = 0;
        }
        store_group(g, e);
        part += ((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7]));
      }
    };
    // 0 for a far value takes three instructions of a thread: only where the warp has one
    if (__any_sync(0xffffffffu, (uint32_t)__double2hiint(fma(widen(low), scale, -mine)) >= kFar)) weigh(std::true_type());
    else weigh(std::false_type());
    exchange(part, top);
    float most = -INFINITY;
    for (int c = 0; c < ranks; ++c) most = max_nan(most, ex.top[last_turn][c]);
    if (!(fabsf(most) < INFINITY)) {  // NaN, -inf only, or +inf
      if (first) {
        report(a.status, AIOSB_DEV_NO_DISTRIBUTION);
        a.next_token[r] = -1;
      }
      break;
    }
    // ---- what the ranks' weights count, and the children's r
    const double all = widen(most) * scale;
    // from the rounded base that the rank's weights are over: its rounding is up to 2^-54 of m / T, and would stand
    // between one rank's weights and another's
    auto factor_of = [&](int c) {
      const float m = ex.top[last_turn][c];
      return m > -INFINITY ? exp_table(__dmul_rn(widen(m), scale) - all, table) : 0.0;
    };
    auto child_weight = [&](int i) {
      const int x = child_x[i];
      if (x < 0) return 0.0;
      const int owner = (x + shift) / per_rank;
      const float m = ex.top[last_turn][owner];
      if (!(m > -INFINITY)) return 0.0;
      return exp_table(*reinterpret_cast<const float*>(&child_r[i]), scale, widen(m) * scale, table) * factor_of(owner);
    };
    if (PROBS && warp == 1) {
      for (int i = lane; i < children; i += 32) child_r[i] = child_weight(i);
    } else if (warp < 2) {
      const int c = lane & (kMaxRanks - 1);
      const double f = c < ranks ? factor_of(c) : 0.0;
      double z = c < ranks ? f * ex.sum[last_turn][c] : 0.0;
#pragma unroll
      for (int o = kMaxRanks / 2; o > 0; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
      if (warp == 0) {
        if (lane < ranks) factor[lane] = f;
        if (lane == 0) all_weights = z;
      } else if (!PROBS) {
        // Where child i is tried, what is left is z, the weights of the tokens that nobody proposed, and those of the
        // proposals from i on: a sum from the last one back, never a difference, which would lose its digits when a
        // rejected token had most of the weight.
        double behind = z;
        int found = -1, last = -1;
        for (int i0 = (children - 1) & ~31; i0 >= 0; i0 -= 32) {
          const int i = i0 + lane;
          const bool tried = i < children && !((repeated[i0 >> 5] >> lane) & 1);
          const double w = tried ? child_weight(i) : 0.0;
          double from = w;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const double y = __shfl_down_sync(0xffffffffu, from, o);
            if (lane + o < 32) from += y;
          }
          from += behind;
          const unsigned yes =
              __ballot_sync(0xffffffffu, w > 0 && (double)node_u[walk.child[min(i, children - 1)]] * from < w);
          const unsigned some = __ballot_sync(0xffffffffu, w > 0);
          if (yes) found = i0 + __ffs(yes) - 1;
          if (some && last < 0) last = i0 + 31 - __clz(some);
          behind = __shfl_sync(0xffffffffu, from, 0);
        }
        int only = -1;
        if (found < 0 && !(z > 0) && last >= 0) {
          // rejecting the last proposal would leave nothing: r stays as it was, that token alone, and a later child
          // with the same token may still be accepted
          only = child_x[last];
          int again = INT32_MAX;
          for (int i = last + 1 + lane; i < children; i += 32)
            if (child_x[i] == only && node_u[walk.child[i]] < 1.f) again = min(again, i);
          again = __reduce_min_sync(0xffffffffu, again);
          if (again < INT32_MAX) found = again;
        }
        if (lane == 0) {
          accepted_child = found;
          only_token = only;
        }
      }
    }
    __syncthreads();

    // ---- with probabilities: the children, in ascending order. r(v) is weights(v) * mult, behind `pending`, the last
    // subtraction
    double mult = factor[rank], pending = 0;
    bool stale = false;  // the runs' sums are not r's
    int found = -1;
    float nan = 0.f;  // NaN: one of the probabilities that were read is no number
    if (!PROBS) {
      if (accepted_child >= 0) found = walk.child[accepted_child];
    } else {
      double total = all_weights;
      for (int i = 0; i < children; ++i) {
        const double rx = child_r[i], qx = probability(child_q[i], nan) * 0x1p896;
        const int child = walk.child[i];
        if (isnan(nan)) break;
        if (rx > 0 && (double)node_u[child] * qx * total < rx) {
          found = child;
          break;
        }
        if (child_x[i] < 0) continue;
        const double inv = 1.0 / total;
        part = 0;
#pragma unroll 1
        for (int p = lo + lane * 8; p < hi; p += kBlockIds) {
          double* const g = group_of(p);
          float qv[8];
          load_probs(q, p - shift, a.vocab, qv);
          double w[8], sum = 0;
          load_group(g, w);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const double qj = probability(qv[j], nan);
            w[j] *= mult;
            if (pending != 0) w[j] = less(w[j] * pending, qj);
            sum += less(w[j] * inv, qj);
          }
          store_group(g, w);
          part += sum;
        }
        mult = 1;
        exchange(part + nan, 0.f);
        const double left = total_sum();
        nan = isnan(left) ? CUDART_NAN_F : 0.f;  // in all threads
        if (isnan(left)) break;
        pending = left > 0 ? inv : 0;  // where nothing is left r stays
        stale = !(left > 0);
        if (left > 0) {
          total = left;
          for (int c = threadIdx.x; c < children; c += kVerifyThreads)
            child_r[c] = less(child_r[c] * inv, probability(child_q[c], nan));
          __syncthreads();
        }
      }
    }
    if (PROBS && isnan(nan)) {
      if (first) {
        report(a.status, AIOSB_DEV_NO_DISTRIBUTION);
        a.next_token[r] = -1;
      }
      break;
    }
    if (found >= 0) {
      cur = found;
      ++depth;
      __syncthreads();  // the children have been read
      if (threadIdx.x == 0) {
        walk.path[depth] = (int16_t)cur;
        walk.on_path[cur >> 5] |= 1u << (cur & 31);
      }
      continue;
    }

    // ---- the next token
    if (!PROBS && only_token >= 0) {
      if (first) a.next_token[r] = only_token;
      break;
    }
    // the first pass's sums and weights are over the ranks' own maxima, later ones are r's (without probabilities
    // there are none: the row's weights have no proposal's)
    const bool direct = stale || pending != 0;
    auto group_weights = [&](int p, double (&w)[8]) {  // the group at p, as the sums have it
      load_group(group_of(p), w);
      float qv[8];
      if (PROBS && pending != 0) load_probs(q, p - shift, a.vocab, qv);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (PROBS && pending != 0) w[j] = less(w[j] * pending, probability(qv[j], nan));
      }
    };
    if (stale) {
      part = 0;
      for (int p = lo + lane * 8; p < hi; p += kBlockIds) {
        double w[8];
        group_weights(p, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) part += w[j];
      }
      exchange(part, 0.f);
    }
    auto rank_sum = [&](int c) { return ex.sum[last_turn][c] * (direct ? 1.0 : factor[c]); };
    double target = 0, before = 0, owner_before = 0;
    for (int c = 0; c < ranks; ++c) target += rank_sum(c);
    target *= (double)a.sample_u[r];
    // the first whose end lies past the target; the last with any weight, should rounding leave none
    int owner = -1;
    for (int c = 0; c < ranks; ++c) {
      const double w = rank_sum(c);
      if (w > 0) {
        owner = c;
        owner_before = before;
        if (before + w > target) break;
      }
      before += w;
    }
    if (owner < 0 && first) {  // no token has any weight
      report(a.status, AIOSB_DEV_NO_DISTRIBUTION);
      a.next_token[r] = -1;
    }
    if (owner == rank) {
      // (over the rank's own maximum: far below the others' its weights times their factor may all be 0)
      if (!direct) target = (target - owner_before) / factor[rank];
      int own_warp = -1;
      double warp_before = 0;
      before = direct ? owner_before : 0;
      for (int w = 0; w < kVerifyWarps; ++w) {
        const double x = warp_sum_of[w];
        if (x > 0) {
          own_warp = w;
          warp_before = before;
          if (before + x > target) break;
        }
        before += x;
      }
      if (warp == own_warp) {
        before = warp_before;
        int pick = -1;
        for (int base = lo; base < hi; base += kBlockIds) {
          const int p = base + lane * 8;
          double w[8] = {}, sum = 0;
          if (p < hi) group_weights(p, w);
          int last = -1;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            if (w[j] > 0) last = p + j - shift;
            sum += w[j];
          }
          double upto = sum;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const double y = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += y;
          }
          const unsigned some = __ballot_sync(0xffffffffu, last >= 0);
          const unsigned past = __ballot_sync(0xffffffffu, last >= 0 && before + upto > target);
          if (past) {
            const int l = __ffs(past) - 1;
            double c = before + (upto - sum);
            pick = last;
#pragma unroll
            for (int j = 0; j < 8; ++j) {  // the first one past the target
              c += w[j];
              if (w[j] > 0 && c > target) {
                pick = p + j - shift;
                c = -INFINITY;
              }
            }
            pick = __shfl_sync(0xffffffffu, pick, l);
            break;
          }
          if (some) pick = __shfl_sync(0xffffffffu, last, 31 - __clz(some));
          before += __shfl_sync(0xffffffffu, upto, 31);
        }
        if (lane == 0) a.next_token[r] = pick;
      }
    }
    break;
  }

  __syncthreads();
  if (rank != 0 || warp != 0) return;
  if (lane == 0) a.accepted[r] = depth;
  write_order(walk, depth, t.n, t.all, a.order + t.start);
}

constexpr int kMaxSamplePlaces = 262144;
constexpr size_t kWeightBytes = sizeof(double) * kMaxSamplePlaces / kMaxRanks;
constexpr size_t kSharedBytes = 80 * 1024;  // of two CTAs on an SM, 32 KiB beside it

template <typename Kernel>
cudaError_t launch_cluster(Kernel kernel, const VerifyArgs& a, int requests, size_t smem, bool (&configured)[64],
                           cudaStream_t stream) {
  const cudaError_t e = allow_shared(kernel, smem > 0 ? (int)kWeightBytes : 0, configured, true);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(requests * a.ranks));
  cfg.blockDim = dim3(kVerifyThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)a.ranks;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kernel, a);
}

int warp_run(int places, int ranks) {
  const int runs = (places + kRunIds - 1) / kRunIds, warps = ranks * kVerifyWarps;
  return (runs + warps - 1) / warps * kRunIds;
}
size_t weight_bytes(int run) { return (size_t)run * kVerifyWarps * sizeof(double); }

// Places of a row (Places): more than its ids where a row may start anywhere on 16 bytes.
int64_t row_places(const void* logits, int64_t stride, int64_t vocab, int64_t tokens, int value_bytes) {
  const bool aligned = aligned16(logits) && (tokens <= 1 || stride * value_bytes % 16 == 0);
  return vocab + (aligned ? 0 : 16 / value_bytes - 1);
}

template <typename T>
cudaError_t launch_verify(VerifyArgs a, int requests, bool greedy, int places, cudaStream_t stream) {
  a.ranks = 1;
  const int sms = sm_count();
  // More CTAs to a request while they find SMs, and a block to each of their warps: two for the argmax, which has
  // little to do with one (1 x 16384 ids 5.7 us with 4 CTAs, 6.2 with 8). Sampling, us: 16 trees of 26, 32001 ids: 4
  // CTAs 26.2, 8 22.9; 2 of 8, 6400 ids: 1 CTA 15.2, 2 12.5; 8 of 8, 50021 ids: 8 CTAs 14.0, 16 12.9, with
  // probabilities 19.6 and 18.5.
  const int64_t each = (int64_t)kVerifyWarps * kBlockIds * (greedy ? 2 : 1);
  while (a.ranks < (greedy ? kGreedyRanks : kMaxRanks) && (int64_t)requests * a.ranks * 2 <= sms &&
         a.vocab >= a.ranks * each)
    a.ranks *= 2;
  static bool configured[3][64] = {};
  if (greedy) return launch_cluster(verify_greedy_kernel<T>, a, requests, 0, configured[0], stream);
  // two CTAs to an SM if the weights allow it
  while (a.ranks < kMaxRanks && weight_bytes(warp_run(places, a.ranks)) > kSharedBytes) a.ranks *= 2;
  a.run = warp_run(places, a.ranks);
  const size_t smem = weight_bytes(a.run);
  if (a.probs != nullptr) return launch_cluster(verify_kernel<T, true>, a, requests, smem, configured[1], stream);
  return launch_cluster(verify_kernel<T, false>, a, requests, smem, configured[2], stream);
}

}  // namespace
}  // namespace aiosb

using namespace aiosb;

extern "C" int aiosb_draft_tree(const int32_t* parents, int64_t tokens, const int32_t* tree_start, int64_t requests,
                                int64_t words, const int32_t* cached_lens, int32_t* mask, int32_t* positions,
                                int32_t* status, void* stream) {
  AIOSB_REQUIRE(tokens >= 0 && requests >= 0 && tokens <= INT32_MAX && requests <= INT32_MAX, AIOSB_ERR_INVALID_ARG,
                "draft_tree: bad sizes");
  AIOSB_REQUIRE(words >= 1 && words <= AIOSB_TREE_MAX_NODES / 32, AIOSB_ERR_UNSUPPORTED,
                "draft_tree: %lld mask words; a tree has at most %d nodes", (long long)words, AIOSB_TREE_MAX_NODES);
  if (tokens == 0 || requests == 0) return AIOSB_OK;
  AIOSB_REQUIRE(parents && tree_start && mask && positions, AIOSB_ERR_INVALID_ARG, "draft_tree: null pointer");
  static bool configured[64] = {false};
  constexpr int most = AIOSB_TREE_MAX_NODES / 32 * (AIOSB_TREE_MAX_NODES / 32) * 128;  // bytes of `bits`
  cudaError_t result = allow_shared(draft_tree_kernel, most, configured);
  if (result == cudaSuccess)
    result = launch_pdl(draft_tree_kernel, dim3((unsigned)requests), dim3(kTreeThreads), (size_t)(words * words * 128),
                        as_stream(stream), parents, tree_start, (int)tokens, (int)words, cached_lens, mask, positions,
                        status);
  return check_launch("draft_tree", result);
}

extern "C" int aiosb_verify_draft(const void* logits, int logits_fp32, int64_t logits_stride, int64_t tokens,
                                  int64_t vocab, const int64_t* draft_tokens, const int32_t* parents,
                                  const int32_t* tree_start, int64_t requests, const float* accept_uniforms,
                                  const float* sample_uniforms, double temperature, int greedy,
                                  const float* draft_probs, int64_t probs_stride, int32_t* accepted,
                                  int64_t* next_token, int32_t* order, int32_t* status, void* stream) {
  AIOSB_REQUIRE(tokens >= 0 && requests >= 0 && vocab >= 1 && tokens <= INT32_MAX && requests <= INT32_MAX / kMaxRanks,
                AIOSB_ERR_INVALID_ARG, "verify_draft: bad sizes");
  const int64_t places = row_places(logits, logits_stride, vocab, tokens, logits_fp32 ? 4 : 2);
  AIOSB_REQUIRE((greedy ? vocab : places) <= (greedy ? 1 << 30 : kMaxSamplePlaces), AIOSB_ERR_UNSUPPORTED,
                "verify_draft: vocabulary too large (sampling: at most %d, less 7 where rows are not on 16 bytes)",
                kMaxSamplePlaces);
  AIOSB_REQUIRE(logits_stride >= vocab || tokens <= 1, AIOSB_ERR_INVALID_ARG,
                "verify_draft: logits row stride below the vocabulary");
  AIOSB_REQUIRE(greedy || (temperature >= 1e-6 && temperature <= 1e6), AIOSB_ERR_INVALID_ARG,
                "verify_draft: the temperature must be in [1e-6, 1e6]");
  AIOSB_REQUIRE(!(greedy && draft_probs != nullptr), AIOSB_ERR_INVALID_ARG,
                "verify_draft: greedy verification takes no draft_probs");
  AIOSB_REQUIRE(draft_probs == nullptr || probs_stride >= vocab || tokens <= 1, AIOSB_ERR_INVALID_ARG,
                "verify_draft: draft_probs row stride below the vocabulary");
  if (requests == 0) return AIOSB_OK;
  AIOSB_REQUIRE(tree_start && accepted && next_token, AIOSB_ERR_INVALID_ARG, "verify_draft: null pointer");
  AIOSB_REQUIRE(tokens == 0 || (logits && draft_tokens && parents && order), AIOSB_ERR_INVALID_ARG,
                "verify_draft: null pointer");
  AIOSB_REQUIRE(greedy || tokens == 0 || (accept_uniforms && sample_uniforms), AIOSB_ERR_INVALID_ARG,
                "verify_draft: sampling needs uniforms");
  VerifyArgs a;
  a.logits = logits;
  a.logits_stride = logits_stride;
  a.tokens = (int)tokens;
  a.vocab = (int)vocab;
  a.draft_tokens = draft_tokens;
  a.parents = parents;
  a.tree_start = tree_start;
  a.accept_u = accept_uniforms;
  a.sample_u = sample_uniforms;
  a.inv_temperature = greedy ? 1.0 : 1.0 / temperature;
  a.probs = draft_probs;
  a.probs_stride = probs_stride;
  a.accepted = accepted;
  a.next_token = next_token;
  a.order = order;
  a.status = status;
  cudaStream_t s = as_stream(stream);
  const auto launch = logits_fp32 ? launch_verify<float> : launch_verify<__nv_bfloat16>;
  return check_launch("verify_draft", launch(a, (int)requests, greedy != 0, (int)places, s));
}
