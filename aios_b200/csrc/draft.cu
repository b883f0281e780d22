// Drafted token trees around the forward: the ancestors' bits and positions of the nodes, and the
// verification of a tree against the target model's distributions.
#include <algorithm>

#include "abi_util.h"
#include "common.cuh"

namespace aiosb {
namespace {

// ---- ancestors' bits -------------------------------------------------------------------------
constexpr int kTreeThreads = 256;

// A CTA per tree, a warp per node: lane w holds word w of the node's bits while the warp walks from
// the node to its root through the parents in shared memory.
__global__ void __launch_bounds__(kTreeThreads)
    draft_tree_kernel(const int32_t* parents, const int32_t* tree_start, int tokens, int words,
                      const int32_t* cached_lens, int32_t* mask, int32_t* positions, int32_t* status) {
  __shared__ int32_t up[AIOSB_TREE_MAX_NODES];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int r = blockIdx.x;
  pdl_enter();
  const int s = tree_start[r], e = tree_start[r + 1];
  const int start = min(max(s, 0), tokens), n = min(max(e, start), tokens) - start;
  if (threadIdx.x == 0 && (s < 0 || e < s || e > tokens || n > words * 32)) report(status, AIOSB_DEV_TREE_RANGE);
  const int staged = min(n, AIOSB_TREE_MAX_NODES);
  for (int i = threadIdx.x; i < staged; i += kTreeThreads) {
    int p = parents[start + i];
    if (p < -1 || p >= i) {
      report(status, AIOSB_DEV_TREE_RANGE);
      p = -1;
    }
    up[i] = p;
  }
  __syncthreads();
  const int base = cached_lens != nullptr ? cached_lens[r] : 0;
  for (int i = warp; i < n; i += kTreeThreads / 32) {
    uint32_t bits = 0;
    int depth = -1;
    // a node behind the staged ones (reported above) has itself alone
    for (int j = i; j >= 0; j = j < staged ? up[j] : -1) {
      if (lane == j >> 5) bits |= 1u << (j & 31);
      ++depth;
    }
    if (lane < words) mask[(int64_t)(start + i) * words + lane] = (int32_t)bits;
    if (lane == 0) positions[start + i] = base + depth;
  }
}

// ---- verification ----------------------------------------------------------------------------
constexpr int kVerifyThreads = 512;
constexpr int kVerifyWarps = kVerifyThreads / 32;
constexpr int kMaxRanks = 8;

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
};

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float load_logit(const __nv_bfloat16* p) { return bf16_to_f(*p); }
__device__ __forceinline__ float load_logit(const float* p) { return *p; }

__device__ __forceinline__ double warp_sum_f64(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// A cluster per request walks its tree from the root. The vocabulary is cut into one run of ids per
// warp of the cluster, in ascending order: a pass over a row leaves each warp the sum of its run, each
// CTA the sum of its warps', and a token is found by these sums from the outside in. Sums are taken in
// a fixed order, in fp64: an accepted or drawn token hangs on comparisons of them.
template <typename T, bool GREEDY, bool PROBS>
__global__ void __launch_bounds__(kVerifyThreads) verify_kernel(const VerifyArgs a) {
  __shared__ int32_t path[AIOSB_TREE_MAX_NODES];
  __shared__ uint32_t on_path[AIOSB_TREE_MAX_NODES / 32];
  __shared__ int64_t rejected[AIOSB_TREE_MAX_NODES];  // without draft_probs: tokens that left r at this node
  __shared__ double scale_by[AIOSB_TREE_MAX_NODES];   // with: 1 / sum(r) before each subtraction of q
  __shared__ double run_sum[kVerifyWarps];
  __shared__ float run_max[kVerifyWarps];
  __shared__ int run_arg[kVerifyWarps];
  __shared__ double peer_sum[2][kMaxRanks];
  __shared__ float peer_max[2][kMaxRanks];
  __shared__ int peer_arg[2][kMaxRanks];
  __shared__ int next_child;

  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int ranks = a.ranks, rank = (int)cluster_ctarank(), r = blockIdx.x / ranks;
  pdl_enter();

  const int s0 = a.tree_start[r], e0 = a.tree_start[r + 1];
  const int start = min(max(s0, 0), a.tokens), all = min(max(e0, start), a.tokens) - start;
  const int n = min(all, AIOSB_TREE_MAX_NODES);
  const bool first = rank == 0 && threadIdx.x == 0;
  if (first && (s0 < 0 || e0 < s0 || e0 > a.tokens || all > n)) report(a.status, AIOSB_DEV_TREE_RANGE);
  if (n == 0) {  // the whole cluster leaves
    if (first) {
      a.accepted[r] = 0;
      a.next_token[r] = -1;
    }
    return;
  }
  const int32_t* const parents = a.parents + start;
  const int run = (a.vocab + ranks * kVerifyWarps - 1) / (ranks * kVerifyWarps);
  const int lo = min((rank * kVerifyWarps + warp) * run, a.vocab), hi = min(lo + run, a.vocab);

  int turn = 0;
  // Every CTA's value to every CTA; the buffers take turns, so that one barrier per exchange is enough:
  // a CTA writes a buffer again only behind the next barrier, which all have reached after reading it.
  auto exchange_max = [&](float v, int arg) {
    if (threadIdx.x < ranks) {
      const uint32_t m = map_shared_rank(smem_u32(&peer_max[turn][rank]), threadIdx.x);
      const uint32_t g = map_shared_rank(smem_u32(&peer_arg[turn][rank]), threadIdx.x);
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(m), "f"(v) : "memory");
      asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(g), "r"(arg) : "memory");
    }
    cluster_sync();
  };
  // Sums each warp's `mine` within the CTA (in run_sum) and exchanges the CTAs' sums; the total.
  auto exchange_sum = [&](double mine) {
    mine = warp_sum_f64(mine);
    __syncthreads();
    if (lane == 0) run_sum[warp] = mine;
    __syncthreads();
    if (threadIdx.x < ranks) {
      double v = 0;
      for (int w = 0; w < kVerifyWarps; ++w) v += run_sum[w];
      const uint32_t p = map_shared_rank(smem_u32(&peer_sum[turn][rank]), threadIdx.x);
      asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(p), "d"(v) : "memory");
    }
    cluster_sync();
    double total = 0;
    for (int c = 0; c < ranks; ++c) total += peer_sum[turn][c];
    turn ^= 1;
    return total;
  };

  int cur = 0, depth = 0;
  int64_t token = -1;   // valid in the CTA (and by all of its threads) that writes it
  bool writes = false;
  if (threadIdx.x < AIOSB_TREE_MAX_NODES / 32) on_path[threadIdx.x] = threadIdx.x == 0 ? 1u : 0u;
  if (threadIdx.x == 0) path[0] = 0;
  cluster_sync();  // every CTA runs: its shared memory may be written

  for (;;) {
    const T* const row = reinterpret_cast<const T*>(a.logits) + (int64_t)(start + cur) * a.logits_stride;
    const float* const q = PROBS ? a.probs + (int64_t)(start + cur) * a.probs_stride : nullptr;
    // ---- the row's maximum (and where it is first)
    float top = -INFINITY;
    int arg = INT32_MAX;
    for (int v = lo + lane; v < hi; v += 32) {
      const float x = load_logit(row + v);
      if (GREEDY && x > top) arg = v;
      top = max_nan(top, x);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float x = __shfl_xor_sync(0xffffffffu, top, o);
      const int b = __shfl_xor_sync(0xffffffffu, arg, o);
      if (GREEDY) arg = x > top ? b : x == top ? min(arg, b) : arg;
      top = max_nan(top, x);
    }
    __syncthreads();
    if (lane == 0) {
      run_max[warp] = top;
      run_arg[warp] = arg;
    }
    __syncthreads();
    top = run_max[0];
    arg = run_arg[0];
    for (int w = 1; w < kVerifyWarps; ++w) {
      if (run_max[w] > top) arg = run_arg[w];
      top = max_nan(top, run_max[w]);
    }
    exchange_max(top, arg);
    top = peer_max[turn][0];
    arg = peer_arg[turn][0];
    for (int c = 1; c < ranks; ++c) {
      if (peer_max[turn][c] > top) arg = peer_arg[turn][c];
      top = max_nan(top, peer_max[turn][c]);
    }
    turn ^= 1;
    if (!(top > -INFINITY) || (!GREEDY && top == INFINITY)) {  // NaN, -inf only, or +inf
      if (first) report(a.status, AIOSB_DEV_NO_DISTRIBUTION);
      writes = rank == 0;
      break;
    }

    // ---- r(v) as it stands: p(v) behind the subtractions so far
    double inv_z = 1;
    int cuts = 0;  // entries of scale_by or rejected
    auto weight = [&](int v) {
      double x = exp((double)(load_logit(row + v) - top) * a.inv_temperature) * inv_z;
      if (PROBS) {
        const double qv = cuts > 0 ? (double)q[v] : 0.0;
        for (int i = 0; i < cuts; ++i) x = fmax(x * scale_by[i] - qv, 0.0);
      } else {
        for (int i = 0; i < cuts; ++i)
          if (rejected[i] == v) x = 0;
      }
      return x;
    };
    auto sum_run = [&]() {
      double part = 0;
      for (int v = lo + lane; v < hi; v += 32) part += weight(v);
      return part;
    };
    double total = 1;
    if (!GREEDY) {
      const double z = exchange_sum(sum_run());
      inv_z = 1.0 / z;
    }

    // ---- its children, in ascending order
    int found = -1, child = cur;
    while (found < 0) {
      __syncthreads();
      if (warp == 0) {
        int c = INT32_MAX;
        for (int j = child + 1 + lane; j - lane < n; j += 32) {
          const unsigned hit = __ballot_sync(0xffffffffu, j < n && parents[j] == cur);
          if (hit) {
            c = j - lane + __ffs(hit) - 1;
            break;
          }
        }
        if (lane == 0) next_child = c;
      }
      __syncthreads();
      child = next_child;
      if (child >= n) break;
      const int64_t x = a.draft_tokens[start + child];
      if (x < 0 || x >= a.vocab) {
        if (first) report(a.status, AIOSB_DEV_TOKEN_RANGE);
        continue;
      }
      if (GREEDY) {
        if (x == arg) found = child;
        continue;
      }
      const double rx = weight((int)x), qx = PROBS ? (double)q[x] : 1.0;
      if ((double)a.accept_u[start + child] * qx * total < rx) {
        found = child;
      } else if (PROBS) {
        __syncthreads();
        if (threadIdx.x == 0) scale_by[cuts] = 1.0 / total;
        __syncthreads();
        ++cuts;
        const double left = exchange_sum(sum_run());
        if (left > 0) total = left;
        else --cuts;
      } else {
        __syncthreads();
        if (threadIdx.x == 0) rejected[cuts] = x;
        __syncthreads();
        if (rx > 0) {
          ++cuts;
          total -= rx;
        }
      }
    }
    if (found >= 0) {
      cur = found;
      ++depth;
      if (threadIdx.x == 0) {
        path[depth] = cur;
        on_path[cur >> 5] |= 1u << (cur & 31);
      }
      continue;
    }

    // ---- the next token
    if (GREEDY) {
      token = arg;
      writes = rank == 0;
      break;
    }
    total = exchange_sum(sum_run());  // in the order of the search below
    const double target = (double)a.sample_u[r] * total;
    double before = 0;
    int owner = -1;
    double owner_before = 0;
    for (int c = 0; c < ranks; ++c) {
      const double w = peer_sum[turn ^ 1][c];
      if (w > 0) {
        owner = c;
        owner_before = before;
        if (before + w > target) break;
      }
      before += w;
    }
    writes = owner == rank;
    if (writes) {
      before = owner_before;
      int own_warp = -1;
      double warp_before = before;
      for (int w = 0; w < kVerifyWarps; ++w) {
        if (run_sum[w] > 0) {
          own_warp = w;
          warp_before = before;
          if (before + run_sum[w] > target) break;
        }
        before += run_sum[w];
      }
      if (warp == own_warp) {
        before = warp_before;
        int pick = -1;
        for (int v0 = lo; v0 < hi; v0 += 32) {
          const double x = v0 + lane < hi ? weight(v0 + lane) : 0.0;
          double c = x;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const double y = __shfl_up_sync(0xffffffffu, c, o);
            if (lane >= o) c += y;
          }
          const unsigned some = __ballot_sync(0xffffffffu, x > 0);
          const unsigned past = __ballot_sync(0xffffffffu, x > 0 && before + c > target);
          if (past) {
            pick = v0 + __ffs(past) - 1;
            break;
          }
          if (some) pick = v0 + 31 - __clz(some);  // the last one, should rounding leave the target past it
          before += __shfl_sync(0xffffffffu, c, 31);
        }
        if (lane == 0) a.next_token[r] = pick;
      }
    }
    token = -2;  // written above
    break;
  }

  __syncthreads();
  if (writes && token != -2 && threadIdx.x == 0) a.next_token[r] = token;
  if (rank != 0) return;
  if (threadIdx.x == 0) a.accepted[r] = depth;
  if (warp == 0) {
    int32_t* const order = a.order + start;
    for (int i = lane; i <= depth; i += 32) order[i] = path[i];
    int at = depth + 1;
    for (int j0 = 0; j0 < all; j0 += 32) {
      const int j = j0 + lane;
      const bool rest = j < all && !(j < n && ((on_path[j >> 5] >> (j & 31)) & 1));
      const unsigned some = __ballot_sync(0xffffffffu, rest);
      if (rest) order[at + __popc(some & ((1u << lane) - 1))] = j;
      at += __popc(some);
    }
  }
}

template <typename T, bool GREEDY, bool PROBS>
cudaError_t launch_verify(const VerifyArgs& a, int requests, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(requests * a.ranks));
  cfg.blockDim = dim3(kVerifyThreads);
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
  return cudaLaunchKernelEx(&cfg, verify_kernel<T, GREEDY, PROBS>, a);
}

template <typename T>
cudaError_t launch_verify(const VerifyArgs& a, int requests, bool greedy, cudaStream_t stream) {
  if (greedy) return launch_verify<T, true, false>(a, requests, stream);
  if (a.probs != nullptr) return launch_verify<T, false, true>(a, requests, stream);
  return launch_verify<T, false, false>(a, requests, stream);
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
  return check_launch("draft_tree", launch_pdl(draft_tree_kernel, dim3((unsigned)requests), dim3(kTreeThreads), 0,
                                               as_stream(stream), parents, tree_start, (int)tokens, (int)words,
                                               cached_lens, mask, positions, status));
}

extern "C" int aiosb_verify_draft(const void* logits, int logits_fp32, int64_t logits_stride, int64_t tokens,
                                  int64_t vocab, const int64_t* draft_tokens, const int32_t* parents,
                                  const int32_t* tree_start, int64_t requests, const float* accept_uniforms,
                                  const float* sample_uniforms, double temperature, int greedy,
                                  const float* draft_probs, int64_t probs_stride, int32_t* accepted,
                                  int64_t* next_token, int32_t* order, int32_t* status, void* stream) {
  AIOSB_REQUIRE(tokens >= 0 && requests >= 0 && vocab >= 1 && tokens <= INT32_MAX && requests <= INT32_MAX / kMaxRanks,
                AIOSB_ERR_INVALID_ARG, "verify_draft: bad sizes");
  AIOSB_REQUIRE(vocab <= (1 << 30), AIOSB_ERR_UNSUPPORTED, "verify_draft: vocabulary too large");
  AIOSB_REQUIRE(logits_stride >= vocab || tokens <= 1, AIOSB_ERR_INVALID_ARG,
                "verify_draft: logits row stride below the vocabulary");
  AIOSB_REQUIRE(greedy || (temperature > 0 && 1.0 / temperature > 0 && 1.0 / temperature < 1e30),
                AIOSB_ERR_INVALID_ARG, "verify_draft: the temperature must be positive");
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
  a.ranks = kMaxRanks;
  cudaStream_t s = as_stream(stream);
  return check_launch("verify_draft", logits_fp32 ? launch_verify<float>(a, (int)requests, greedy != 0, s)
                                                  : launch_verify<__nv_bfloat16>(a, (int)requests, greedy != 0, s));
}
