// Attention of drafted token trees over a paged cache:
//   o[i] = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(scale q_i . k_j) over the keys that node i sees,
// its request's history and the nodes of its tree whose mask bit is set (0 if it sees none).
//
// All query heads of a KV head read the same keys, so the rows of a product are (node, query head of
// the group) pairs: row = node * group + head. One pass over the keys holds each row's maximum m and
// sum l; a chunk rescales the row's output by 2^(m_old - m_new).
#include <algorithm>

#include "tree.cuh"

namespace aiosb {
namespace {

constexpr int kRows = 64;   // rows of a CTA: 16 to a warp
constexpr int kChunk = 64;  // keys of a chunk
constexpr int kThreads = 128;

template <int D>
constexpr int kPitch = D + 8;  // elements of a staged row: 16 more bytes keep ldmatrix free of bank conflicts
template <int D>
constexpr size_t kSmallSmem = 2 * 2 * (size_t)kChunk * kPitch<D> * 2;  // K and V, two chunks each

// Whole requests: a CTA takes 64 rows of one KV head through all of their keys, on mma.sync from two staged chunks in
// turn: with few keys there is nothing to deal out, and a TMEM round trip is longer than a chunk's products. Bound by
// launch and two dependent loads (slots, then keys): 1 request, 32 + 8 keys, 8 nodes, 12/4 heads of 64 in 5.7 us.
template <int D>
__global__ void __launch_bounds__(kThreads) attn_tree_small_kernel(const TreeAttnArgs a) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  __nv_bfloat16* const stage = reinterpret_cast<__nv_bfloat16*>(smem_raw);
  __shared__ uint32_t bad[2];  // keys of the chunk whose V holds an infinity or a NaN
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int h = blockIdx.y, r = blockIdx.z;

  pdl_enter();
  const TreeRequest t = tree_request(a, r, blockIdx.x == 0 && h == 0 && threadIdx.x == 0);
  const int rows = t.nodes * a.group, row0 = blockIdx.x * kRows;
  if (row0 >= rows) return;

  // this lane's two rows: row0 + 16 warp + lane / 4 and the one 8 below it
  const int my_row[2] = {row0 + warp * 16 + lane / 4, row0 + warp * 16 + lane / 4 + 8};
  const bool works = row0 + warp * 16 < rows;
  const int32_t* bits[2];
  uint32_t qf[D / 16][4];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int row = min(my_row[i], rows - 1);
    const int node = t.start + row / a.group, head = h * a.group + row % a.group;
    bits[i] = a.mask + (int64_t)node * a.words;
    const uint32_t* src = reinterpret_cast<const uint32_t*>(a.q + node * a.q_stride + (int64_t)head * D) + lane % 4;
#pragma unroll
    for (int k = 0; k < D / 16; ++k) {
      qf[k][i] = src[k * 8];
      qf[k][2 + i] = src[k * 8 + 4];
    }
  }

  auto load_chunk = [&](int k0, int buf) {
    __nv_bfloat16* const ks = stage + buf * 2 * kChunk * kPitch<D>;
    __nv_bfloat16* const vs = ks + kChunk * kPitch<D>;
    for (int i = threadIdx.x; i < kChunk * (D / 8); i += kThreads) {
      const int j = i / (D / 8), c = i % (D / 8);
      if (k0 + j < t.keys) {
        const int64_t at = (tree_slot(a, a.page_table[t.table + k0 + j]) * a.hkv + h) * D + c * 8;
        cp_async16(ks + j * kPitch<D> + c * 8, a.k_cache + at);
        cp_async16(vs + j * kPitch<D> + c * 8, a.v_cache + at);
      } else {  // weights of keys past the end are 0, and 0 times what lies there must be 0
        *reinterpret_cast<uint4*>(vs + j * kPitch<D> + c * 8) = make_uint4(0, 0, 0, 0);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };

  float o[D / 8][4];
#pragma unroll
  for (int n = 0; n < D / 8; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[n][e] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

  load_chunk(0, 0);
  for (int k0 = 0, buf = 0; k0 < t.keys; k0 += kChunk, buf ^= 1) {
    if (k0 + kChunk < t.keys) {
      load_chunk(k0 + kChunk, buf ^ 1);
      asm volatile("cp.async.wait_group 1;" ::: "memory");
    } else {
      asm volatile("cp.async.wait_group 0;" ::: "memory");
    }
    const bool tree = k0 + kChunk > t.cached;  // the chunk has keys that some node does not see
    if (tree && threadIdx.x < 2) bad[threadIdx.x] = 0;
    __syncthreads();
    __nv_bfloat16* const ks = stage + buf * 2 * kChunk * kPitch<D>;
    __nv_bfloat16* const vs = ks + kChunk * kPitch<D>;
    if (tree) {
      // A key that a node does not see gets weight 0, and 0 * inf is NaN: infinities and NaN leave V
      // before the product, and the nodes that do see them get them below.
      for (int i = threadIdx.x; i < kChunk * (D / 8); i += kThreads) {
        uint4* const p = reinterpret_cast<uint4*>(vs + i / (D / 8) * kPitch<D> + i % (D / 8) * 8);
        uint4 v = *p;
        if (!(finite_bf16x2(v.x) && finite_bf16x2(v.y) && finite_bf16x2(v.z) && finite_bf16x2(v.w))) {
          *p = make_uint4(drop_nonfinite_bf16x2(v.x), drop_nonfinite_bf16x2(v.y), drop_nonfinite_bf16x2(v.z),
                          drop_nonfinite_bf16x2(v.w));
          const int j = i / (D / 8);
          atomicOr(&bad[j / 32], 1u << (j % 32));
        }
      }
      __syncthreads();
    }
    if (works) {
      float s[kChunk / 8][4];
#pragma unroll
      for (int n = 0; n < kChunk / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[n][e] = 0.f;
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
#pragma unroll
        for (int n = 0; n < kChunk / 16; ++n) {
          uint32_t b[4];
          ldmatrix4(b, smem_u32(ks + (n * 16 + (lane & 7) + (lane & 16 ? 8 : 0)) * kPitch<D> + k * 16 +
                                (lane & 8 ? 8 : 0)));
          mma_16816(s[2 * n], qf[k], b[0], b[1]);
          mma_16816(s[2 * n + 1], qf[k], b[2], b[3]);
        }
      }
      float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int n = 0; n < kChunk / 8; ++n) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float v = s[n][e] * a.scale_log2;
          if (tree) {
            const int key = k0 + n * 8 + (lane & 3) * 2 + (e & 1), j = key - t.cached;
            const bool seen = key < t.keys && (j < 0 || (((uint32_t)bits[e >> 1][j >> 5] >> (j & 31)) & 1));
            if (!seen) v = -INFINITY;
          }
          s[n][e] = v;
          top[e >> 1] = fmaxf(top[e >> 1], v);  // a NaN reaches the result through the sum
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 1));
        top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 2));
        const float m_new = fmaxf(m[i], top[i]);
        // nothing seen yet: any finite reference will do
        const float ref = m_new == -INFINITY ? 0.f : m_new;
        const float corr = exp2_fast(m[i] - ref);
        m[i] = m_new;
        float sum = 0.f;
#pragma unroll
        for (int n = 0; n < kChunk / 8; ++n) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            s[n][2 * i + e] = exp2_fast(s[n][2 * i + e] - ref);
            sum += s[n][2 * i + e];
          }
        }
        l[i] = l[i] * corr + sum;
#pragma unroll
        for (int n = 0; n < D / 8; ++n) {
          o[n][2 * i] *= corr;
          o[n][2 * i + 1] *= corr;
        }
      }
#pragma unroll
      for (int k = 0; k < kChunk / 16; ++k) {
        uint32_t p[2][4];  // the weights as the A operand, upper and lower halves
#pragma unroll
        for (int i = 0; i < 4; ++i)
          split_bf16x2(make_float2(s[2 * k + i / 2][i % 2 * 2], s[2 * k + i / 2][i % 2 * 2 + 1]), p[0][i], p[1][i]);
#pragma unroll
        for (int n = 0; n < D / 16; ++n) {
          uint32_t b[4];
          ldmatrix4_trans(b, smem_u32(vs + (k * 16 + (lane & 15)) * kPitch<D> + n * 16 + (lane & 16 ? 8 : 0)));
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            mma_16816(o[2 * n], p[i], b[0], b[1]);
            mma_16816(o[2 * n + 1], p[i], b[2], b[3]);
          }
        }
      }
      if (tree && (bad[0] | bad[1])) {
#pragma unroll 1
        for (int j = 0; j < kChunk; ++j) {
          if (!((bad[j / 32] >> (j % 32)) & 1)) continue;
          const int key = k0 + j, b = key - t.cached;
          const __nv_bfloat16* v = a.v_cache + (tree_slot(a, a.page_table[t.table + key]) * a.hkv + h) * D;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            if (b >= 0 && !(((uint32_t)bits[i][b >> 5] >> (b & 31)) & 1)) continue;
#pragma unroll
            for (int n = 0; n < D / 8; ++n) {
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const float x = bf16_to_f(v[n * 8 + (lane & 3) * 2 + e]);
                if (!(fabsf(x) < INFINITY)) o[n][2 * i + e] += x;
              }
            }
          }
        }
      }
    }
    __syncthreads();
  }

#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float sum = l[i] + __shfl_xor_sync(0xffffffffu, l[i], 1);
    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
    if (my_row[i] >= rows) continue;
    const float inv = m[i] == -INFINITY && sum == 0.f ? 0.f : 1.f / sum;
    uint32_t* dst = reinterpret_cast<uint32_t*>(a.out + (int64_t)(t.start + my_row[i] / a.group) * a.out_stride +
                                                (int64_t)(h * a.group + my_row[i] % a.group) * D) +
                    lane % 4;
#pragma unroll
    for (int n = 0; n < D / 8; ++n) dst[n * 4] = pack_bf16x2(o[n][2 * i] * inv, o[n][2 * i + 1] * inv);
  }
}

template <int D>
cudaError_t launch_small(const TreeAttnArgs& a, int64_t max_nodes, cudaStream_t stream) {
  const auto kernel = attn_tree_small_kernel<D>;
  static bool configured[64] = {false};
  cudaError_t e = allow_shared(kernel, (int)kSmallSmem<D>, configured);
  if (e != cudaSuccess) return e;
  const dim3 grid((unsigned)((max_nodes * a.group + kRows - 1) / kRows), (unsigned)a.hkv, (unsigned)a.requests);
  return launch_pdl(kernel, grid, dim3(kThreads), kSmallSmem<D>, stream, a);
}

// Whether the keys are dealt over the SMs (attn_tree_split.cu): for longer histories, or many rows, which its tensor
// cores take faster. Measured, whole / dealt, us: 16 requests of 26 nodes, 8/2 heads of 96: 64 keys 10.9 / 13.5, 128
// 14.6 / 14.9, 256 20.8 / 16.9, 1024 60 / 19.5; 1 of 5 nodes, 32/8 heads of 128: 64 11.7 / 11.5, 128 16.7 / 15.1. 64
// requests, 32 keys, thousands of rows, 8/2 heads of 96: 15.9 11.1 / 15.3, 20.5 16.1 / 18.7, 30.7 27.6 / 19.3; 12/4 of
// 64: 20.0 15.6 / 18.9, 23.8 15.7 / 19.1, 30.7 22.5 / 21.0; 32/8 of 128: 53 41.6 / 37.5, 123 126 / 50.
bool splits(int64_t max_cached, int64_t tokens, int64_t heads) { return max_cached > 128 || tokens * heads > 24000; }

}  // namespace
}  // namespace aiosb

using namespace aiosb;

extern "C" int64_t aiosb_attention_tree_work_bytes(int64_t tokens, int64_t requests, int64_t mask_words,
                                                   int64_t max_cached, int64_t num_qo_heads, int64_t num_kv_heads,
                                                   int64_t head_dim) {
  if (tokens <= 0 || requests <= 0 || num_kv_heads <= 0) return 0;
  if (max_cached > 0 && !splits(max_cached, tokens, num_qo_heads)) return 0;  // 0: the page table's width, any
  const int64_t rows = std::min(mask_words * 32, tokens) * (num_qo_heads / num_kv_heads);
  return tree_split_work_bytes(tree_split_grid(), tree_split_unit_rows(rows), (int)head_dim);
}

extern "C" int aiosb_attention_tree(const void* q, int64_t q_stride, int64_t tokens, const void* k_cache,
                                    const void* v_cache, int64_t num_slots, const int32_t* page_table,
                                    int64_t table_stride, int64_t table_rows, int64_t table_width,
                                    const int32_t* row_table, const int32_t* cached_lens, const int32_t* tree_start,
                                    int64_t requests, const int32_t* mask, int64_t mask_words, int64_t max_cached,
                                    int64_t num_qo_heads, int64_t num_kv_heads, int64_t head_dim, float scale,
                                    void* out, int64_t out_stride, void* work, int64_t work_bytes, int32_t* status,
                                    void* stream) {
  AIOSB_REQUIRE(num_kv_heads > 0 && num_qo_heads > 0 && num_qo_heads % num_kv_heads == 0, AIOSB_ERR_INVALID_ARG,
                "query head count must be divisible by KV head count");
  AIOSB_REQUIRE(head_dim == 64 || head_dim == 96 || head_dim == 128, AIOSB_ERR_UNSUPPORTED,
                "attention_tree: head_dim %lld unsupported (64, 96, 128)", (long long)head_dim);
  AIOSB_REQUIRE(tokens >= 0 && requests >= 0 && num_slots >= 0 && table_rows >= 0 && table_width >= 0 &&
                    max_cached >= 0 && work_bytes >= 0 && scale > 0 && scale < INFINITY,
                AIOSB_ERR_INVALID_ARG, "attention_tree: bad sizes");
  AIOSB_REQUIRE(mask_words >= 1 && mask_words <= AIOSB_TREE_MAX_NODES / 32, AIOSB_ERR_UNSUPPORTED,
                "attention_tree: %lld mask words; a tree has at most %d nodes", (long long)mask_words,
                AIOSB_TREE_MAX_NODES);
  const int64_t group = num_qo_heads / num_kv_heads;
  AIOSB_REQUIRE(group <= AIOSB_TREE_MAX_GROUP && num_kv_heads <= 65535 && requests <= 65535 &&
                    tokens * group <= INT32_MAX && table_width <= (1 << 30) && table_rows < INT32_MAX,
                AIOSB_ERR_UNSUPPORTED, "attention_tree: too many rows, heads or requests");
  AIOSB_REQUIRE(q_stride >= num_qo_heads * head_dim && out_stride >= num_qo_heads * head_dim && q_stride % 8 == 0 &&
                    out_stride % 8 == 0,
                AIOSB_ERR_INVALID_ARG, "attention_tree: q and out row strides must cover a row and be multiples of 8");
  AIOSB_REQUIRE(table_stride >= table_width, AIOSB_ERR_INVALID_ARG,
                "attention_tree: page-table stride below its width");
  if (tokens == 0 || requests == 0) return AIOSB_OK;
  AIOSB_REQUIRE(num_slots > 0 && table_rows > 0, AIOSB_ERR_INVALID_ARG, "attention_tree: empty cache or page table");
  AIOSB_REQUIRE(q && k_cache && v_cache && page_table && row_table && cached_lens && tree_start && mask && out,
                AIOSB_ERR_INVALID_ARG, "attention_tree: null pointer");
  AIOSB_REQUIRE(aligned16(q) && aligned16(k_cache) && aligned16(v_cache) && aligned16(out), AIOSB_ERR_MISALIGNED,
                "attention_tree: q, out and the KV cache must be 16-byte aligned");
  const bool split = splits(max_cached > 0 ? max_cached : table_width, tokens, num_qo_heads);
  const int64_t max_nodes = std::min<int64_t>(mask_words * 32, tokens);
  const int unit_rows = tree_split_unit_rows(max_nodes * group), grid = tree_split_grid();
  AIOSB_REQUIRE(!split || (work != nullptr && aligned16(work) &&
                           work_bytes >= tree_split_work_bytes(grid, unit_rows, (int)head_dim)),
                AIOSB_ERR_INVALID_ARG, "attention_tree: work area missing, misaligned or too small");
  TreeAttnArgs a;
  a.q = (const __nv_bfloat16*)q;
  a.q_stride = q_stride;
  a.k_cache = (const __nv_bfloat16*)k_cache;
  a.v_cache = (const __nv_bfloat16*)v_cache;
  a.num_slots = num_slots;
  a.page_table = page_table;
  a.table_stride = table_stride;
  a.table_rows = (int)table_rows;
  a.table_width = (int)table_width;
  a.row_table = row_table;
  a.cached_lens = cached_lens;
  a.tree_start = tree_start;
  a.mask = mask;
  a.words = (int)mask_words;
  a.requests = (int)requests;
  a.tokens = (int)tokens;
  a.hq = (int)num_qo_heads;
  a.hkv = (int)num_kv_heads;
  a.group = (int)group;
  a.scale_log2 = (float)(scale * 1.4426950408889634);
  a.out = (__nv_bfloat16*)out;
  a.out_stride = out_stride;
  a.work = work;
  a.status = status;
  cudaStream_t s = as_stream(stream);
  cudaError_t e;
  if (split) e = launch_tree_split(a, (int)head_dim, grid, unit_rows, s);
  else if (head_dim == 64) e = launch_small<64>(a, max_nodes, s);
  else if (head_dim == 96) e = launch_small<96>(a, max_nodes, s);
  else e = launch_small<128>(a, max_nodes, s);
  return check_launch("attention_tree", e);
}
