// Shared by the kernels of drafted token trees: the requests' trees and the attention's arguments.
//
// Tree of request r: rows tree_start[r] .. tree_start[r + 1] of the flat token arrays. Its keys are
// the `cached` tokens of its page-table row, which every node sees, and one key per node behind
// them (page-table entry cached + j is node j's slot), which node i sees if bit j of its mask is set.
#pragma once

#include "abi_util.h"
#include "common.cuh"

namespace aiosb {

struct TreeAttnArgs {
  const __nv_bfloat16* q;  // [tokens, q_stride], heads of a token side by side
  int64_t q_stride;
  const __nv_bfloat16* k_cache;  // [num_slots, hkv, d]
  const __nv_bfloat16* v_cache;
  int64_t num_slots;
  const int32_t* page_table;  // [table_rows, table_stride], table_width entries each
  int64_t table_stride;
  int table_rows, table_width;
  const int32_t* row_table;    // [requests]
  const int32_t* cached_lens;  // [requests]
  const int32_t* tree_start;   // [requests + 1]
  const int32_t* mask;         // [tokens, words]
  int words;
  int requests, tokens;
  int hq, hkv, group;
  float scale_log2;  // scale * log2(e): exponents are taken to base 2
  __nv_bfloat16* out;
  int64_t out_stride;
  void* work;
  int32_t* status;
};

struct TreeRequest {
  int start, nodes;  // rows of the flat token arrays
  int cached, keys;  // keys [0, cached) are history, [cached, keys) the tree's
  int64_t table;  // of its page-table row, in entries
};

// Request r with its numbers held inside the arrays; `tell`: report what had to be cut.
__device__ __forceinline__ TreeRequest tree_request(const TreeAttnArgs& a, int r, bool tell) {
  TreeRequest t;
  const int s = a.tree_start[r], e = a.tree_start[r + 1], c = a.cached_lens[r], row = a.row_table[r];
  t.start = min(max(s, 0), a.tokens);
  const int nodes = min(max(e, t.start), a.tokens) - t.start;
  t.nodes = min(nodes, 32 * a.words);
  const bool row_ok = row >= 0 && row < a.table_rows;
  t.cached = row_ok ? min(max(c, 0), a.table_width) : 0;
  t.keys = row_ok ? t.cached + min(t.nodes, a.table_width - t.cached) : 0;
  t.table = (row_ok ? row : 0) * a.table_stride;
  if (tell && (s < 0 || e < s || e > a.tokens || t.nodes != nodes ||
               (nodes > 0 && (t.cached != c || t.keys - t.cached != t.nodes))))
    report(a.status, AIOSB_DEV_TREE_RANGE);
  return t;
}

__device__ __forceinline__ int64_t tree_slot(const TreeAttnArgs& a, int32_t slot) {
  if (slot >= 0 && slot < a.num_slots) return slot;
  report(a.status, AIOSB_DEV_SLOT_RANGE);
  return 0;
}

// 2^x to fp32, x <= 0 or so: one special-function instruction, off by 2^-22.
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two weights as bf16, cut off, and what is left of them as bf16 again: both halves go through the second product, as in
// the prefill attention. The rest is below 2^-7 of a weight and rounded by 2^-8 of itself, so that the weights of the
// product are off by 2^-15 of each at most, where one bf16 would be off by 2^-8. A rest of a weight above 0 is above 0 as
// well (the factor's 2^-20 of the weight): beside an infinite value a product with 0, or a negative one, would be NaN.
__device__ __forceinline__ void split_bf16x2(float2 x, uint32_t& upper, uint32_t& lower) {
  constexpr float c = 1.f + 0x1p-20f;
  upper = __byte_perm(__float_as_uint(x.x), __float_as_uint(x.y), 0x7632);
  lower = pack_bf16x2(fmaf(x.x, c, -bf16_lo(upper)), fmaf(x.y, c, -bf16_hi(upper)));
}

__device__ __forceinline__ bool finite_bf16x2(uint32_t v) {
  return (v & 0x7F800000u) != 0x7F800000u && (v & 0x7F80u) != 0x7F80u;
}
__device__ __forceinline__ uint32_t drop_nonfinite_bf16x2(uint32_t v) {
  if ((v & 0x7F800000u) == 0x7F800000u) v &= 0x0000FFFFu;
  if ((v & 0x7F80u) == 0x7F80u) v &= 0xFFFF0000u;
  return v;
}

// mma.sync m16n8k16 and the loads of its operands
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

// attn_tree_split.cu: the keys of all requests dealt over `grid` CTAs.
int tree_split_grid();
int tree_split_unit_rows(int64_t max_rows);
int64_t tree_split_work_bytes(int grid, int unit_rows, int d);
cudaError_t launch_tree_split(const TreeAttnArgs& a, int d, int grid, int unit_rows, cudaStream_t stream);

}  // namespace aiosb
