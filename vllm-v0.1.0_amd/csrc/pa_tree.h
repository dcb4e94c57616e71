// What the three files of the paged attention with several queries per sequence
// share: the arguments of its kernels, and the launches by element type.
#pragma once

#include "pa_common.h"

namespace pa {

struct TreeArgs {
  void* out;                // [num_tokens, num_heads, head_size]
  const void* q;
  const char* kc;
  const char* vc;
  const int32_t* tables;
  const int32_t* ctx;
  const int32_t* starts;    // [num_seqs + 1]
  const uint8_t* mask;      // [num_tokens, >= max_query] truth values, or null: a chain
  float* weights;           // [num_blocks, num_kv_heads, block_size], or null
  float* ml;                // per (sequence, kv head, partition, row): maximum, sum, sum before rounding, unused
  float* acc;               // per (sequence, kv head, partition, row): head_size sums
  float* logits;            // per (sequence, kv head, row): logit_stride logits, base 2
  int64_t q_stride, mask_stride, logit_stride;
  float c;                  // |scale| * log2(e); 1 where the scale is 0
  int q_mode;               // 0: q as stored, 1: -q (scale < 0), 2: q = 0 (scale == 0)
  int num_seqs, num_tokens, num_heads, num_kv_heads, group;
  int num_blocks, block_bits, table_width;
  int max_ctx, max_query, max_rows;
  int parts, part_len;      // context partitions of part_len positions
  int row_tiles;            // workgroups along a sequence's rows
};

// What a launch does with one sequence, the same for every kernel that asks.
struct TreeSeq {
  int first, queries, rows, ctx, parts;
  bool bad;  // the arguments contradict each other: its rows are filled with NaN
};

__device__ __forceinline__ TreeSeq tree_seq(const TreeArgs& a, int s) {
  TreeSeq r;
  const int lo = a.starts[s], hi = a.starts[s + 1];
  r.first = lo < 0 ? 0 : (lo > a.num_tokens ? a.num_tokens : lo);
  const int end = hi > a.num_tokens ? a.num_tokens : hi;
  r.queries = end > r.first ? end - r.first : 0;
  r.ctx = a.ctx[s];
  r.bad = lo < 0 || hi > a.num_tokens || hi < lo || r.queries > a.max_query || r.ctx < r.queries || r.ctx > a.max_ctx ||
          r.ctx > ((int64_t)a.table_width << a.block_bits);
  r.rows = r.queries * a.group;
  const int p = (r.ctx + a.part_len - 1) / a.part_len;
  r.parts = p < 1 ? 1 : (p < a.parts ? p : a.parts);
  return r;
}

__device__ __forceinline__ int64_t tree_row(const TreeArgs& a, int s, int head, int part, int row) {
  return (((int64_t)s * a.num_kv_heads + head) * a.parts + part) * a.max_rows + row;
}

// The kernel for a launch of at most `rows` rows a sequence and kv head, by the rows of a workgroup.
enum TreeForm { kTreeFew16 = 16, kTreeFew32 = 32, kTreeMany64 = 64, kTreeMany128 = 128, kTreeMany256 = 256 };
inline TreeForm tree_form(int64_t rows) {
  if (rows <= 16) return kTreeFew16;
  if (rows <= 32) return kTreeFew32;
  if (rows <= 64) return kTreeMany64;
  if (rows <= 128) return kTreeMany128;
  return kTreeMany256;
}

// pa_tree_f16.hip, pa_tree_bf16.hip, pa_tree_f32.hip
int tree_launch_f16(const TreeArgs& a, int head_size, unsigned grid, hipStream_t st);
int tree_launch_bf16(const TreeArgs& a, int head_size, unsigned grid, hipStream_t st);
int tree_launch_f32(const TreeArgs& a, int head_size, unsigned grid, hipStream_t st);

}  // namespace pa
