// What the three files of the paged attention with several queries per sequence
// share: the arguments of its kernels, and the launches by element type.
#pragma once

#include "pa_common.h"

namespace pa {

constexpr int kPartTokens = 128;  // a context partition is a multiple of this: a step for each of 4 waves
constexpr int kTreeSorted = 256;  // at most so many sequences are put in order by a workgroup: one to a thread

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
  int parts, part_len;      // at most so many context partitions, of at most part_len positions
  int row_tiles;            // workgroups along a sequence's rows
  int form;                 // TreeForm
  bool sorted;              // whether sequences are taken by falling length of their partitions
};

// What a launch does with one sequence, the same for every kernel that asks.
struct TreeSeq {
  int first, queries, rows, ctx, parts, part_len;
  bool bad;  // the arguments contradict each other: its rows are filled with NaN
};

// As few partitions as part_len allows, of one length: a last one of any length would leave others waiting.
__device__ __forceinline__ int tree_part_len(const TreeArgs& a, int ctx) {
  const int p = (int)(((int64_t)ctx + a.part_len - 1) / a.part_len);
  return (int)(((int64_t)ctx + p - 1) / p + kPartTokens - 1) / kPartTokens * kPartTokens;
}

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
  const int ctx = r.bad || r.ctx < 1 ? 1 : r.ctx;
  r.part_len = tree_part_len(a, ctx);
  r.parts = (ctx + r.part_len - 1) / r.part_len;
  return r;
}

__device__ __forceinline__ int64_t tree_row(const TreeArgs& a, int s, int head, int part, int row) {
  return (((int64_t)s * a.num_kv_heads + head) * a.parts + part) * a.max_rows + row;
}

// Whether a workgroup of tile_rows rows has a sequence's logits to itself
__device__ __forceinline__ bool tree_whole(const TreeSeq& sq, int tile_rows) { return sq.parts == 1 && sq.rows <= tile_rows; }

// Four positions' weights into the weight cache: added, but the new tokens' own start from 0
__device__ __forceinline__ void add_weights(const TreeArgs& a, const TreeSeq& sq, int seq, int head, int pos, f32x4 w) {
  const int block = a.tables[(int64_t)seq * a.table_width + (pos >> a.block_bits)];
  if ((unsigned)block >= (unsigned)a.num_blocks) return;
  // four positions of one block: block sizes are multiples of 8
  float* to = a.weights + (((int64_t)block * a.num_kv_heads + head) << a.block_bits) + (pos & ((1 << a.block_bits) - 1));
  const f32x4 old = *reinterpret_cast<const f32x4*>(to);
  const int fresh = sq.ctx - sq.queries;
#pragma unroll
  for (int i = 0; i < 4; i++) w[i] = pos + i >= sq.ctx ? old[i] : (pos + i >= fresh ? w[i] : old[i] + w[i]);
  *reinterpret_cast<f32x4*>(to) = w;
}

// LDS of the few-rows kernel: what joining its waves takes and, where logits are kept, the rows of a workgroup times
// a partition's length.  They may take 76 KiB, what two workgroups to a CU leave each other: a context that fits is
// weighed without a second kernel and without its logits' way through memory (96 sequences of up to 4096 tokens, 4
// rows, 182 us; with 48 KiB and parts of 1408 tokens 227, although three workgroups share a CU then).
constexpr int kTreeLogitFloats = 19456;
static_assert(4 * 16 * 2 * (128 + 4) <= kTreeLogitFloats, "joining the waves' largest shares takes no more than the logits may");
constexpr int tree_few_floats(int head_size, int row_tiles, int logit_rows, int part_len) {
  const int join = 4 * 16 * row_tiles * (head_size + 4), logits = logit_rows * (part_len + 4);
  return join > logits ? join : logits;
}

// The kernel for a launch of at most `rows` rows a sequence and kv head, by the rows of a workgroup.
enum TreeForm { kTreeFew16 = 16, kTreeFew32 = 32, kTreeMany64 = 64, kTreeMany128 = 128 };
inline TreeForm tree_form(int64_t rows, bool accumulate, bool fp32) {
  if (rows <= 16) return kTreeFew16;
  if (rows <= 32 || accumulate) return kTreeFew32;  // only the few-rows kernel keeps its logits
  if (rows <= 64 || fp32) return kTreeMany64;  // fp32 queries of two tiles a wave do not fit its registers
  return kTreeMany128;
}

// pa_tree_f16.hip, pa_tree_bf16.hip, pa_tree_f32.hip
int tree_launch_f16(const TreeArgs& a, int head_size, unsigned grid, hipStream_t st);
int tree_launch_bf16(const TreeArgs& a, int head_size, unsigned grid, hipStream_t st);
int tree_launch_f32(const TreeArgs& a, int head_size, unsigned grid, hipStream_t st);

}  // namespace pa
