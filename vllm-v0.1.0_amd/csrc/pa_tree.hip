// Cached attention of several queries per sequence: the entry points, the launch
// plan, the kernel that joins context partitions and adds up the weight cache.
// The attention kernel itself is in pa_tree_kernel.h.
#include <math.h>

#include <algorithm>

#include "pa_tree.h"

namespace pa {
namespace {

// ---- joining partitions, and the weight cache -----------------------------------------------
//
// Workgroups below join_groups: head_size / 4 lanes to a row, out = sum_p 2^(m_p - m) acc_p / sum_p 2^(m_p - m) l_p.
// The others: 1024 positions of a (sequence, kv head) each, 4 to a lane, w(pos) += sum over rows
// 2^(logit - m) / l with l from before the weights' rounding; positions of the new tokens start from 0.
// Neither waits for the other: each makes the row statistics it needs from the partitions' own.
// Bound by the logits' read for long contexts (4 bytes a position and row next to the head's
// 512 of keys and values), by the launch for short ones.
// 2 sequences of 40009 tokens in 32 partitions, 48 rows a kv head: 7.3 us for 13 MB; one sequence: 4.
constexpr int kChunk = 1024;
constexpr int kStatRows = 256;

// A row and 4 of its elements.  One pass, all loads of four partitions on their way at once: the running
// maximum is raised as in the attention itself.
template <typename T>
__device__ __forceinline__ void join_row(const TreeArgs& a, int D, int64_t row_id, int d) {
  const int64_t per_seq = (int64_t)a.max_query * a.num_heads;
  const int seq = (int)(row_id / per_seq);
  const int rest = (int)(row_id - seq * per_seq);
  const int query = rest / a.num_heads, h = rest - query * a.num_heads;
  const TreeSeq sq = tree_seq(a, seq);
  if (sq.bad || query >= sq.queries || sq.parts == 1) return;  // one partition: the result is there
  const int head = h / a.group, row = query * a.group + (h - head * a.group);
  const int64_t first = tree_row(a, seq, head, 0, row);
  float high = -INFINITY, sum = 0.f;
  f32x4 x = {0, 0, 0, 0};
  for (int p = 0; p < sq.parts; p += 4) {
    float2 st[4];
    f32x4 v[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int64_t at = first + (int64_t)(p + i < sq.parts ? p + i : sq.parts - 1) * a.max_rows;
      st[i] = *reinterpret_cast<const float2*>(a.ml + at * 4);
      v[i] = *reinterpret_cast<const f32x4*>(a.acc + at * D + d);
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
      // a partition past the last is the last again, and weighs nothing; its sums may be infinite, which no weight of
      // 0 would take out
      const bool there = p + i < sq.parts;
      const float m = there ? st[i].x : -INFINITY;
      v[i] = there ? v[i] : f32x4{0, 0, 0, 0};
      const float top = fmaxf(high, m);
      const float was = __builtin_amdgcn_exp2f(high - top), is = __builtin_amdgcn_exp2f(m - top);
      high = top;
      sum = sum * was + st[i].y * is;
      x = x * was + v[i] * is;
    }
  }
  const float inv = sum == 0.f ? 0.f : 1.0f / sum;
  typedef T T4 __attribute__((ext_vector_type(4)));
  *reinterpret_cast<T4*>(static_cast<T*>(a.out) + ((int64_t)(sq.first + query) * a.num_heads + h) * D + d) =
      __builtin_convertvector(x * inv, T4);
}

template <typename T>
__global__ void __launch_bounds__(256) pa_tree_join_kernel(const TreeArgs a, const int D, const unsigned join_groups,
                                                           const int chunks, const int tile_rows) {
  if (blockIdx.x < join_groups) {
    const int lanes = D / 4, rows = 256 / lanes, r = (int)threadIdx.x / lanes;
    const int64_t row = (int64_t)blockIdx.x * rows + r;
    if (r < rows && row < (int64_t)a.num_seqs * a.max_query * a.num_heads) join_row<T>(a, D, row, ((int)threadIdx.x - r * lanes) * 4);
    return;
  }
  const unsigned id = blockIdx.x - join_groups;
  const int chunk = (int)(id % (unsigned)chunks);
  const int head = (int)(id / (unsigned)chunks % (unsigned)a.num_kv_heads);
  const int seq = (int)(id / (unsigned)chunks / (unsigned)a.num_kv_heads);
  const TreeSeq sq = tree_seq(a, seq);
  if (sq.bad || sq.rows == 0 || chunk * kChunk >= sq.ctx || tree_whole(sq, tile_rows)) return;
  __shared__ float sm_m[kStatRows], sm_inv[kStatRows];
  const int pos = chunk * kChunk + (int)threadIdx.x * 4;
  f32x4 w = {0, 0, 0, 0};
  const float* lg = a.logits + ((int64_t)seq * a.num_kv_heads + head) * a.max_rows * a.logit_stride + pos;
  for (int r0 = 0; r0 < sq.rows; r0 += kStatRows) {
    const int n = sq.rows - r0 < kStatRows ? sq.rows - r0 : kStatRows;
    __syncthreads();
    if ((int)threadIdx.x < n) {
      float high = -INFINITY, sum = 0.f;
      for (int p = 0; p < sq.parts; p++) high = fmaxf(high, a.ml[tree_row(a, seq, head, p, r0 + threadIdx.x) * 4]);
      for (int p = 0; p < sq.parts; p++) {
        const float* st = a.ml + tree_row(a, seq, head, p, r0 + threadIdx.x) * 4;
        sum = __builtin_fmaf(st[2], __builtin_amdgcn_exp2f(st[0] - high), sum);
      }
      sm_m[threadIdx.x] = high;
      sm_inv[threadIdx.x] = sum == 0.f ? 0.f : 1.0f / sum;
    }
    __syncthreads();
    if (pos < sq.ctx) {
#pragma unroll 4
      for (int r = 0; r < n; r++) {
        const f32x4 x = *reinterpret_cast<const f32x4*>(lg + (int64_t)(r0 + r) * a.logit_stride);
#pragma unroll
        for (int i = 0; i < 4; i++) w[i] = __builtin_fmaf(__builtin_amdgcn_exp2f(x[i] - sm_m[r]), sm_inv[r], w[i]);
      }
    }
  }
  if (pos < sq.ctx) add_weights(a, sq, seq, head, pos, w);
}

// ---- launch plan ---------------------------------------------------------------------------------

struct TreePlan {
  int parts, part_len, row_tiles, tile_rows;
  int64_t max_rows, logit_stride;
  size_t ml_bytes, acc_bytes, logit_bytes;
  size_t bytes() const { return ml_bytes + acc_bytes + logit_bytes; }
};

constexpr int kChipCUs = 256;
constexpr int kMaxParts = 64;
constexpr int kMinPart = 256;
constexpr int kMaxContext = 1 << 30;

TreePlan tree_plan(int num_seqs, int num_heads, int num_kv_heads, int head_size, int max_ctx, int max_query, bool accumulate,
                   bool fp32) {
  TreePlan p;
  p.max_rows = (int64_t)max_query * (num_heads / num_kv_heads);
  const int rows = tree_form(p.max_rows, accumulate, fp32);
  p.row_tiles = (int)std::max<int64_t>(1, (p.max_rows + rows - 1) / rows);
  const int64_t groups = std::max<int64_t>(1, (int64_t)num_seqs * num_kv_heads * p.row_tiles);
  // As many partitions as two workgroups to a CU allow: those are resident at once, and one more would wait for
  // them (8 sequences of up to 4096 tokens, trees of 64, 8 kv heads of 32: 55 us; for one workgroup to a CU 70,
  // for three 68).  None is shorter than two steps of every wave (one sequence of 1024 tokens, 26 drafted, 32
  // heads: 13.5 us; with parts of 128 14.4, of 512 15.9).
  const int64_t want = 2 * kChipCUs / groups;
  const int64_t most = std::max<int64_t>(1, (max_ctx + kMinPart - 1) / kMinPart);
  const int64_t parts = std::max<int64_t>(1, std::min<int64_t>({want, most, (int64_t)kMaxParts}));
  int64_t len = (max_ctx + parts - 1) / parts;
  if (accumulate) {  // a row's logits and 4 floats behind them, for every row of a workgroup
    const int64_t room = (kTreeLogitFloats / std::min<int64_t>(rows, p.max_rows) - 4) / kPartTokens * kPartTokens;
    if (len > room) {
      const int64_t n = (max_ctx + room - 1) / room;
      len = (max_ctx + n - 1) / n;
    }
  }
  len = std::max<int64_t>(kPartTokens, (len + kPartTokens - 1) / kPartTokens * kPartTokens);
  p.part_len = (int)len;
  p.parts = (int)std::max<int64_t>(1, ((int64_t)max_ctx + p.part_len - 1) / p.part_len);
  p.tile_rows = rows;
  const bool logits = accumulate && (p.parts > 1 || p.row_tiles > 1);
  const size_t cells = (size_t)num_seqs * num_kv_heads * p.parts * p.max_rows;
  p.ml_bytes = p.parts > 1 || logits ? cells * 16 : 0;
  p.acc_bytes = p.parts > 1 ? cells * head_size * 4 : 0;
  p.logit_stride = ((int64_t)max_ctx + 31) / 32 * 32;
  p.logit_bytes = logits ? (size_t)num_seqs * num_kv_heads * p.max_rows * p.logit_stride * 4 : 0;
  return p;
}

// Whether a launch of these bounds can be planned: a workgroup takes at most 128 rows of a kv head, a launch has at most
// 2^31 workgroups, and the plan's sums stay within 64 bits below that.
bool tree_fits(int num_seqs, int num_heads, int num_kv_heads, int max_ctx, int max_query) {
  const int64_t cells = (int64_t)num_seqs * num_kv_heads, rows = (int64_t)max_query * (num_heads / num_kv_heads);
  return max_ctx <= kMaxContext && cells <= 0x7fffffff && rows <= 0x7fffffff && cells * ((rows + 127) / 128) <= 0x7fffffff;
}

int tree_entry(const char* what, void* out, const void* query, const void* key_cache, const void* value_cache,
               float* weight_cache, bool accumulate, float scale, const int32_t* block_tables, const int32_t* context_lens,
               const int32_t* query_starts, const uint8_t* tree_mask, int64_t mask_stride, int num_seqs, int num_tokens,
               int num_heads, int num_kv_heads, int head_size, int block_size, int num_blocks, int max_num_blocks_per_seq,
               int max_context_len, int max_query_len, int64_t q_stride, int dtype, void* workspace,
               size_t workspace_bytes, void* stream) {
  clear_error();
  if (dtype != PA_DTYPE_F32 && dtype != PA_DTYPE_F16 && dtype != PA_DTYPE_BF16)
    return fail(PA_ERR_UNSUPPORTED, "%s: unsupported data type code: %d", what, dtype);
  if (head_size != 64 && head_size != 80 && head_size != 96 && head_size != 128)
    return fail(PA_ERR_UNSUPPORTED, "%s: unsupported head size: %d", what, head_size);
  if (block_size != 8 && block_size != 16 && block_size != 32)
    return fail(PA_ERR_UNSUPPORTED, "%s: unsupported block size: %d", what, block_size);
  PA_REQUIRE(num_seqs >= 0 && num_tokens >= 0 && num_heads >= 0 && num_kv_heads >= 0 && num_blocks >= 0 &&
                 max_num_blocks_per_seq >= 0 && max_context_len >= 0 && max_query_len >= 0,
             "%s: negative size", what);
  if (num_seqs == 0 || num_tokens == 0 || num_heads == 0 || max_query_len == 0) return PA_OK;
  PA_REQUIRE(num_kv_heads > 0 && num_heads % num_kv_heads == 0, "%s: num_heads %d is no multiple of num_kv_heads %d", what,
             num_heads, num_kv_heads);
  PA_REQUIRE(out && query && key_cache && value_cache && block_tables && context_lens && query_starts &&
                 (weight_cache || !accumulate),
             "%s: null pointer argument", what);
  PA_REQUIRE(aligned16(out) && aligned16(key_cache) && aligned16(value_cache) && aligned16(weight_cache),
             "%s: out and the caches must be 16-byte aligned", what);
  PA_REQUIRE(isfinite(scale * 1.44269504088896340736f), "%s: scale must be finite, its product with log2(e) too", what);
  PA_REQUIRE(num_tokens == 1 || q_stride >= (int64_t)num_heads * head_size, "%s: query row stride is shorter than a token row", what);
  PA_REQUIRE((int64_t)max_num_blocks_per_seq * block_size >= max_context_len,
             "%s: block tables of %d blocks cannot hold max_context_len %d", what, max_num_blocks_per_seq, max_context_len);
  PA_REQUIRE(max_query_len <= max_context_len, "%s: max_query_len %d exceeds max_context_len %d (which counts the new tokens)",
             what, max_query_len, max_context_len);
  PA_REQUIRE(max_context_len <= kMaxContext, "%s: max_context_len %d is too large", what, max_context_len);
  PA_REQUIRE(tree_mask == nullptr || mask_stride >= 0, "%s: negative mask stride", what);
  PA_REQUIRE(num_blocks > 0, "%s: the caches have no blocks", what);
  PA_REQUIRE((int64_t)num_kv_heads * head_size * block_size * elem_size(dtype) <= 0x7fffffff, "%s: a block of a cache exceeds 2 GiB", what);
  PA_REQUIRE(tree_fits(num_seqs, num_heads, num_kv_heads, max_context_len, max_query_len), "%s: too many rows for one launch", what);
  const TreePlan p = tree_plan(num_seqs, num_heads, num_kv_heads, head_size, max_context_len, max_query_len, accumulate,
                                dtype == PA_DTYPE_F32);
  const int64_t items = (int64_t)num_seqs * num_kv_heads * p.parts;
  const int64_t grid = (items + 7) / 8 * 8 * p.row_tiles;
  const int rows_per_group = 256 / (head_size / 4);
  const int64_t join_groups = p.parts > 1 ? ((int64_t)num_seqs * max_query_len * num_heads + rows_per_group - 1) / rows_per_group : 0;
  const int chunks = (max_context_len + kChunk - 1) / kChunk;
  const int64_t join_grid = join_groups + (p.logit_bytes ? (int64_t)num_seqs * num_kv_heads * chunks : 0);
  PA_REQUIRE(grid <= 0x7fffffff && join_grid <= 0x7fffffff, "%s: too many rows for one launch", what);
  PA_REQUIRE(p.bytes() == 0 || (workspace && aligned16(workspace) && workspace_bytes >= p.bytes()),
             "%s: workspace of %zu bytes, 16-byte aligned, needed", what, p.bytes());

  TreeArgs a = {};
  a.out = out;
  a.q = query;
  a.kc = static_cast<const char*>(key_cache);
  a.vc = static_cast<const char*>(value_cache);
  a.tables = block_tables;
  a.ctx = context_lens;
  a.starts = query_starts;
  a.mask = tree_mask;
  a.weights = accumulate ? weight_cache : nullptr;
  char* ws = static_cast<char*>(workspace);
  a.ml = reinterpret_cast<float*>(ws);
  a.acc = reinterpret_cast<float*>(ws + p.ml_bytes);
  a.logits = p.logit_bytes ? reinterpret_cast<float*>(ws + p.ml_bytes + p.acc_bytes) : nullptr;
  a.q_stride = q_stride;
  a.mask_stride = mask_stride;
  a.logit_stride = p.logit_stride;
  a.c = scale == 0.f ? 1.f : fabsf(scale) * 1.44269504088896340736f;
  a.q_mode = scale == 0.f ? 2 : (scale < 0.f ? 1 : 0);
  a.num_seqs = num_seqs;
  a.num_tokens = num_tokens;
  a.num_heads = num_heads;
  a.num_kv_heads = num_kv_heads;
  a.group = num_heads / num_kv_heads;
  a.num_blocks = num_blocks;
  a.block_bits = block_size == 8 ? 3 : (block_size == 16 ? 4 : 5);
  a.table_width = max_num_blocks_per_seq;
  a.max_ctx = max_context_len;
  a.max_query = max_query_len;
  a.max_rows = (int)p.max_rows;
  a.parts = p.parts;
  a.part_len = p.part_len;
  a.row_tiles = p.row_tiles;
  a.form = p.tile_rows;
  // Where workgroups wait for a CU, the longest sequences go first, if a partition may be long enough to repay the ranking
  // that every workgroup makes for itself, the longer the more sequences there are.  Ragged batches, longest first
  // against as they come: 24 to 96 sequences of up to 4096 tokens, 7 to 14 % less time, and of 2048 5 to 9 %; at the border
  // (64 sequences of 768, 128 of 1024) -8 to +5 %; below it 128 sequences of 512 +9 %, 256 of 384 +35 %, 256 of 64 +140 %.
  // Batches of one length lose 1 to 2 % by it at 4096 tokens.
  a.sorted = num_seqs > 1 && num_seqs <= kTreeSorted && items * p.row_tiles > kChipCUs && p.part_len >= std::max(768, 8 * num_seqs);
  hipStream_t st = static_cast<hipStream_t>(stream);
  int rc;
  switch (dtype) {
    case PA_DTYPE_F32: rc = tree_launch_f32(a, head_size, (unsigned)grid, st); break;
    case PA_DTYPE_F16: rc = tree_launch_f16(a, head_size, (unsigned)grid, st); break;
    default: rc = tree_launch_bf16(a, head_size, (unsigned)grid, st); break;
  }
  if (rc != PA_OK || join_grid == 0) return rc;
  const dim3 jg((unsigned)join_grid), jb(256);
  switch (dtype) {
    case PA_DTYPE_F32: hipLaunchKernelGGL((pa_tree_join_kernel<float>), jg, jb, 0, st, a, head_size, (unsigned)join_groups, chunks, p.tile_rows); break;
    case PA_DTYPE_F16: hipLaunchKernelGGL((pa_tree_join_kernel<_Float16>), jg, jb, 0, st, a, head_size, (unsigned)join_groups, chunks, p.tile_rows); break;
    default: hipLaunchKernelGGL((pa_tree_join_kernel<__bf16>), jg, jb, 0, st, a, head_size, (unsigned)join_groups, chunks, p.tile_rows); break;
  }
  PA_CHECK_LAUNCH(what);
  return PA_OK;
}

}  // namespace
}  // namespace pa

extern "C" size_t pa_tree_workspace_bytes(int num_seqs, int num_heads, int num_kv_heads, int head_size, int max_context_len,
                                          int max_query_len, int accumulate, int dtype) {
  if (num_seqs <= 0 || num_heads <= 0 || num_kv_heads <= 0 || head_size <= 0 || max_context_len <= 0 || max_query_len <= 0 ||
      num_heads % num_kv_heads != 0 || !pa::tree_fits(num_seqs, num_heads, num_kv_heads, max_context_len, max_query_len))
    return 0;
  return pa::tree_plan(num_seqs, num_heads, num_kv_heads, head_size, max_context_len, max_query_len, accumulate != 0,
                       dtype == PA_DTYPE_F32)
      .bytes();
}

extern "C" int pa_tree_cached_kv_attention(
    void* out, const void* query, const void* key_cache, const void* value_cache, float scale, const int32_t* block_tables,
    const int32_t* context_lens, const int32_t* query_starts, const uint8_t* tree_mask, int64_t mask_stride, int num_seqs,
    int num_tokens, int num_heads, int num_kv_heads, int head_size, int block_size, int num_blocks,
    int max_num_blocks_per_seq, int max_context_len, int max_query_len, int64_t q_stride, int dtype, void* workspace,
    size_t workspace_bytes, void* stream) {
  return pa::tree_entry("pa_tree_cached_kv_attention", out, query, key_cache, value_cache, nullptr, false, scale, block_tables,
                        context_lens, query_starts, tree_mask, mask_stride, num_seqs, num_tokens, num_heads, num_kv_heads,
                        head_size, block_size, num_blocks, max_num_blocks_per_seq, max_context_len, max_query_len, q_stride,
                        dtype, workspace, workspace_bytes, stream);
}

extern "C" int pa_cached_kv_attention_accumulate(
    void* out, const void* query, const void* key_cache, const void* value_cache, float* weight_cache, float scale,
    const int32_t* block_tables, const int32_t* context_lens, const int32_t* query_starts, int num_seqs, int num_tokens,
    int num_heads, int num_kv_heads, int head_size, int block_size, int num_blocks, int max_num_blocks_per_seq,
    int max_context_len, int max_query_len, int64_t q_stride, int dtype, void* workspace, size_t workspace_bytes,
    void* stream) {
  return pa::tree_entry("pa_cached_kv_attention_accumulate", out, query, key_cache, value_cache, weight_cache, true, scale,
                        block_tables, context_lens, query_starts, nullptr, 0, num_seqs, num_tokens, num_heads, num_kv_heads,
                        head_size, block_size, num_blocks, max_num_blocks_per_seq, max_context_len, max_query_len, q_stride,
                        dtype, workspace, workspace_bytes, stream);
}
