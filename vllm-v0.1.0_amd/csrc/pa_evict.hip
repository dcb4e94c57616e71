// Eviction from the paged cache by accumulated attention weight, for gfx950
// (MI355X).  No counterpart in the reference, whose cache only drops whole
// sequences.
//
// Of every (sequence, kv head) with more than `budget` positions, the last
// `num_recent` stay and, of the ones before, the budget - num_recent of the
// largest weight (equal weights: the lowest positions).  What stays keeps its
// order and moves to the front of the sequence's blocks: keys, values and
// weights, in place.  Heads choose for themselves, so slot i of a block holds
// another position in every head, which attention does not mind: keys carry
// their rotation.
//
// pa_evict_select_kernel: one workgroup to a (sequence, kv head).  The weights'
// bits, made to order like whole numbers, are searched for the last one that
// stays in three passes of 11, 11 and 10 bits (a histogram in LDS each), then
// every wave counts its stretch, and lists it behind the others'.  Up to kKeys
// weights are held in LDS; longer contexts read them from L2 again.
//
// pa_evict_move_kernel: one wave to 1 KiB of every block of a (sequence, kv head):
// a run of keys' chunks, of values' rows, or the weights.  It walks the blocks
// from the first that loses a position: a slot is written from a position at or
// behind it, so whatever is still to be read is never overwritten, and waves
// never share a byte.  Keys go straight to their slots, 16 bytes each; values,
// whose positions lie side by side in a row, are collected in LDS until a block
// is full.  Bound by HBM: with a quarter of the positions kept at random every
// 128-byte line of the old blocks holds one that stays, so the whole of them is
// read (the values' rows of a block even with one position in sixteen).
#include "pa_common.h"

namespace pa {

struct EvictArgs {
  char* kc;
  char* vc;
  float* weights;           // [num_blocks, heads, block]
  const int32_t* tables;
  const int32_t* ctx;
  int32_t* kept;            // [num_seqs, heads, budget]
  uint64_t* masks;          // [num_seqs, heads, words]: which of 64 positions stay
  int32_t* ranks;           // [num_seqs, heads, words]: how many stay before them
  int32_t* first;           // [num_seqs, heads]: the first block that loses a position, -1: none
  int heads, block_bits, num_blocks, table_width, max_ctx, budget, recent, words;
  int tile_bytes;           // of one head's share of a block: head_size * block * element size
  int slices;               // ceil(tile_bytes / 1024)
  int64_t tasks;            // (sequence, head, slice) of the move
};

namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr int kKeys = 8192;
constexpr int kBins = 2048;

// A weight as a whole number of the same order: NaN first of all, then by value, both zeros alike.
__device__ __forceinline__ uint32_t order_key(uint32_t bits) {
  if ((bits & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
  if (bits == 0x80000000u) bits = 0;
  return (bits >> 31) ? ~bits : (bits | 0x80000000u);
}

__global__ void __launch_bounds__(kThreads) pa_evict_select_kernel(const EvictArgs a) {
  const int sh = blockIdx.x, seq = sh / a.heads, head = sh - seq * a.heads;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int n = a.ctx[seq];
  const int32_t* table = a.tables + (int64_t)seq * a.table_width;
  int32_t* kept = a.kept + (int64_t)sh * a.budget;
  bool bad = n < 0 || n > a.max_ctx || n > ((int64_t)a.table_width << a.block_bits);
  if (!bad) {
    bool out = false;
    for (int e = tid; e < (n + (1 << a.block_bits) - 1) >> a.block_bits; e += kThreads) out |= (unsigned)table[e] >= (unsigned)a.num_blocks;
    bad = __syncthreads_or(out) != 0;
  }
  if (bad || n <= a.budget) {  // nothing moves
    for (int i = tid; i < a.budget; i += kThreads) kept[i] = !bad && i < n ? i : -1;
    if (tid == 0) a.first[sh] = -1;
    return;
  }
  __shared__ uint32_t sm_key[kKeys];
  __shared__ uint32_t sm_hist[kBins];
  __shared__ uint32_t sm_scan[kWaves];
  __shared__ uint32_t sm_bin, sm_need;
  __shared__ int sm_gt[kWaves], sm_eq[kWaves], sm_first;
  const int candidates = n - a.recent;
  const uint32_t* weights = reinterpret_cast<const uint32_t*>(a.weights);
  const auto fetch = [&](int p) {
    const int64_t b = table[p >> a.block_bits];
    return order_key(weights[((b * a.heads + head) << a.block_bits) + (p & ((1 << a.block_bits) - 1))]);
  };
  for (int p = tid; p < candidates && p < kKeys; p += kThreads) sm_key[p] = fetch(p);
  if (tid == 0) sm_first = n;
  const auto key = [&](int p) { return p < kKeys ? sm_key[p] : fetch(p); };

  uint32_t limit = 0, need = (uint32_t)(a.budget - a.recent);  // need: how many of the keys with limit's upper bits stay
  const bool any = need > 0;
  if (any) {
#pragma unroll 1
    for (int pass = 0; pass < 3; pass++) {
      const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0), bits = pass == 2 ? 10 : 11;
      for (int i = tid; i < kBins; i += kThreads) sm_hist[i] = 0;
      __syncthreads();
      for (int p = tid; p < candidates; p += kThreads) {
        const uint32_t k = key(p);
        if (pass == 0 || (k >> (shift + bits)) == (limit >> (shift + bits))) atomicAdd(&sm_hist[(k >> shift) & ((1u << bits) - 1u)], 1u);
      }
      __syncthreads();
      // bins from the highest down, two to a thread: the one in which the need-th key lies
      const uint32_t hi = sm_hist[kBins - 1 - 2 * tid], lo = sm_hist[kBins - 2 - 2 * tid];
      uint32_t sum = hi + lo;
#pragma unroll
      for (int off = 1; off < 64; off <<= 1) {
        const uint32_t v = __shfl_up(sum, off);
        if (lane >= off) sum += v;
      }
      if (lane == 63) sm_scan[wave] = sum;
      __syncthreads();
      uint32_t before = 0;
      for (int w = 0; w < wave; w++) before += sm_scan[w];
      before += sum - (hi + lo);
      if (before < need && need <= before + hi + lo) {
        const bool in_hi = need <= before + hi;
        sm_bin = in_hi ? kBins - 1 - 2 * tid : kBins - 2 - 2 * tid;
        sm_need = need - before - (in_hi ? 0 : hi);
      }
      __syncthreads();
      limit |= sm_bin << shift;
      need = sm_need;
      __syncthreads();
    }
  } else {
    __syncthreads();
  }
  // Every wave a stretch of whole words of 64 positions: counts first, then the list.
  const int seg = ((n + kWaves - 1) / kWaves + 63) / 64 * 64;
  const int lo = wave * seg, hi = lo + seg < n ? lo + seg : n;
  const auto judge = [&](int p, bool* gt, bool* eq) {
    *gt = *eq = false;
    if (p >= n) return;
    if (p >= candidates) {
      *gt = true;
    } else if (any) {
      const uint32_t k = key(p);
      *gt = k > limit;
      *eq = k == limit;
    }
  };
  int gts = 0, eqs = 0;
  for (int p = lo; p < hi; p += 64) {
    bool gt, eq;
    judge(p + lane, &gt, &eq);
    gts += __popcll(__ballot(gt));
    eqs += __popcll(__ballot(eq));
  }
  if (lane == 0) {
    sm_gt[wave] = gts;
    sm_eq[wave] = eqs;
  }
  __syncthreads();
  int run = 0, ties = 0;
  for (int w = 0; w < wave; w++) {
    run += sm_gt[w];
    ties += sm_eq[w];
  }
  const int wanted = any ? (int)need : 0;
  run += ties < wanted ? ties : wanted;
  const uint64_t below = (1ull << lane) - 1ull;
  int dropped = n;
  for (int p = lo; p < hi; p += 64) {
    bool gt, eq;
    judge(p + lane, &gt, &eq);
    const uint64_t em = __ballot(eq);
    const bool stays = gt || (eq && ties + __popcll(em & below) < wanted);
    ties += __popcll(em);
    const uint64_t mask = __ballot(stays);
    if (stays) kept[run + __popcll(mask & below)] = p + lane;
    if (lane == 0) {
      a.masks[(int64_t)sh * a.words + (p >> 6)] = mask;
      a.ranks[(int64_t)sh * a.words + (p >> 6)] = run;
    }
    run += __popcll(mask);
    if (dropped == n && ~mask != 0) {
      const int at = p + __ffsll((unsigned long long)~mask) - 1;
      if (at < n) dropped = at;
    }
  }
  if (lane == 0 && dropped < n) atomicMin(&sm_first, dropped);
  __syncthreads();
  if (tid == 0) a.first[sh] = sm_first >> a.block_bits;
}

constexpr int kAhead = 4;  // blocks whose loads are in flight beside the ones being placed

// X: elements of 16 bytes.  The tables that no store of the kernel touches are arguments of their
// own: their loads, the same for all lanes, then go through the scalar cache and its counter, and no
// wait for them waits for the blocks that are on their way.
template <typename T, int X>
__global__ void __launch_bounds__(256)
pa_evict_move_kernel(const EvictArgs a, const int32_t* __restrict__ tables, const int32_t* __restrict__ ctx,
                     const uint64_t* __restrict__ all_masks, const int32_t* __restrict__ all_ranks,
                     const int32_t* __restrict__ firsts, char* __restrict__ kc, char* __restrict__ vc,
                     float* __restrict__ weights) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t task = (int64_t)blockIdx.x * 4 + wave;
  if (task >= a.tasks) return;
  const int kinds = 2 * a.slices + 1;
  const int sh = (int)(task / kinds), kind = (int)(task - (int64_t)sh * kinds);
  const int first = firsts[sh];
  if (first < 0) return;
  const int seq = sh / a.heads, head = sh - seq * a.heads;
  const int n = ctx[seq], B = 1 << a.block_bits, blocks = (n + B - 1) >> a.block_bits;
  const int32_t* table = tables + (int64_t)seq * a.table_width;
  const uint64_t* masks = all_masks + (int64_t)sh * a.words;
  const int32_t* ranks = all_ranks + (int64_t)sh * a.words;

  if (kind == 2 * a.slices) {  // weights, 64 positions at a time
    const auto slot = [&](int p) { return ((((int64_t)table[p >> a.block_bits]) * a.heads + head) << a.block_bits) + (p & (B - 1)); };
    const int last = (n - 1) >> 6;
    int w = (first << a.block_bits) >> 6;
    float next = 0.f;
    if (w * 64 + lane < n) next = weights[slot(w * 64 + lane)];
    for (; w <= last; w++) {
      const float v = next;
      if ((w + 1) * 64 + lane < n) next = weights[slot((w + 1) * 64 + lane)];
      const uint64_t mask = masks[w];
      if ((mask >> lane) & 1) weights[slot(ranks[w] + __popcll(mask & ((1ull << lane) - 1ull)))] = v;
    }
    return;
  }
  const bool values = kind >= a.slices;
  const int at = (values ? kind - a.slices : kind) * 1024 + lane * 16;  // this lane's bytes of the tile
  const bool mine = at < a.tile_bytes;
  char* base = (values ? vc : kc) + (int64_t)head * a.tile_bytes;
  const int64_t block_bytes = (int64_t)a.heads * a.tile_bytes;
  const int vec = at >> 4;
  const int per_row = B / X;                                            // values: vectors of a row
  const int token = values ? (vec & (per_row - 1)) * X : vec & (B - 1);  // the (first) token of this lane's vector
  __shared__ __attribute__((aligned(16))) T sm[4][128 * X];
  T* strip = sm[wave] + (lane / per_row) * 2 * B;                       // this lane's row: two blocks of tokens

  const auto bits_of = [&](int b, int* rank) {  // which tokens of block b stay, and the slot of the first
    const int p = b << a.block_bits;
    const uint64_t mask = masks[p >> 6];
    *rank = ranks[p >> 6] + __popcll(mask & ((1ull << (p & 63)) - 1ull));
    return (uint32_t)(mask >> (p & 63)) & (B == 32 ? 0xffffffffu : (1u << B) - 1u);
  };
  const auto fetch = [&](int b) {
    u32x4 v = {0, 0, 0, 0};
    if (b < blocks) {
      int rank;
      if (bits_of(b, &rank) != 0 && mine) v = *reinterpret_cast<const u32x4*>(base + (int64_t)table[b] * block_bytes + at);
    }
    return v;
  };
  const auto flush = [&](int slot_block) {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    const u32x4 v = *reinterpret_cast<const u32x4*>(strip + (slot_block & 1) * B + token);
    if (mine) *reinterpret_cast<u32x4*>(base + (int64_t)table[slot_block] * block_bytes + at) = v;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  };
  u32x4 ahead[kAhead];
#pragma unroll
  for (int u = 0; u < kAhead; u++) ahead[u] = fetch(first + u);
  int filled = first << a.block_bits;  // slots done
  for (int b0 = first; b0 < blocks; b0 += kAhead) {
    u32x4 now[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; u++) now[u] = ahead[u];
#pragma unroll
    for (int u = 0; u < kAhead; u++) ahead[u] = fetch(b0 + kAhead + u);
#pragma unroll
    for (int u = 0; u < kAhead; u++) {
      if (b0 + u >= blocks) break;
      int rank;
      const uint32_t bits = bits_of(b0 + u, &rank);
      if (bits == 0) continue;
      const int e0 = rank >> a.block_bits;
      if (!values) {
        const int e1 = e0 + 1 < blocks ? e0 + 1 : e0;
        const int to = rank + __popc(bits & ((1u << token) - 1u));
        const int64_t t0 = table[e0], t1 = table[e1];
        if (mine && ((bits >> token) & 1u))
          *reinterpret_cast<u32x4*>(base + ((to >> a.block_bits) == e0 ? t0 : t1) * block_bytes + at + ((to & (B - 1)) - token) * 16) = now[u];
      } else {
#pragma unroll
        for (int i = 0; i < X; i++) {
          const T e = (T)(X == 4 ? now[u][i & 3] : now[u][i >> 1] >> (16 * (i & 1)));
          if ((bits >> (token + i)) & 1u) strip[(rank + __popc(bits & ((1u << (token + i)) - 1u))) & (2 * B - 1)] = e;
        }
        filled = rank + __popc(bits);
        if ((rank ^ filled) >> a.block_bits) flush(e0);
      }
    }
  }
  if (values && (filled & (B - 1))) {  // the last block's slots behind the budget stay as they are
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    const int slot_block = filled >> a.block_bits, left = (filled & (B - 1)) - token;
    T* to = reinterpret_cast<T*>(base + (int64_t)table[slot_block] * block_bytes + at);
#pragma unroll
    for (int i = 0; i < X; i++)
      if (mine && i < left) to[i] = strip[(slot_block & 1) * B + token + i];
  }
}

struct EvictPlan {
  int words;
  size_t mask_bytes, rank_bytes, first_bytes;
  size_t bytes() const { return mask_bytes + rank_bytes + first_bytes; }
};

EvictPlan evict_plan(int num_seqs, int heads, int max_ctx) {
  EvictPlan p;
  p.words = (max_ctx + 63) / 64;
  const size_t cells = (size_t)num_seqs * heads;
  p.mask_bytes = cells * p.words * 8;
  p.rank_bytes = (cells * p.words * 4 + 15) / 16 * 16;
  p.first_bytes = (cells * 4 + 15) / 16 * 16;
  return p;
}

}  // namespace
}  // namespace pa

extern "C" size_t pa_evict_workspace_bytes(int num_seqs, int num_kv_heads, int max_context_len) {
  if (num_seqs <= 0 || num_kv_heads <= 0 || max_context_len < 0) return 0;
  return pa::evict_plan(num_seqs, num_kv_heads, max_context_len).bytes();
}

extern "C" int pa_evict_cached_kv(void* key_cache, void* value_cache, float* weight_cache, const int32_t* block_tables,
                                  const int32_t* context_lens, int32_t* kept_positions, int num_seqs, int num_kv_heads,
                                  int head_size, int block_size, int num_blocks, int max_num_blocks_per_seq,
                                  int max_context_len, int budget, int num_recent, int dtype, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  using namespace pa;
  clear_error();
  const char* what = "pa_evict_cached_kv";
  if (dtype != PA_DTYPE_F32 && dtype != PA_DTYPE_F16 && dtype != PA_DTYPE_BF16)
    return fail(PA_ERR_UNSUPPORTED, "%s: unsupported data type code: %d", what, dtype);
  if (block_size != 8 && block_size != 16 && block_size != 32)
    return fail(PA_ERR_UNSUPPORTED, "%s: unsupported block size: %d", what, block_size);
  PA_REQUIRE(num_seqs >= 0 && num_kv_heads >= 0 && head_size >= 0 && num_blocks >= 0 && max_num_blocks_per_seq >= 0 &&
                 max_context_len >= 0,
             "%s: negative size", what);
  PA_REQUIRE(budget >= 1, "%s: budget %d must be positive", what, budget);
  PA_REQUIRE(num_recent >= 0 && num_recent <= budget, "%s: num_recent %d must be in [0, budget %d]", what, num_recent, budget);
  if (num_seqs == 0 || num_kv_heads == 0) return PA_OK;
  const int x = 16 / elem_size(dtype);
  PA_REQUIRE(head_size > 0 && head_size <= 4096 && head_size % x == 0, "%s: head size %d must be a multiple of %d, at most 4096",
             what, head_size, x);
  PA_REQUIRE(key_cache && value_cache && weight_cache && block_tables && context_lens && kept_positions,
             "%s: null pointer argument", what);
  PA_REQUIRE(aligned16(key_cache) && aligned16(value_cache) && aligned16(weight_cache), "%s: the caches must be 16-byte aligned", what);
  PA_REQUIRE((int64_t)max_num_blocks_per_seq * block_size >= max_context_len,
             "%s: block tables of %d blocks cannot hold max_context_len %d", what, max_num_blocks_per_seq, max_context_len);
  PA_REQUIRE(max_context_len <= (1 << 30), "%s: max_context_len %d is too large", what, max_context_len);
  const EvictPlan p = evict_plan(num_seqs, num_kv_heads, max_context_len);
  PA_REQUIRE(workspace && aligned16(workspace) && workspace_bytes >= p.bytes(),
             "%s: workspace of %zu bytes, 16-byte aligned, needed", what, p.bytes());
  const int64_t cells = (int64_t)num_seqs * num_kv_heads;
  EvictArgs a = {};
  a.kc = static_cast<char*>(key_cache);
  a.vc = static_cast<char*>(value_cache);
  a.weights = weight_cache;
  a.tables = block_tables;
  a.ctx = context_lens;
  a.kept = kept_positions;
  char* ws = static_cast<char*>(workspace);
  a.masks = reinterpret_cast<uint64_t*>(ws);
  a.ranks = reinterpret_cast<int32_t*>(ws + p.mask_bytes);
  a.first = reinterpret_cast<int32_t*>(ws + p.mask_bytes + p.rank_bytes);
  a.heads = num_kv_heads;
  a.block_bits = block_size == 8 ? 3 : (block_size == 16 ? 4 : 5);
  a.num_blocks = num_blocks;
  a.table_width = max_num_blocks_per_seq;
  a.max_ctx = max_context_len;
  a.budget = budget;
  a.recent = num_recent;
  a.words = p.words;
  a.tile_bytes = head_size * block_size * elem_size(dtype);
  a.slices = (a.tile_bytes + 1023) / 1024;
  a.tasks = cells * (2 * a.slices + 1);
  PA_REQUIRE(cells <= 0x7fffffff && (a.tasks + 3) / 4 <= 0x7fffffff, "%s: too many heads for one launch", what);
  hipStream_t st = static_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(pa_evict_select_kernel, dim3((unsigned)cells), dim3(kThreads), 0, st, a);
  PA_CHECK_LAUNCH(what);
  if (max_context_len <= budget) return PA_OK;  // no sequence can lose a position
  const dim3 grid((unsigned)((a.tasks + 3) / 4));
  if (elem_size(dtype) == 4)
    hipLaunchKernelGGL((pa_evict_move_kernel<uint32_t, 4>), grid, dim3(256), 0, st, a, a.tables, a.ctx, a.masks, a.ranks, a.first, a.kc, a.vc, a.weights);
  else
    hipLaunchKernelGGL((pa_evict_move_kernel<uint16_t, 8>), grid, dim3(256), 0, st, a, a.tables, a.ctx, a.masks, a.ranks, a.first, a.kc, a.vc, a.weights);
  PA_CHECK_LAUNCH(what);
  return PA_OK;
}
