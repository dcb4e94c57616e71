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
// weights are held in LDS with their part of the block table, and moved from
// there; longer contexts read the rest from L2 in every pass.
//
// pa_evict_move_kernel: one wave to 4 chunks of the keys of a (sequence, kv head), or to 16 rows of its values.  It
// walks the slots from the first that changes, and takes each from where the list says: a slot comes from a position at
// or behind it, so what later slots need is never overwritten, and waves never share a byte.  A key's piece is one
// load and one store; a value's is put together of single elements, as positions lie side by side in a row.  128 slots'
// loads are on their way at once, the block table's for the next 128 and the list's for the ones behind them too.
// Bound by HBM: with a quarter of the positions kept at random nearly every 128-byte line of the old blocks holds one
// that stays, so the whole of them is read (the values' rows of a block even with one position in sixteen).
//
// A wave is a workgroup: a gather keeps a CU's address unit for its 64 elements, and waves of one workgroup share
// one (a sequence of 8192 positions to 2048 in all 48 us, four waves to a workgroup 70; 32 sequences 290 and 315).
// 32 sequences of 8 kv heads of 128, 16 bits, of 8192 positions to 2048, random weights: 22 us to select, 264 to
// move, 1.28 GB by the counters = 4.8 TB/s.  Few heads of long contexts are bound by the walk itself, 128 slots at a
// time: 2 sequences of one head, 15445 positions to 6464, 85 to 110 us.  With 32 rows to a wave instead of 16, 7 % more (and 8 sequences of
// 16000 to 4000 236 in all against 182: too few waves), with 2 or 1 chunks of the keys no less.  A walk over the old
// positions, each sent to its slot, took 40 % longer: the slots have to be counted along the way, and its loads wait
// for conditional stores.
#include <type_traits>

#include "pa_common.h"

namespace pa {

struct EvictArgs {
  char* kc;
  char* vc;
  float* weights;           // [num_blocks, heads, block]
  const int32_t* tables;
  const int32_t* ctx;
  int32_t* kept;            // [num_seqs, heads, budget]
  int32_t* first;           // [num_seqs, heads]: the first position that goes, -1: none
  int heads, head_size, block_bits, num_blocks, table_width, max_ctx, budget, recent;
  int tile_bytes;           // of one head's share of a block: head_size * block * element size
  int key_tasks, value_tasks;  // waves of a (sequence, head): for its keys, for its values, and one for its weights
};

namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr int kKeys = 16384;
constexpr int kEntries = kKeys / 8;  // of the block table, at the smallest block
constexpr int kBins = 2048;
constexpr int kBatch = 8;            // loads of a thread on their way at once

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
  __shared__ uint32_t sm_bits[kKeys];
  __shared__ int32_t sm_table[kEntries];
  __shared__ uint32_t sm_hist[kBins];
  __shared__ uint32_t sm_scan[kWaves];
  __shared__ uint32_t sm_bin, sm_need;
  __shared__ int sm_gt[kWaves], sm_eq[kWaves], sm_first;
  const int candidates = n - a.recent, held = n < kKeys ? n : kKeys;
  uint32_t* weights = reinterpret_cast<uint32_t*>(a.weights);
  const int within = (1 << a.block_bits) - 1;
  for (int e = tid; e <= (held - 1) >> a.block_bits; e += kThreads) sm_table[e] = table[e];
  if (tid == 0) sm_first = n;
  __syncthreads();
  const auto slot = [&](int block, int p) { return (((int64_t)block * a.heads + head) << a.block_bits) + (p & within); };
  for (int p0 = tid; p0 < held; p0 += kBatch * kThreads) {
    uint32_t v[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; i++) {
      const int p = p0 + i * kThreads < held ? p0 + i * kThreads : held - 1;
      v[i] = weights[slot(sm_table[p >> a.block_bits], p)];
    }
#pragma unroll
    for (int i = 0; i < kBatch; i++)
      if (p0 + i * kThreads < held) sm_bits[p0 + i * kThreads] = v[i];
  }
  __syncthreads();
  // positions tid, tid + kThreads, ... from LDS, then from memory, several at once
  const auto each_key = [&](auto use) {
    for (int p = tid; p < candidates && p < kKeys; p += kThreads) use(order_key(sm_bits[p]));
    for (int p0 = kKeys + tid; p0 < candidates; p0 += kBatch * kThreads) {
      int32_t b[kBatch];
      uint32_t v[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; i++) b[i] = table[(p0 + i * kThreads < candidates ? p0 + i * kThreads : candidates - 1) >> a.block_bits];
#pragma unroll
      for (int i = 0; i < kBatch; i++) {
        const int p = p0 + i * kThreads < candidates ? p0 + i * kThreads : candidates - 1;
        v[i] = weights[slot(b[i], p)];
      }
#pragma unroll
      for (int i = 0; i < kBatch; i++)
        if (p0 + i * kThreads < candidates) use(order_key(v[i]));
    }
  };
  const auto key = [&](int p) { return order_key(p < kKeys ? sm_bits[p] : weights[slot(table[p >> a.block_bits], p)]); };

  uint32_t limit = 0, need = (uint32_t)(a.budget - a.recent);  // need: how many of the keys with limit's upper bits stay
  const bool any = need > 0;
  if (any) {
#pragma unroll 1
    for (int pass = 0; pass < 3; pass++) {
      const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0), bits = pass == 2 ? 10 : 11;
      for (int i = tid; i < kBins; i += kThreads) sm_hist[i] = 0;
      __syncthreads();
      each_key([&](uint32_t k) {
        if (pass == 0 || (k >> (shift + bits)) == (limit >> (shift + bits))) atomicAdd(&sm_hist[(k >> shift) & ((1u << bits) - 1u)], 1u);
      });
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
#pragma unroll
      for (int w = 0; w < kWaves; w++) before += w < wave ? sm_scan[w] : 0u;  // all reads at once
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
#pragma unroll
  for (int w = 0; w < kWaves; w++) {
    run += w < wave ? sm_gt[w] : 0;
    ties += w < wave ? sm_eq[w] : 0;
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
    if (stays) {
      const int to = run + __popcll(mask & below);
      kept[to] = p + lane;
      if (n <= kKeys) weights[slot(sm_table[to >> a.block_bits], to)] = sm_bits[p + lane];
    }
    run += __popcll(mask);
    if (dropped == n && ~mask != 0) {
      const int at = p + __ffsll((unsigned long long)~mask) - 1;
      if (at < n) dropped = at;
    }
  }
  if (lane == 0 && dropped < n) atomicMin(&sm_first, dropped);
  __syncthreads();
  if (tid == 0) a.first[sh] = sm_first;
}

constexpr int kSlots = 16;  // a wave's step
constexpr int kRows = 16;   // and its rows of the values

// X: elements of 16 bytes
template <typename T, int X>
__global__ void __launch_bounds__(64)
pa_evict_move_kernel(const EvictArgs a, const int32_t* __restrict__ tables, const int32_t* __restrict__ all_kept,
                     const int32_t* __restrict__ firsts, char* __restrict__ kc, char* __restrict__ vc,
                     float* __restrict__ weights) {
  const int lane = threadIdx.x;
  const unsigned task = blockIdx.x;
  const int kinds = a.key_tasks + a.value_tasks + 1;
  const int sh = (int)(task / (unsigned)kinds), kind = (int)(task - (unsigned)sh * (unsigned)kinds);
  const int first = firsts[sh];
  if (first < 0) return;
  const int seq = sh / a.heads, head = sh - seq * a.heads;
  const int bits = a.block_bits, B = 1 << bits, last = a.budget - 1;
  const int32_t* table = tables + (int64_t)seq * a.table_width;
  const int32_t* kept = all_kept + (int64_t)sh * a.budget;
  const auto within = [&](int slot) { return slot < last ? slot : last; };  // slots past the last: the last again

  if (kind == a.key_tasks + a.value_tasks) {  // the weights of a context that was too long for the selection's LDS
    if (a.ctx[seq] <= kKeys) return;
    const auto at = [&](int block, int p) { return (((int64_t)block * a.heads + head) << bits) + (p & (B - 1)); };
    constexpr int U = 8;
    for (int w0 = first & ~63; w0 <= last; w0 += 64 * U) {
      int p[U];
      float v[U];
      int64_t to[U];
#pragma unroll
      for (int u = 0; u < U; u++) p[u] = kept[within(w0 + 64 * u + lane)];
#pragma unroll
      for (int u = 0; u < U; u++) {
        const int slot = within(w0 + 64 * u + lane);
        v[u] = weights[at(table[p[u] >> bits], p[u])];
        to[u] = at(table[slot >> bits], slot);
      }
#pragma unroll
      for (int u = 0; u < U; u++)
        if (w0 + 64 * u + lane <= last) weights[to[u]] = v[u];
    }
    return;
  }
  const int64_t block_bytes = (int64_t)a.heads * a.tile_bytes;
  // 64 slots at a time, one to a lane: where it is (block * B + offset) and where it comes from, in pages of
  // which the next is on its way and the list for the one behind it too.  Lanes get them from each other: as
  // loads of their own they would be two to an element, and the address units' time is what values are bound by.
  struct Page { int position, from, to; };
  const auto ask = [&](int w) { return kept[within(w + lane)]; };
  const auto look_up = [&](int position, int w) {
    Page r;
    r.position = position;
    r.from = table[position >> bits];
    r.to = table[within(w + lane) >> bits];
    return r;
  };
  const auto source = [&](const Page& g) { return g.from << bits | (g.position & (B - 1)); };
  const auto target = [&](const Page& g, int w) { return g.to << bits | (within(w + lane) & (B - 1)); };
  const auto lane_of = [](int v, int l) { return __builtin_amdgcn_ds_bpermute(l * 4, v); };
  const int w0 = first & ~(kSlots - 1);

  if (kind < a.key_tasks) {
    constexpr int G = 2, U = 64 / kSlots;  // pages, and steps of a page
    const int t = lane & (kSlots - 1), chunk = kind * 4 + lane / kSlots;
    const bool mine = chunk < a.head_size / X;
    char* base = kc + (int64_t)head * a.tile_bytes + (mine ? chunk : 0) * B * 16;
    const auto address = [&](int slot) { return base + (int64_t)(slot >> bits) * block_bytes + (slot & (B - 1)) * 16; };
    Page page[G];
    int next[G];
#pragma unroll
    for (int q = 0; q < G; q++) {
      page[q] = look_up(ask(w0 + 64 * q), w0 + 64 * q);
      next[q] = ask(w0 + 64 * (G + q));
    }
    for (int w = w0; w <= last; w += 64 * G) {
      u32x4 v[G][U];
      char* dst[G][U];
#pragma unroll
      for (int q = 0; q < G; q++) {
        const int from = source(page[q]), to = target(page[q], w + 64 * q);
#pragma unroll
        for (int u = 0; u < U; u++) {
          v[q][u] = *reinterpret_cast<const u32x4*>(address(lane_of(from, u * kSlots + t)));
          dst[q][u] = address(lane_of(to, u * kSlots + t));
        }
      }
      Page ahead[G];
#pragma unroll
      for (int q = 0; q < G; q++) ahead[q] = look_up(next[q], w + 64 * (G + q));
#pragma unroll
      for (int q = 0; q < G; q++) next[q] = ask(w + 64 * (2 * G + q));
#pragma unroll
      for (int q = 0; q < G; q++)
#pragma unroll
        for (int u = 0; u < U; u++)
          if (mine && w + 64 * q + kSlots * u + t <= last) *reinterpret_cast<u32x4*>(dst[q][u]) = v[q][u];
#pragma unroll
      for (int q = 0; q < G; q++) page[q] = ahead[q];
    }
    return;
  }

  // Values: a slot and four rows to a load, so that its 64 elements lie in few lines: a block's four rows are one or
  // two.  16-bit elements are exchanged among four lanes, which store four slots each: a batch that has been through
  // it before, 59 us with four waves to a workgroup; a lane to a row and eight slots of it, 64 rows' lines to a load, 71.
  constexpr int U = 64 / kSlots, G = 2, LOADS = kRows / 4;
  const int t = lane & (kSlots - 1), sub = lane / kSlots, row0 = (kind - a.key_tasks) * kRows;
  const int row_bytes = B * (int)sizeof(T);
  char* base = vc + (int64_t)head * a.tile_bytes + (int64_t)(row0 + sub) * row_bytes;
  const auto address = [&](int slot) { return base + (int64_t)(slot >> bits) * block_bytes + (slot & (B - 1)) * (int)sizeof(T); };
  // four rows are all within the head or none: the head size is a multiple of X
  const auto rows = [&](int k) { return row0 + 4 * k < a.head_size ? 4 * k * row_bytes : 0; };
  Page page[G];
  int next[G];
#pragma unroll
  for (int q = 0; q < G; q++) {
    page[q] = look_up(ask(w0 + 64 * q), w0 + 64 * q);
    next[q] = ask(w0 + 64 * (G + q));
  }
  for (int w = w0; w <= last; w += 64 * G) {
    T v[G][U][LOADS];
    char* dst[G][U];
#pragma unroll
    for (int q = 0; q < G; q++) {
      const int from = source(page[q]), to = target(page[q], w + 64 * q);
#pragma unroll
      for (int u = 0; u < U; u++) {
        const char* src = address(lane_of(from, u * kSlots + t));
#pragma unroll
        for (int k = 0; k < LOADS; k++) v[q][u][k] = *reinterpret_cast<const T*>(src + rows(k));
        dst[q][u] = address(lane_of(to, u * kSlots + t));
      }
    }
    Page ahead[G];
#pragma unroll
    for (int q = 0; q < G; q++) ahead[q] = look_up(next[q], w + 64 * (G + q));
#pragma unroll
    for (int q = 0; q < G; q++) next[q] = ask(w + 64 * (2 * G + q));
    const auto put = [&](auto whole) {
      constexpr bool kWhole = decltype(whole)::value;  // all slots within the budget, all rows within the head
#pragma unroll
      for (int q = 0; q < G; q++)
#pragma unroll
        for (int u = 0; u < U; u++) {
          const int slot = w + 64 * q + kSlots * u + t;
          if constexpr (X == 4) {
#pragma unroll
            for (int k = 0; k < LOADS; k++)
              if (kWhole || (slot <= last && row0 + 4 * k < a.head_size)) *reinterpret_cast<T*>(dst[q][u] + 4 * k * row_bytes) = v[q][u][k];
          } else {
            const int mine = t & 3, quad = slot - mine;  // of four lanes' slots and four loads' rows a lane stores its row
            char* to = dst[q][u] + 4 * mine * row_bytes - (kWhole || slot <= last ? slot - quad : last - quad) * (int)sizeof(T);
#pragma unroll
            for (int k = 0; k < LOADS; k += 4) {
              uint32_t pair[2], r[2];
#pragma unroll
              for (int i = 0; i < 2; i++) {
                const uint32_t x = v[q][u][k + 2 * i], y = v[q][u][k + 2 * i + 1];
                const uint32_t other = (uint32_t)__builtin_amdgcn_mov_dpp((int)(mine & 1 ? x : y), 0xb1, 0xf, 0xf, true);
                pair[i] = mine & 1 ? other | y << 16 : x | other << 16;
              }
              const uint32_t other = (uint32_t)__builtin_amdgcn_mov_dpp((int)(mine & 2 ? pair[0] : pair[1]), 0x4e, 0xf, 0xf, true);
              r[0] = mine & 2 ? other : pair[0];
              r[1] = mine & 2 ? pair[1] : other;
              const bool in = row0 + 4 * (k + mine) < a.head_size;
              if (kWhole || (in && quad + 3 <= last)) {
                *reinterpret_cast<uint2*>(to + 4 * k * row_bytes) = make_uint2(r[0], r[1]);
              } else if (in) {  // the slots behind the budget stay as they are
#pragma unroll
                for (int i = 0; i < 4; i++)
                  if (quad + i <= last) reinterpret_cast<T*>(to + 4 * k * row_bytes)[i] = (T)(r[i >> 1] >> (16 * (i & 1)));
              }
            }
          }
        }
    };
    if (w + 64 * G - 1 <= last && row0 + kRows <= a.head_size) put(std::true_type{});
    else put(std::false_type{});
#pragma unroll
    for (int q = 0; q < G; q++) page[q] = ahead[q];
  }
}

size_t evict_bytes(int num_seqs, int heads) { return ((size_t)num_seqs * heads * 4 + 15) / 16 * 16; }

}  // namespace
}  // namespace pa

extern "C" size_t pa_evict_workspace_bytes(int num_seqs, int num_kv_heads) {
  return num_seqs <= 0 || num_kv_heads <= 0 ? 0 : pa::evict_bytes(num_seqs, num_kv_heads);
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
  PA_REQUIRE((int64_t)num_blocks * block_size <= 0x7fffffff, "%s: more than 2^31 slots", what);
  PA_REQUIRE(workspace && aligned16(workspace) && workspace_bytes >= evict_bytes(num_seqs, num_kv_heads),
             "%s: workspace of %zu bytes, 16-byte aligned, needed", what, evict_bytes(num_seqs, num_kv_heads));
  const int64_t cells = (int64_t)num_seqs * num_kv_heads;
  EvictArgs a = {};
  a.kc = static_cast<char*>(key_cache);
  a.vc = static_cast<char*>(value_cache);
  a.weights = weight_cache;
  a.tables = block_tables;
  a.ctx = context_lens;
  a.kept = kept_positions;
  a.first = static_cast<int32_t*>(workspace);
  a.heads = num_kv_heads;
  a.block_bits = block_size == 8 ? 3 : (block_size == 16 ? 4 : 5);
  a.num_blocks = num_blocks;
  a.table_width = max_num_blocks_per_seq;
  a.max_ctx = max_context_len;
  a.budget = budget;
  a.recent = num_recent;
  a.head_size = head_size;
  a.tile_bytes = head_size * block_size * elem_size(dtype);
  a.key_tasks = (head_size / x + 3) / 4;
  a.value_tasks = (head_size + kRows - 1) / kRows;
  const int64_t tasks = cells * (a.key_tasks + a.value_tasks + 1);
  PA_REQUIRE(tasks <= 0x7fffffff, "%s: too many heads for one launch", what);
  hipStream_t st = static_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(pa_evict_select_kernel, dim3((unsigned)cells), dim3(kThreads), 0, st, a);
  PA_CHECK_LAUNCH(what);
  if (max_context_len <= budget) return PA_OK;  // no sequence can lose a position
  const dim3 grid((unsigned)tasks);
  if (elem_size(dtype) == 4)
    hipLaunchKernelGGL((pa_evict_move_kernel<uint32_t, 4>), grid, dim3(64), 0, st, a, a.tables, a.kept, a.first, a.kc, a.vc, a.weights);
  else
    hipLaunchKernelGGL((pa_evict_move_kernel<uint16_t, 8>), grid, dim3(64), 0, st, a, a.tables, a.kept, a.first, a.kc, a.vc, a.weights);
  PA_CHECK_LAUNCH(what);
  return PA_OK;
}
