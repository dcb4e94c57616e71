// Attention of several new tokens per sequence (a tree of drafted tokens, a
// chain, or one) over the paged cache, on the matrix cores of gfx950.
//
//   out[t] = sum_j softmax_j(scale q_t . k_j) v_j  over j < ctx - T and the drafted
//            positions ctx - T + i that mask[t][i] (or i <= t) lets t see
//
// The rows of a (sequence, kv head) are its T queries times the query heads that
// share the head.  Both caches are read in the order that memory has, straight
// into the operands of v_mfma_f32_16x16x32 (16 bit) / 16x16x4 (fp32), without LDS:
//   S^T = K . Q^T   a key block is [head_size / x][block][x], x elements = 16 bytes:
//                   a lane's 16-byte load of (token, chunk) is its share of the A operand;
//   O^T += V^T . P^T  a value block is [head_size][block]: a lane's 16-byte load of
//                   8 tokens of one row is its share of the A operand, and the S^T
//                   accumulator, rounded to the type, is the B operand as it stands
//                   once token 8 (m / 4) + 4 a + m % 4 sits in row m of the a-th of
//                   two products (16 bit; fp32 needs no such order).
// A row's running maximum is raised only when a logit exceeds it by 2^8 (the
// weights then reach 2^8, which fp32 sums and both 16-bit types hold), so that
// lanes exchange nothing in the common step: l and O keep to one scale anyway.
// The sum of the weights is a product with a row of ones: it adds up what the
// rounded weights really were.  fp16 weights carry a factor 2^6, so that one of
// 2^-20 of the row's largest still has all its bits.
#pragma once

#include "pa_tree.h"

namespace pa {
namespace tree {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr float kNoMax = -1e30f;   // below every logit, and finite: exp2(-inf - kNoMax) = 0
constexpr float kMaxSlack = 8.f;   // how far a logit may exceed the running maximum

struct F16 {
  typedef _Float16 storage;
  typedef f16x8 frag;
  static constexpr int kX = 8, kTokens = 32;
  static constexpr float kBias = 6.f;
  static __device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(frag, a), __builtin_bit_cast(frag, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ u32x4 pack(const float* p) {
    frag f;
#pragma unroll
    for (int i = 0; i < 8; i++) f[i] = (_Float16)p[i];
    return __builtin_bit_cast(u32x4, f);
  }
  static constexpr uint32_t kOnes = 0x3c003c00u, kInf = 0x7c00u, kSign = 0x8000u;
};

struct BF16 {
  typedef __bf16 storage;
  typedef bf16x8 frag;
  static constexpr int kX = 8, kTokens = 32;
  static constexpr float kBias = 0.f;
  static __device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(frag, a), __builtin_bit_cast(frag, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ u32x4 pack(const float* p) {
    frag f;
#pragma unroll
    for (int i = 0; i < 8; i++) f[i] = (__bf16)p[i];
    return __builtin_bit_cast(u32x4, f);
  }
  static constexpr uint32_t kOnes = 0x3f803f80u, kInf = 0x7f80u, kSign = 0x8000u;
};

// One 16-byte load holds 4 elements: a product of 16 x 16 x 16 is four instructions, each with one
// element of every lane's vectors (the order of the sum's index is the same on both sides).
struct F32 {
  typedef float storage;
  static constexpr int kX = 4, kTokens = 16;
  static constexpr float kBias = 0.f;
  static __device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
#pragma unroll
    for (int i = 0; i < 4; i++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[i]), __uint_as_float(b[i]), c, 0, 0, 0);
    return c;
  }
  static __device__ __forceinline__ u32x4 pack(const float* p) {
    return u32x4{__float_as_uint(p[0]), __float_as_uint(p[1]), __float_as_uint(p[2]), __float_as_uint(p[3])};
  }
  static constexpr uint32_t kOnes = 0x3f800000u, kInf = 0x7f800000u, kSign = 0x80000000u;
};

// element i of a vector of kX, as its bits
template <typename E> __device__ __forceinline__ uint32_t element(u32x4 v, int i) {
  if (sizeof(typename E::storage) == 4) return v[i];
  return (v[i >> 1] >> (16 * (i & 1))) & 0xffffu;
}

// `with` in the places (16 or 32 bits) whose bits in v the predicate picks, 0 elsewhere
template <typename E, typename F> __device__ __forceinline__ u32x4 where(u32x4 v, F pick, u32x4 with) {
  u32x4 r;
  if (sizeof(typename E::storage) == 4) {
#pragma unroll
    for (int i = 0; i < 4; i++) r[i] = pick(i, v[i]) ? with[i] : 0u;
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++)
      r[i] = (pick(2 * i, v[i] & 0xffffu) ? with[i] & 0xffffu : 0u) | (pick(2 * i + 1, v[i] >> 16) ? with[i] & 0xffff0000u : 0u);
  }
  return r;
}

template <bool STREAM> __device__ __forceinline__ u32x4 load16(const char* p) {
  if (STREAM) return __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p));
  return *reinterpret_cast<const u32x4*>(p);
}

// x elements of a query row from element `at`, whatever its alignment
template <typename E> __device__ __forceinline__ u32x4 load_query(const typename E::storage* p, bool aligned, int mode) {
  u32x4 v;
  if (aligned) {
    v = *reinterpret_cast<const u32x4*>(p);
  } else {
    typename E::storage t[E::kX];
#pragma unroll
    for (int i = 0; i < E::kX; i++) t[i] = p[i];
    __builtin_memcpy(&v, t, 16);
  }
  if (mode == 1) {
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] ^= sizeof(typename E::storage) == 2 ? 0x80008000u : 0x80000000u;
  }
  if (mode == 2) v = u32x4{0, 0, 0, 0};
  return v;
}

// RT: 16-row tiles of a wave.  WR: waves along the rows; the other 4 / WR take turns at the steps of
// the context and add up through LDS.  ACC: the logits are kept for the weight cache.
template <typename E, int D, int RT, int WR, bool ACC>
__global__ void __launch_bounds__(256) pa_tree_kernel(const TreeArgs a) {
  typedef typename E::storage T;
  constexpr int X = E::kX, TS = E::kTokens, WK = 4 / WR;
  constexpr int KS = (D / X + 3) / 4;       // products over the head size: 4 chunks of x at a time
  constexpr int NA = TS / 16;               // 16-token products of a step
  constexpr int NJ = D / 16;
  constexpr int PT = 4 * NA;                // tokens of a step in one lane
  constexpr int ROWS = 16 * RT * WR;
  constexpr bool STREAM = WR == 1;          // else waves of a workgroup and its neighbours read the same blocks
  static_assert(D % 16 == 0, "head size");

  // Workgroups that share a (sequence, partition, head) share an XCD and its L2; the groups go round the XCDs.
  const unsigned id = blockIdx.x;
  const unsigned k8 = id >> 3;
  const unsigned item = (k8 / (unsigned)a.row_tiles) * 8u + (id & 7u);
  const int tile = (int)(k8 % (unsigned)a.row_tiles);
  const unsigned items = (unsigned)a.num_seqs * (unsigned)a.parts * (unsigned)a.num_kv_heads;
  if (item >= items) return;
  const int head = (int)(item % (unsigned)a.num_kv_heads);
  const unsigned sp = item / (unsigned)a.num_kv_heads;
  const int part = (int)(sp % (unsigned)a.parts), seq = (int)(sp / (unsigned)a.parts);

  const TreeSeq sq = tree_seq(a, seq);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  if (sq.bad) {
    if (part == 0 && tile == 0) {
      const uint32_t nan = sizeof(T) == 4 ? 0x7fc00000u : (E::kInf == 0x7c00u ? 0x7e00u : 0x7fc0u);
      for (int t = 0; t < sq.queries; t++)
        for (int i = tid; i < a.group * D; i += 256) {
          const int64_t at = ((int64_t)(sq.first + t) * a.num_heads + (int64_t)head * a.group) * D + i;
          if (sizeof(T) == 4) static_cast<uint32_t*>(a.out)[at] = nan;
          else static_cast<uint16_t*>(a.out)[at] = (uint16_t)nan;
        }
    }
    return;
  }
  const int row0 = tile * ROWS;
  if (row0 >= sq.rows || part >= sq.parts) return;

  const int wr = wave % WR, wk = wave / WR;
  const int n = lane & 15, g = lane >> 4;
  const int B = 1 << a.block_bits;
  const int p0 = part * a.part_len;
  const int p1 = part == sq.parts - 1 ? sq.ctx : p0 + a.part_len;
  const int steps = (p1 - p0 + TS - 1) / TS;
  const int seen_by_all = sq.ctx - sq.queries;

  // this lane's rows, one of each tile
  int query[RT], hq[RT];
  bool valid[RT];
  u32x4 qf[RT][KS];
#pragma unroll
  for (int t = 0; t < RT; t++) {
    const int r = row0 + (wr * RT + t) * 16 + n;
    valid[t] = r < sq.rows;
    query[t] = valid[t] ? r / a.group : 0;
    hq[t] = valid[t] ? r - query[t] * a.group : 0;
    const T* qp = static_cast<const T*>(a.q) + (int64_t)(sq.first + query[t]) * a.q_stride + (int64_t)(head * a.group + hq[t]) * D;
    const bool aligned = ((reinterpret_cast<uintptr_t>(a.q) | (uintptr_t)(a.q_stride * (int64_t)sizeof(T))) & 15u) == 0;
#pragma unroll
    for (int ks = 0; ks < KS; ks++) {
      const int chunk = ks * 4 + g;
      qf[t][ks] = valid[t] && chunk < D / X ? load_query<E>(qp + chunk * X, aligned, a.q_mode) : u32x4{0, 0, 0, 0};
    }
  }

  f32x4 o[RT][NJ], l[RT];
  float m[RT], lx[RT];
#pragma unroll
  for (int t = 0; t < RT; t++) {
    m[t] = kNoMax;
    lx[t] = 0.f;
    l[t] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < NJ; j++) o[t][j] = f32x4{0, 0, 0, 0};
  }
  const u32x4 ones = u32x4{E::kOnes, E::kOnes, E::kOnes, E::kOnes};

  const int32_t* table = a.tables + (int64_t)seq * a.table_width;
  const int last_entry = (sq.ctx - 1) >> a.block_bits;
  const int64_t block_bytes = (int64_t)a.num_kv_heads * D * B * (int)sizeof(T);
  const char* kc = a.kc + (int64_t)head * D * B * (int)sizeof(T);
  const char* vc = a.vc + (int64_t)head * D * B * (int)sizeof(T);
  // the first of this lane's tokens of a step: on the key side (row m = n) and on the value side
  const int ktok = TS == 32 ? 8 * (n >> 2) + (n & 3) : n;
  const int vtok = PT * g;
  bool bad_block = false;

  struct Ids { int k, v; };
  const auto load_ids = [&](int step) {
    Ids r;
    const int tok = p0 + step * TS;
    int ek = (tok + ktok) >> a.block_bits, ev = (tok + vtok) >> a.block_bits;
    ek = ek < last_entry ? ek : last_entry;
    ev = ev < last_entry ? ev : last_entry;
    r.k = table[ek];
    r.v = table[ev];
    return r;
  };
  const auto checked = [&](int b) {
    const bool ok = (unsigned)b < (unsigned)a.num_blocks;
    bad_block |= !ok;
    return ok ? b : 0;
  };
  u32x4 kf[NA][KS], vf[NJ];
  const auto load_k = [&](int b, int step) {
    const char* base = kc + (int64_t)checked(b) * block_bytes + (((p0 + step * TS + ktok) & (B - 1)) + g * B) * 16;
#pragma unroll
    for (int i = 0; i < NA; i++)
#pragma unroll
      for (int ks = 0; ks < KS; ks++) {
        if (KS * 4 * X == D || ks < KS - 1 || ks * 4 + g < D / X) kf[i][ks] = load16<STREAM>(base + (i * 4 + ks * 4 * B) * 16);
        else kf[i][ks] = u32x4{0, 0, 0, 0};
      }
  };
  const auto load_v = [&](int b, int step) {
    const char* base = vc + (int64_t)checked(b) * block_bytes + (((p0 + step * TS + vtok) & (B - 1)) + n * B) * (int)sizeof(T);
#pragma unroll
    for (int j = 0; j < NJ; j++) vf[j] = load16<STREAM>(base + (int64_t)j * 16 * B * (int)sizeof(T));
  };

  int step = wk;
  if (step < steps) {
    Ids now = load_ids(step);
    Ids next = load_ids(step + WK < steps ? step + WK : step);
    load_k(now.k, step);
    load_v(now.v, step);
    for (; step < steps; step += WK) {
      const bool more = step + WK < steps;
      const int tok = p0 + step * TS;
      f32x4 s[RT][NA];
#pragma unroll
      for (int t = 0; t < RT; t++)
#pragma unroll
        for (int i = 0; i < NA; i++) {
          s[t][i] = f32x4{0, 0, 0, 0};
#pragma unroll
          for (int ks = 0; ks < KS; ks++) s[t][i] = E::mma(kf[i][ks], qf[t][ks], s[t][i]);
        }
      // the table entries two steps ahead go out before the next keys: waiting for them waits for nothing else
      const Ids after = load_ids(step + 2 * WK < steps ? step + 2 * WK : step);
      if (more) load_k(next.k, step + WK);

      const bool masked = tok + TS > seen_by_all;
      u32x4 pf[RT];
#pragma unroll
      for (int t = 0; t < RT; t++) {
        float x[PT];
#pragma unroll
        for (int i = 0; i < PT; i++) x[i] = s[t][i >> 2][i & 3];
        if (masked) {
#pragma unroll
          for (int i = 0; i < PT; i++) {
            const int pos = tok + vtok + i, d = pos - seen_by_all;
            bool sees = pos < sq.ctx;
            if (sees && d >= 0)
              sees = a.mask == nullptr ? d <= query[t] : a.mask[(int64_t)(sq.first + query[t]) * a.mask_stride + d] != 0;
            if (!sees) x[i] = -__builtin_inff();
          }
        }
        float top = x[0];
#pragma unroll
        for (int i = 1; i < PT; i++) top = fmaxf(top, x[i]);
        top *= a.c;
        if (__builtin_amdgcn_ballot_w64(top > m[t] + (E::kBias + kMaxSlack)) != 0) {
          float high = fmaxf(m[t], top - E::kBias);
          high = fmaxf(high, __shfl_xor(high, 16));
          high = fmaxf(high, __shfl_xor(high, 32));
          const float f = __builtin_amdgcn_exp2f(m[t] - high);
          m[t] = high;
          lx[t] *= f;
          l[t] *= f;
#pragma unroll
          for (int j = 0; j < NJ; j++) o[t][j] *= f;
        }
        if (ACC && valid[t]) {
          float* lg = a.logits + (((int64_t)seq * a.num_kv_heads + head) * a.max_rows + row0 + (wr * RT + t) * 16 + n) * a.logit_stride + tok + vtok;
#pragma unroll
          for (int i = 0; i < PT; i += 4) *reinterpret_cast<f32x4*>(lg + i) = f32x4{x[i] * a.c, x[i + 1] * a.c, x[i + 2] * a.c, x[i + 3] * a.c};
        }
#pragma unroll
        for (int i = 0; i < PT; i++) x[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[i], a.c, -m[t]));
        if (ACC) {
#pragma unroll
          for (int i = 0; i < PT; i++) lx[t] += x[i];
        }
        pf[t] = E::pack(x);
        l[t] = E::mma(ones, pf[t], l[t]);
      }

      if (masked) {
        // What lies behind the context is nobody's and may be anything: it is taken as 0.  A drafted
        // position may hold infinities or NaN that only the rows that see it must show, and a product
        // with a weight of 0 would hand them to all: such elements are taken out, and put back where
        // the weight is not 0.
        bool odd = false;
#pragma unroll
        for (int j = 0; j < NJ; j++) {
          vf[j] = where<E>(vf[j], [&](int i, uint32_t) { return tok + vtok + i < sq.ctx; }, vf[j]);
#pragma unroll
          for (int i = 0; i < X; i++) odd |= (element<E>(vf[j], i) & E::kInf) == E::kInf;
        }
        if (__builtin_amdgcn_ballot_w64(odd) != 0) {
#pragma unroll 1
          for (int kind = 0; kind < 3; kind++) {  // +inf, -inf, NaN
            const float special = kind == 0 ? __builtin_inff() : (kind == 1 ? -__builtin_inff() : __builtin_nanf(""));
#pragma unroll
            for (int j = 0; j < NJ; j++) {
              const u32x4 is = where<E>(vf[j], [&](int, uint32_t b) {
                if (kind == 0) return b == E::kInf;
                if (kind == 1) return b == (E::kInf | E::kSign);
                return (b & (E::kSign - 1u)) > E::kInf;
              }, ones);
#pragma unroll
              for (int t = 0; t < RT; t++) {
                const f32x4 hit = E::mma(is, pf[t], f32x4{0, 0, 0, 0});
#pragma unroll
                for (int i = 0; i < 4; i++) o[t][j][i] += hit[i] > 0.f ? special : 0.f;
              }
            }
          }
#pragma unroll
          for (int j = 0; j < NJ; j++)
            vf[j] = where<E>(vf[j], [&](int, uint32_t b) { return (b & E::kInf) != E::kInf; }, vf[j]);
        }
      }
#pragma unroll
      for (int t = 0; t < RT; t++)
#pragma unroll
        for (int j = 0; j < NJ; j++) o[t][j] = E::mma(vf[j], pf[t], o[t][j]);
      if (more) load_v(next.v, step + WK);
      next = after;
    }
  }

  // A block number outside the cache: the row must not pass for a result.
  const bool any_bad = __builtin_amdgcn_ballot_w64(bad_block) != 0;
  if (ACC) {
#pragma unroll
    for (int t = 0; t < RT; t++) {
      lx[t] += __shfl_xor(lx[t], 16);
      lx[t] += __shfl_xor(lx[t], 32);
    }
  }
  float lsum[RT];
#pragma unroll
  for (int t = 0; t < RT; t++) lsum[t] = any_bad ? __builtin_nanf("") : l[t][0];

  const auto finish = [&](int row, int d, f32x4 v, float mx, float sum, float exact) {  // row: of the workgroup; 4 elements from d
    const int r = row0 + row;
    if (a.parts > 1) {
      *reinterpret_cast<f32x4*>(a.acc + tree_row(a, seq, head, part, r) * D + d) = v;
    } else {
      const int qi = r / a.group;
      T* op = static_cast<T*>(a.out) + ((int64_t)(sq.first + qi) * a.num_heads + (int64_t)head * a.group + (r - qi * a.group)) * D + d;
      const float inv = sum == 0.f ? 0.f : 1.0f / sum;  // nothing seen: zeros
      T res[4];
#pragma unroll
      for (int i = 0; i < 4; i++) res[i] = (T)(v[i] * inv);
      __builtin_memcpy(__builtin_assume_aligned(op, 4 * sizeof(T)), res, sizeof(res));
    }
    if ((a.parts > 1 || ACC) && d == 0)
      *reinterpret_cast<f32x4*>(a.ml + tree_row(a, seq, head, part, r) * 4) = f32x4{mx, sum, exact, 0.f};
  };

  if (WK == 1) {
#pragma unroll
    for (int t = 0; t < RT; t++)
      if (valid[t]) {
#pragma unroll
        for (int j = 0; j < NJ; j++) finish((wr * RT + t) * 16 + n, 16 * j + 4 * g, o[t][j], m[t], lsum[t], any_bad ? lsum[t] : lx[t]);
      }
    return;
  }
  // the waves' shares of a row: their maxima first, then the sums at the common scale
  constexpr int ST = D + 4;  // rows of LDS start 4 banks apart
  __shared__ float sm_m[WK][ROWS], sm_l[WK][ROWS], sm_x[WK][ROWS];
  __shared__ __attribute__((aligned(16))) float sm_o[WK][ROWS][WK == 1 ? 4 : ST];
  if (g == 0) {
#pragma unroll
    for (int t = 0; t < RT; t++) sm_m[wk][(wr * RT + t) * 16 + n] = m[t];
  }
  __syncthreads();
#pragma unroll
  for (int t = 0; t < RT; t++) {
    const int row = (wr * RT + t) * 16 + n;
    float high = sm_m[0][row];
#pragma unroll
    for (int w = 1; w < WK; w++) high = fmaxf(high, sm_m[w][row]);
    const float f = __builtin_amdgcn_exp2f(m[t] - high);
    if (g == 0) {
      sm_l[wk][row] = lsum[t] * f;
      sm_x[wk][row] = (any_bad ? lsum[t] : lx[t]) * f;
    }
#pragma unroll
    for (int j = 0; j < NJ; j++) *reinterpret_cast<f32x4*>(&sm_o[wk][row][16 * j + 4 * g]) = o[t][j] * f;
  }
  __syncthreads();
  for (int i = tid; i < ROWS * (D / 4); i += 256) {
    const int row = i / (D / 4), d = (i - row * (D / 4)) * 4;
    if (row0 + row >= sq.rows) break;
    f32x4 v = *reinterpret_cast<const f32x4*>(&sm_o[0][row][d]);
    float high = sm_m[0][row], sum = sm_l[0][row], exact = sm_x[0][row];
#pragma unroll
    for (int w = 1; w < WK; w++) {
      v += *reinterpret_cast<const f32x4*>(&sm_o[w][row][d]);
      high = fmaxf(high, sm_m[w][row]);
      sum += sm_l[w][row];
      exact += sm_x[w][row];
    }
    finish(row, d, v, high, sum, exact);
  }
}

template <typename E, int D, bool ACC>
static void tree_pick_form(const TreeArgs& a, unsigned grid, hipStream_t st) {
  const TreeForm f = tree_form(a.max_rows);
  if (f.row_tiles_per_wave == 1) hipLaunchKernelGGL((pa_tree_kernel<E, D, 1, 1, ACC>), dim3(grid), dim3(256), 0, st, a);
  else if (f.row_waves == 1) hipLaunchKernelGGL((pa_tree_kernel<E, D, 2, 1, ACC>), dim3(grid), dim3(256), 0, st, a);
  else if (f.row_waves == 2) hipLaunchKernelGGL((pa_tree_kernel<E, D, 2, 2, ACC>), dim3(grid), dim3(256), 0, st, a);
  else hipLaunchKernelGGL((pa_tree_kernel<E, D, 2, 4, ACC>), dim3(grid), dim3(256), 0, st, a);
}

template <typename E>
static int tree_launch(const TreeArgs& a, int head_size, unsigned grid, hipStream_t st) {
  const bool acc = a.weights != nullptr;
  switch (head_size) {
    case 64: acc ? tree_pick_form<E, 64, true>(a, grid, st) : tree_pick_form<E, 64, false>(a, grid, st); break;
    case 80: acc ? tree_pick_form<E, 80, true>(a, grid, st) : tree_pick_form<E, 80, false>(a, grid, st); break;
    case 96: acc ? tree_pick_form<E, 96, true>(a, grid, st) : tree_pick_form<E, 96, false>(a, grid, st); break;
    default: acc ? tree_pick_form<E, 128, true>(a, grid, st) : tree_pick_form<E, 128, false>(a, grid, st); break;
  }
  PA_CHECK_LAUNCH("cached attention of several queries");
  return PA_OK;
}

}  // namespace tree
}  // namespace pa
