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
  typedef f32x4 frag;
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
    typename E::frag t;
#pragma unroll
    for (int i = 0; i < E::kX; i++) t[i] = p[i];
    v = __builtin_bit_cast(u32x4, t);
  }
  if (mode == 1) {
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] ^= sizeof(typename E::storage) == 2 ? 0x80008000u : 0x80000000u;
  }
  if (mode == 2) v = u32x4{0, 0, 0, 0};
  return v;
}

// The workgroup's item.  Workgroups that share a (sequence, partition, head) share an XCD and its L2;
// the groups go round the XCDs.
struct Item {
  int seq, part, head, tile;
  bool exists;
};
__device__ __forceinline__ Item tree_item(const TreeArgs& a) {
  const unsigned k8 = blockIdx.x >> 3;
  const unsigned item = (k8 / (unsigned)a.row_tiles) * 8u + (blockIdx.x & 7u);
  Item r;
  r.tile = (int)(k8 % (unsigned)a.row_tiles);
  r.exists = item < (unsigned)a.num_seqs * (unsigned)a.parts * (unsigned)a.num_kv_heads;
  r.head = (int)(item % (unsigned)a.num_kv_heads);
  const unsigned sp = item / (unsigned)a.num_kv_heads;
  r.part = (int)(sp % (unsigned)a.parts);
  r.seq = (int)(sp / (unsigned)a.parts);
  return r;
}

// The rows of a sequence whose arguments contradict each other
template <typename E, int D>
__device__ __forceinline__ void fill_nan(const TreeArgs& a, const TreeSeq& sq, int head) {
  typedef typename E::storage T;
  for (int t = 0; t < sq.queries; t++)
    for (int i = threadIdx.x; i < a.group * D; i += blockDim.x)
      static_cast<T*>(a.out)[((int64_t)(sq.first + t) * a.num_heads + (int64_t)head * a.group) * D + i] = (T)__builtin_nanf("");
}

// RT tiles of 16 rows in one wave: a lane holds row n = lane % 16 of each, as a column of the products
// (the 4 lanes of a row hold the tokens PT g .. PT g + PT - 1 of a step and the elements 16 j + 4 g ..
// of the result).
template <typename E, int D, int RT>
struct Rows {
  typedef typename E::storage T;
  static constexpr int X = E::kX, TS = E::kTokens, KS = (D / X + 3) / 4, NA = TS / 16, NJ = D / 16, PT = 4 * NA;
  u32x4 qf[RT][KS];
  f32x4 o[RT][NJ], l[RT];
  float m[RT], lx[RT];
  int query[RT], row[RT];
  bool valid[RT];

  __device__ __forceinline__ void init(const TreeArgs& a, const TreeSeq& sq, int head, int row0, int lane) {
    const int n = lane & 15, g = lane >> 4;
    const bool aligned = ((reinterpret_cast<uintptr_t>(a.q) | (uintptr_t)(a.q_stride * (int64_t)sizeof(T))) & 15u) == 0;
#pragma unroll
    for (int t = 0; t < RT; t++) {
      row[t] = row0 + t * 16 + n;
      valid[t] = row[t] < sq.rows;
      query[t] = valid[t] ? row[t] / a.group : 0;
      const int hq = valid[t] ? row[t] - query[t] * a.group : 0;
      const T* qp = static_cast<const T*>(a.q) + (int64_t)(sq.first + query[t]) * a.q_stride + (int64_t)(head * a.group + hq) * D;
#pragma unroll
      for (int ks = 0; ks < KS; ks++) {
        const int chunk = ks * 4 + g;
        qf[t][ks] = valid[t] && chunk < D / X ? load_query<E>(qp + chunk * X, aligned, a.q_mode) : u32x4{0, 0, 0, 0};
      }
      m[t] = kNoMax;
      lx[t] = 0.f;
      l[t] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int j = 0; j < NJ; j++) o[t][j] = f32x4{0, 0, 0, 0};
    }
  }

  // Logits to rounded weights, the running maximum and sums kept.  tok: the step's first token.
  __device__ __forceinline__ u32x4 weigh(const TreeArgs& a, const TreeSeq& sq, int t, const f32x4* s, int tok, int g, bool masked,
                                         float* logits) {
    float x[PT];
#pragma unroll
    for (int i = 0; i < PT; i++) x[i] = s[i >> 2][i & 3];
    if (masked) {
      const int free_end = sq.ctx - sq.queries;
#pragma unroll
      for (int i = 0; i < PT; i++) {
        const int pos = tok + PT * g + i, d = pos - free_end;
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
    if (logits != nullptr && valid[t]) {
      float* to = logits + row[t] * a.logit_stride + tok + PT * g;
#pragma unroll
      for (int i = 0; i < PT; i += 4) *reinterpret_cast<f32x4*>(to + i) = f32x4{x[i] * a.c, x[i + 1] * a.c, x[i + 2] * a.c, x[i + 3] * a.c};
    }
#pragma unroll
    for (int i = 0; i < PT; i++) x[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[i], a.c, -m[t]));
    if (logits != nullptr) {
#pragma unroll
      for (int i = 0; i < PT; i++) lx[t] += x[i];
    }
    const u32x4 p = E::pack(x);
    l[t] = E::mma(u32x4{E::kOnes, E::kOnes, E::kOnes, E::kOnes}, p, l[t]);
    return p;
  }

  // One run of 16 elements of the values in a step that ends past what all rows see.  What lies behind the
  // context is nobody's and may be anything: it is taken as 0.  A drafted position may hold infinities or
  // NaN that only the rows that see it must show, and a product with a weight of 0 would hand them to all:
  // such elements are taken out, and put back where the weight is not 0.
  __device__ __forceinline__ u32x4 clean(const TreeSeq& sq, u32x4 v, const u32x4* pf, int j, int tok, int g) {
    v = where<E>(v, [&](int i, uint32_t) { return tok + PT * g + i < sq.ctx; }, v);
    bool odd = false;
#pragma unroll
    for (int i = 0; i < X; i++) odd |= (element<E>(v, i) & E::kInf) == E::kInf;
    if (__builtin_amdgcn_ballot_w64(odd) != 0) {
      const u32x4 ones = u32x4{E::kOnes, E::kOnes, E::kOnes, E::kOnes};
#pragma unroll 1
      for (int kind = 0; kind < 3; kind++) {  // +inf, -inf, NaN
        const float special = kind == 0 ? __builtin_inff() : (kind == 1 ? -__builtin_inff() : __builtin_nanf(""));
        const u32x4 is = where<E>(v, [&](int, uint32_t b) {
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
      v = where<E>(v, [&](int, uint32_t b) { return (b & E::kInf) != E::kInf; }, v);
    }
    return v;
  }

  __device__ __forceinline__ void finish_exact() {
#pragma unroll
    for (int t = 0; t < RT; t++) {
      lx[t] += __shfl_xor(lx[t], 16);
      lx[t] += __shfl_xor(lx[t], 32);
    }
  }
};

// 4 elements from d of a row's sums: the result where the sequence has one partition, else the partition's share
template <typename E, int D>
__device__ __forceinline__ void store_row(const TreeArgs& a, const TreeSeq& sq, const Item& it, int row, int d, f32x4 v, float mx,
                                          float sum, float exact) {
  typedef typename E::storage T;
  if (sq.parts > 1) {
    *reinterpret_cast<f32x4*>(a.acc + tree_row(a, it.seq, it.head, it.part, row) * D + d) = v;
  } else {
    const int qi = row / a.group;
    T* op = static_cast<T*>(a.out) + ((int64_t)(sq.first + qi) * a.num_heads + (int64_t)it.head * a.group + (row - qi * a.group)) * D + d;
    const float inv = sum == 0.f ? 0.f : 1.0f / sum;  // nothing seen: zeros
    typedef T T4 __attribute__((ext_vector_type(4)));
    *reinterpret_cast<T4*>(op) = __builtin_convertvector(v * inv, T4);
  }
  if ((sq.parts > 1 || a.weights != nullptr) && d == 0)
    *reinterpret_cast<f32x4*>(a.ml + tree_row(a, it.seq, it.head, it.part, row) * 4) = f32x4{mx, sum, exact, 0.f};
}

// ---- few rows: the caches go straight into the operands ------------------------------------------------
//
// All 4 waves have the same RT tiles of rows; they take turns at the steps of the context and add up
// through LDS.  A wave holds the keys and the values of one step: the next keys are on their way while
// the weights are made, the next values while the next logits are.
template <typename E, int D, int B, int RT>
__global__ void __launch_bounds__(256, (RT == 1 ? 3 : 2)) pa_tree_few_kernel(const TreeArgs a) {
  typedef typename E::storage T;
  typedef Rows<E, D, RT> R;
  constexpr int X = R::X, TS = R::TS, KS = R::KS, NA = R::NA, NJ = R::NJ, PT = R::PT, WK = 4, ROWS = 16 * RT;
  const Item it = tree_item(a);
  if (!it.exists) return;
  const TreeSeq sq = tree_seq(a, it.seq);
  const int tid = threadIdx.x, lane = tid & 63, wk = __builtin_amdgcn_readfirstlane(tid >> 6);
  if (sq.bad) {
    if (it.part == 0 && it.tile == 0) fill_nan<E, D>(a, sq, it.head);
    return;
  }
  const int row0 = it.tile * ROWS;
  if (row0 >= sq.rows || it.part >= sq.parts) return;
  const int n = lane & 15, g = lane >> 4;
  const int p0 = it.part * a.part_len;
  const int p1 = it.part == sq.parts - 1 ? sq.ctx : p0 + a.part_len;
  const int steps = (p1 - p0 + TS - 1) / TS;
  float* logits = a.weights == nullptr ? nullptr : a.logits + ((int64_t)it.seq * a.num_kv_heads + it.head) * a.max_rows * a.logit_stride;

  R r;
  r.init(a, sq, it.head, row0, lane);

  const int32_t* table = a.tables + (int64_t)it.seq * a.table_width;
  const int last_entry = (sq.ctx - 1) / B;
  const int64_t block_bytes = (int64_t)a.num_kv_heads * D * B * (int)sizeof(T);
  const char* kc = a.kc + (int64_t)it.head * D * B * (int)sizeof(T);
  const char* vc = a.vc + (int64_t)it.head * D * B * (int)sizeof(T);
  // the first of this lane's tokens of a step: on the key side (row m = n) and on the value side
  const int ktok = TS == 32 ? 8 * (n >> 2) + (n & 3) : n;
  const int vtok = PT * g;
  bool bad_block = false;

  struct Ids { int k, v; };
  const auto load_ids = [&](int step) {
    Ids ids;
    const int tok = p0 + step * TS;
    const int ek = (tok + ktok) / B, ev = (tok + vtok) / B;
    ids.k = table[ek < last_entry ? ek : last_entry];
    ids.v = table[ev < last_entry ? ev : last_entry];
    return ids;
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
        if (KS * 4 * X == D || ks < KS - 1 || ks * 4 + g < D / X) kf[i][ks] = load16<true>(base + (i * 4 + ks * 4 * B) * 16);
        else kf[i][ks] = u32x4{0, 0, 0, 0};
      }
  };
  const auto load_v = [&](int b, int step) {
    const char* base = vc + (int64_t)checked(b) * block_bytes + (((p0 + step * TS + vtok) & (B - 1)) + n * B) * (int)sizeof(T);
#pragma unroll
    for (int j = 0; j < NJ; j++) vf[j] = load16<true>(base + j * 16 * B * (int)sizeof(T));
  };

  int step = wk;
  if (step < steps) {
    Ids next = load_ids(step);
    load_k(next.k, step);
    load_v(next.v, step);
    next = load_ids(step + WK < steps ? step + WK : step);
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
          for (int ks = 0; ks < KS; ks++) s[t][i] = E::mma(kf[i][ks], r.qf[t][ks], s[t][i]);
        }
      // the table entries two steps ahead go out before the next keys: waiting for them waits for nothing else
      const Ids after = load_ids(step + 2 * WK < steps ? step + 2 * WK : step);
      if (more) load_k(next.k, step + WK);
      const bool masked = tok + TS > sq.ctx - sq.queries;
      u32x4 pf[RT];
#pragma unroll
      for (int t = 0; t < RT; t++) pf[t] = r.weigh(a, sq, t, s[t], tok, g, masked, logits);
      if (masked) {
#pragma unroll
        for (int j = 0; j < NJ; j++) vf[j] = r.clean(sq, vf[j], pf, j, tok, g);
      }
#pragma unroll
      for (int t = 0; t < RT; t++)
#pragma unroll
        for (int j = 0; j < NJ; j++) r.o[t][j] = E::mma(vf[j], pf[t], r.o[t][j]);
      if (more) load_v(next.v, step + WK);
      next = after;
    }
  }
  // a block number outside the cache: the rows must not pass for a result
  const bool any_bad = __builtin_amdgcn_ballot_w64(bad_block) != 0;
  r.finish_exact();

  // the waves' shares of a row: their maxima first, then the sums at the common scale
  constexpr int ST = D + 4;  // rows of LDS start 4 banks apart
  __shared__ float sm_m[WK][ROWS], sm_l[WK][ROWS], sm_x[WK][ROWS];
  __shared__ __attribute__((aligned(16))) float sm_o[WK][ROWS][ST];
  if (g == 0) {
#pragma unroll
    for (int t = 0; t < RT; t++) sm_m[wk][t * 16 + n] = r.m[t];
  }
  __syncthreads();
#pragma unroll
  for (int t = 0; t < RT; t++) {
    const int row = t * 16 + n;
    float high = sm_m[0][row];
#pragma unroll
    for (int w = 1; w < WK; w++) high = fmaxf(high, sm_m[w][row]);
    const float f = any_bad ? __builtin_nanf("") : __builtin_amdgcn_exp2f(r.m[t] - high);
    if (g == 0) {
      sm_l[wk][row] = r.l[t][0] * f;
      sm_x[wk][row] = r.lx[t] * f;
    }
#pragma unroll
    for (int j = 0; j < NJ; j++) *reinterpret_cast<f32x4*>(&sm_o[wk][row][16 * j + 4 * g]) = r.o[t][j] * f;
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
    store_row<E, D>(a, sq, it, row0 + row, d, v, high, sum, exact);
  }
}

// ---- many rows: a step's keys and values are staged in LDS for all waves -----------------------------------
//
// NW waves of RT tiles each.  A step's operands are KS x NA + D / 16 pieces of 1 KiB, in LDS exactly as the
// products take them (a lane's 16 bytes at 16 * lane: no bank conflicts); wave w fetches pieces w, w + NW, ...
// from the caches at the addresses that the few-rows kernel would use.  Two buffers: while step i is
// consumed, the pieces of i + 1 are in registers or on their way, those of i + 2 are on their way; one
// barrier a step.
template <typename E, int D, int RT, int NW>
__global__ void __launch_bounds__(NW * 64, 2) pa_tree_many_kernel(const TreeArgs a) {
  typedef typename E::storage T;
  typedef Rows<E, D, RT> R;
  constexpr int X = R::X, TS = R::TS, KS = R::KS, NA = R::NA, NJ = R::NJ, PT = R::PT, ROWS = 16 * RT * NW;
  constexpr int PIECES = NA * KS + NJ, F = (PIECES + NW - 1) / NW;
  __shared__ __attribute__((aligned(16))) u32x4 sm[2][PIECES * 64];
  __shared__ int sm_bad;
  const Item it = tree_item(a);
  if (!it.exists) return;
  const TreeSeq sq = tree_seq(a, it.seq);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  if (sq.bad) {
    if (it.part == 0 && it.tile == 0) fill_nan<E, D>(a, sq, it.head);
    return;
  }
  const int row0 = it.tile * ROWS;
  if (row0 >= sq.rows || it.part >= sq.parts) return;
  const int n = lane & 15, g = lane >> 4;
  const int bits = a.block_bits, B = 1 << bits;
  const int p0 = it.part * a.part_len;
  const int p1 = it.part == sq.parts - 1 ? sq.ctx : p0 + a.part_len;
  const int steps = (p1 - p0 + TS - 1) / TS;
  float* logits = a.weights == nullptr ? nullptr : a.logits + ((int64_t)it.seq * a.num_kv_heads + it.head) * a.max_rows * a.logit_stride;
  const bool has_rows = row0 + wave * 16 * RT < sq.rows;
  if (tid == 0) sm_bad = 0;

  R r;
  r.init(a, sq, it.head, row0 + wave * 16 * RT, lane);

  const int32_t* table = a.tables + (int64_t)it.seq * a.table_width;
  const int last_entry = (sq.ctx - 1) >> bits;
  const int64_t block_bytes = (int64_t)a.num_kv_heads * D * B * (int)sizeof(T);
  const char* kc = a.kc + (int64_t)it.head * D * B * (int)sizeof(T);
  const char* vc = a.vc + (int64_t)it.head * D * B * (int)sizeof(T);
  const int ktok = TS == 32 ? 8 * (n >> 2) + (n & 3) : n;
  const int vtok = PT * g;
  bool bad_block = false;

  struct Ids { int k, v; };
  const auto load_ids = [&](int step) {
    Ids ids;
    const int tok = p0 + step * TS;
    const int ek = (tok + ktok) >> bits, ev = (tok + vtok) >> bits;
    ids.k = table[ek < last_entry ? ek : last_entry];
    ids.v = table[ev < last_entry ? ev : last_entry];
    return ids;
  };
  const auto checked = [&](int b) {
    const bool ok = (unsigned)b < (unsigned)a.num_blocks;
    bad_block |= !ok;
    return ok ? b : 0;
  };
  const auto fetch = [&](u32x4* v, Ids ids, int step) {
    const int tok = p0 + step * TS;
    const char* kb = kc + (int64_t)checked(ids.k) * block_bytes + (((tok + ktok) & (B - 1)) + g * B) * 16;
    const char* vb = vc + (int64_t)checked(ids.v) * block_bytes + (((tok + vtok) & (B - 1)) + n * B) * (int)sizeof(T);
#pragma unroll
    for (int f = 0; f < F; f++) {
      const int piece = wave + f * NW;  // the same for the whole wave
      v[f] = u32x4{0, 0, 0, 0};
      if (piece < NA * KS) {
        const int i = piece / KS, ks = piece - i * KS;
        if (KS * 4 * X == D || ks * 4 + g < D / X) v[f] = load16<false>(kb + (i * 4 + ks * 4 * B) * 16);
      } else if (piece < PIECES) {
        v[f] = load16<false>(vb + (piece - NA * KS) * 16 * B * (int)sizeof(T));
      }
    }
  };
  const auto put = [&](const u32x4* v, int buffer) {
#pragma unroll
    for (int f = 0; f < F; f++)
      if (wave + f * NW < PIECES) sm[buffer][(wave + f * NW) * 64 + lane] = v[f];
  };
  const auto consume = [&](int step, const u32x4* buf) {
    if (!has_rows) return;
    const int tok = p0 + step * TS;
    f32x4 s[RT][NA];
#pragma unroll
    for (int t = 0; t < RT; t++)
#pragma unroll
      for (int i = 0; i < NA; i++) s[t][i] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < NA; i++)
#pragma unroll
      for (int ks = 0; ks < KS; ks++) {
        const u32x4 k = buf[(i * KS + ks) * 64 + lane];
#pragma unroll
        for (int t = 0; t < RT; t++) s[t][i] = E::mma(k, r.qf[t][ks], s[t][i]);
      }
    const bool masked = tok + TS > sq.ctx - sq.queries;
    u32x4 pf[RT];
#pragma unroll
    for (int t = 0; t < RT; t++) pf[t] = r.weigh(a, sq, t, s[t], tok, g, masked, logits);
#pragma unroll
    for (int j = 0; j < NJ; j++) {
      u32x4 v = buf[(NA * KS + j) * 64 + lane];
      if (masked) v = r.clean(sq, v, pf, j, tok, g);
#pragma unroll
      for (int t = 0; t < RT; t++) r.o[t][j] = E::mma(v, pf[t], r.o[t][j]);
    }
  };

  // step i's pieces pass through held[i & 1]; a step past the last is the last again
  const auto clamp = [&](int step) { return step < steps ? step : steps - 1; };
  u32x4 held[2][F];
  Ids ids = load_ids(0);
  fetch(held[0], ids, 0);
  ids = load_ids(clamp(1));
  Ids after = load_ids(clamp(2));
  fetch(held[1], ids, clamp(1));
  put(held[0], 0);
  __syncthreads();
  const auto turn = [&](int step, int parity) {
    ids = after;
    after = load_ids(clamp(step + 3));
    fetch(held[parity], ids, clamp(step + 2));
    consume(step, sm[parity]);
    put(held[1 - parity], 1 - parity);
    __syncthreads();
  };
  for (int step = 0; step < steps; step += 2) {
    turn(step, 0);
    if (step + 1 < steps) turn(step + 1, 1);
  }
  if (bad_block) sm_bad = 1;
  __syncthreads();
  const bool any_bad = sm_bad != 0;
  r.finish_exact();
#pragma unroll
  for (int t = 0; t < RT; t++)
    if (r.valid[t]) {
      const float sum = any_bad ? __builtin_nanf("") : r.l[t][0], exact = any_bad ? __builtin_nanf("") : r.lx[t];
#pragma unroll
      for (int j = 0; j < NJ; j++) store_row<E, D>(a, sq, it, r.row[t], 16 * j + 4 * g, r.o[t][j], r.m[t], sum, exact);
    }
}

template <typename E, int D>
static void tree_pick_form(const TreeArgs& a, unsigned grid, hipStream_t st) {
  const int form = tree_form(a.max_rows);
  if (form == kTreeMany64) hipLaunchKernelGGL((pa_tree_many_kernel<E, D, 1, 4>), dim3(grid), dim3(256), 0, st, a);
  else if (form == kTreeMany128) hipLaunchKernelGGL((pa_tree_many_kernel<E, D, 2, 4>), dim3(grid), dim3(256), 0, st, a);
  else if (form == kTreeMany256) hipLaunchKernelGGL((pa_tree_many_kernel<E, D, 2, 8>), dim3(grid), dim3(512), 0, st, a);
  else {
#define PA_TREE_FEW(B)                                                                                                   \
  do {                                                                                                                   \
    if (form == kTreeFew16) hipLaunchKernelGGL((pa_tree_few_kernel<E, D, B, 1>), dim3(grid), dim3(256), 0, st, a);       \
    else hipLaunchKernelGGL((pa_tree_few_kernel<E, D, B, 2>), dim3(grid), dim3(256), 0, st, a);                          \
  } while (0)
    if (a.block_bits == 3) PA_TREE_FEW(8);
    else if (a.block_bits == 4) PA_TREE_FEW(16);
    else PA_TREE_FEW(32);
#undef PA_TREE_FEW
  }
}

template <typename E>
static int tree_launch(const TreeArgs& a, int head_size, unsigned grid, hipStream_t st) {
  switch (head_size) {
    case 64: tree_pick_form<E, 64>(a, grid, st); break;
    case 80: tree_pick_form<E, 80>(a, grid, st); break;
    case 96: tree_pick_form<E, 96>(a, grid, st); break;
    default: tree_pick_form<E, 128>(a, grid, st); break;
  }
  PA_CHECK_LAUNCH("cached attention of several queries");
  return PA_OK;
}

}  // namespace tree
}  // namespace pa
