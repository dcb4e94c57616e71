// Attention of several new tokens per sequence (a tree of drafted tokens, a
// chain, or one) over the paged cache, on the matrix cores of gfx950.
//
//   out[t] = sum_j softmax_j(scale q_t . k_j) v_j  over j < ctx - T and the drafted
//            positions ctx - T + i that mask[t][i] (or i <= t) lets t see
//
// The rows of a (sequence, kv head) are its T queries times the query heads that
// share the head.  Both caches are read in the order that memory has, which is
// that of the operands of v_mfma_f32_16x16x32 (16 bit) / 16x16x4 (fp32): straight
// into them where rows are few, through LDS as they are where all waves share a step:
//   S^T = K . Q^T   a key block is [head_size / x][block][x], x elements = 16 bytes:
//                   a lane's 16-byte load of (token, chunk) is its share of the A operand;
//   O^T += V^T . P^T  a value block is [head_size][block]: a lane's 16-byte load of
//                   8 tokens of one row is its share of the A operand, and the S^T
//                   accumulator, rounded to the type, is the B operand as it stands
//                   once token 8 (m / 4) + 4 a + m % 4 sits in row m of the a-th of
//                   two products (16 bit; fp32 needs no such order).
// A row's running maximum is raised only when a logit, in base 2, exceeds it by 8,
// so that lanes exchange nothing in the common step: l and O keep to one scale
// anyway.  Weights then reach 2^8, and in fp16, where they carry a factor 2^6 so
// that one of 2^-20 of the row's largest still has all its bits, 2^14 of the 65504
// that the type holds.  They are rounded to the type, as a matrix product takes
// operands of one type: off by half a step each, out by at most that of sum p |v|
// and of itself (seen: 0.0003 in fp16 and 0.0023 in bf16 of the outputs' size, with
// weights of fp32 0.0002 and 0.0017).  The sum of the weights is a product with a
// row of ones: it adds up what the rounded weights really were.
#pragma once

#include <type_traits>

#include "pa_tree.h"

namespace pa {
namespace tree {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr float kNoMax = -3.402823466e38f;  // below every logit, and finite: exp2(-inf - kNoMax) = 0
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
  static constexpr uint32_t kOnes = 0x3c003c00u, kExponent = 0x7c007c00u, kLow = 0x04000400u, kSign = 0x80008000u;
  static constexpr int kToSign = 5;  // from an exponent's lowest bit to the sign's
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
  static constexpr uint32_t kOnes = 0x3f803f80u, kExponent = 0x7f807f80u, kLow = 0x00800080u, kSign = 0x80008000u;
  static constexpr int kToSign = 8;
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
  static constexpr uint32_t kOnes = 0x3f800000u, kExponent = 0x7f800000u, kLow = 0x00800000u, kSign = 0x80000000u;
  static constexpr int kToSign = 8;
};

// The elements of one word that are infinite or NaN, by their sign bits: an exponent of all ones carries
// into the sign's place.  Whole numbers only: compares would need a pair of scalar registers each, and
// steps that are seldom taken must not weigh on the loop around them.
template <typename E> __device__ __forceinline__ uint32_t odd_signs(uint32_t w) { return ((w & E::kExponent) + E::kLow) & E::kSign; }
// of those, the NaN: their other bits, plus all ones, carry into the exponent's lowest place
template <typename E> __device__ __forceinline__ uint32_t nan_signs(uint32_t w) {
  const uint32_t rest = ~(E::kExponent | E::kSign);
  return ((((w & rest) + rest) & E::kLow) << E::kToSign) & odd_signs<E>(w);
}
// sign bits to all bits of their elements
template <typename E> __device__ __forceinline__ uint32_t whole(uint32_t signs) {
  return sizeof(typename E::storage) == 4 ? (uint32_t)((int32_t)signs >> 31) : (signs >> 15) * 0xffffu;
}

// v with only its first `count` elements (0 .. x) kept
template <typename E> __device__ __forceinline__ u32x4 first_elements(u32x4 v, int count) {
  u32x4 r;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    if (sizeof(typename E::storage) == 4) r[i] = i < count ? v[i] : 0u;
    else r[i] = 2 * i + 1 < count ? v[i] : (2 * i < count ? v[i] & 0xffffu : 0u);
  }
  return r;
}

template <bool STREAM> __device__ __forceinline__ u32x4 load16(const char* p) {
  if (STREAM) return __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p));
  return *reinterpret_cast<const u32x4*>(p);
}

// x elements of a query row
template <typename E> __device__ __forceinline__ u32x4 load_query(const typename E::storage* p, bool aligned) {
  if (aligned) return *reinterpret_cast<const u32x4*>(p);
  typename E::frag t;
#pragma unroll
  for (int i = 0; i < E::kX; i++) t[i] = p[i];
  return __builtin_bit_cast(u32x4, t);
}

// A barrier that orders LDS alone: __syncthreads() would wait for the loads that are on their way, too.
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// Until the last product's result can be read (8 and 10 instructions' time).  Before a branch that the results are
// used behind: where a short way and a long one meet again, the compiler was seen to count its waits along the long
// one alone, and along the short one the first element read was an old one.
template <typename E> __device__ __forceinline__ void settle() {
  __builtin_amdgcn_sched_barrier(0);
  if (sizeof(typename E::storage) == 4) asm volatile("s_nop 9");
  else asm volatile("s_nop 7");
  __builtin_amdgcn_sched_barrier(0);
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

// The steps of a partition, and those at its start that all of a workgroup's rows see: in a chain a row sees up
// to itself, so later positions are left out (not where every row's logits are kept) and earlier ones are open.
struct Span { int steps, open_steps; };
template <bool KEEP>
__device__ __forceinline__ Span tree_span(const TreeArgs& a, const TreeSeq& sq, int row0, int rows, int p0, int p1, int step) {
  const int shared = sq.ctx - sq.queries;
  int end = p1, open = shared;
  if (a.mask == nullptr) {
    const int last = (row0 + rows < sq.rows ? row0 + rows : sq.rows) - 1;
    const int reach = shared + last / a.group + 1;
    if (!KEEP && reach < end) end = reach;
    open = shared + row0 / a.group + 1;
  }
  Span r;
  r.steps = end > p0 ? (end - p0 + step - 1) / step : 0;
  r.open_steps = open > p0 ? (open - p0) / step : 0;
  if (r.open_steps > r.steps) r.open_steps = r.steps;
  return r;
}

// The sequence that stands `place`-th by falling length of its partitions, those alike in their order.  Workgroups
// are dealt out in the order of their items: with the longest first, a CU that is done early takes up a shorter one,
// and no long one is left to run alone at the end.
__device__ __forceinline__ int by_length(const TreeArgs& a, int place, int* len, int* found) {
  const int t = threadIdx.x, n = a.num_seqs;
  int mine = -1;
  if (t < n) {
    const int ctx = a.ctx[t];
    mine = ctx < 1 ? 0 : tree_part_len(a, ctx);
  }
  len[t] = mine;
  __syncthreads();
  int before = 0;
  if (t < n) {
    for (int j = 0; j < n; j += 4) {
      const int4 o = *reinterpret_cast<const int4*>(len + j);
      before += (o.x > mine) | ((o.x == mine) & (j < t)) ? 1 : 0;
      before += (o.y > mine) | ((o.y == mine) & (j + 1 < t)) ? 1 : 0;
      before += (o.z > mine) | ((o.z == mine) & (j + 2 < t)) ? 1 : 0;
      before += (o.w > mine) | ((o.w == mine) & (j + 3 < t)) ? 1 : 0;
    }
    if (before == place) *found = t;
  }
  __syncthreads();
  return __builtin_amdgcn_readfirstlane(*found);
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
  bool huge;  // some row's maximum is past 2^24 (the same for the whole wave)
  int query[RT], row[RT];
  bool valid[RT];

  // The rows and their queries, as they lie in memory; set() makes them operands once they are there.
  __device__ __forceinline__ void init(const TreeArgs& a, const TreeSeq& sq, int head, int row0, int lane) {
    const int n = lane & 15, g = lane >> 4;
    const bool aligned = ((reinterpret_cast<uintptr_t>(a.q) | (uintptr_t)(a.q_stride * (int64_t)sizeof(T))) & 15u) == 0;
    huge = false;
    const T* qp[RT];
#pragma unroll
    for (int t = 0; t < RT; t++) {
      row[t] = row0 + t * 16 + n;
      valid[t] = row[t] < sq.rows;
      query[t] = valid[t] ? row[t] / a.group : 0;
      const int hq = valid[t] ? row[t] - query[t] * a.group : 0;
      qp[t] = static_cast<const T*>(a.q) + (int64_t)(sq.first + query[t]) * a.q_stride + (int64_t)(head * a.group + hq) * D;
      m[t] = kNoMax;
      lx[t] = 0.f;
      l[t] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int j = 0; j < NJ; j++) o[t][j] = f32x4{0, 0, 0, 0};
    }
    // every lane reads a row that is there and a chunk within it, so that all the loads go out together
    const auto load = [&](bool whole_chunks) {
#pragma unroll
      for (int t = 0; t < RT; t++)
#pragma unroll
        for (int ks = 0; ks < KS; ks++) qf[t][ks] = load_query<E>(qp[t] + (ks * 4 + g < D / X ? ks * 4 + g : 0) * X, whole_chunks);
    };
    if (aligned) load(true);
    else load(false);
  }

  __device__ __forceinline__ void set(const TreeArgs& a, int g) {
    const uint32_t flip = a.q_mode == 1 ? E::kSign : 0u;  // the scale's sign; a scale of 0 takes q as 0
#pragma unroll
    for (int t = 0; t < RT; t++)
#pragma unroll
      for (int ks = 0; ks < KS; ks++) {
        const bool there = valid[t] & (ks * 4 + g < D / X) & (a.q_mode != 2);
#pragma unroll
        for (int i = 0; i < 4; i++) qf[t][ks][i] = there ? qf[t][ks][i] ^ flip : 0u;
      }
  }

  // Which of a lane's places of a step the rows see, in a step that ends past what all see: loads first, so that
  // they are on their way while the logits are made.  tok: the step's first token.
  struct Seen { uint64_t b[RT]; };
  __device__ __forceinline__ Seen look(const TreeArgs& a, const TreeSeq& sq, int tok, int g) {
    Seen v;
    const int d0 = tok + PT * g - (sq.ctx - sq.queries);  // d0 + i: the drafted position, if not negative
#pragma unroll
    for (int t = 0; t < RT; t++) {
      v.b[t] = 0;
      if (a.mask == nullptr) continue;
      const uint8_t* row = a.mask + (int64_t)(sq.first + query[t]) * a.mask_stride;
      if (a.max_query >= 8) {  // 8 places at once, within the row, then moved to where they belong
        const int last = a.max_query - 8, from = d0 < 0 ? 0 : (d0 < last ? d0 : last);
        __builtin_memcpy(&v.b[t], row + from, 8);
      } else {
#pragma unroll
        for (int i = 0; i < 7; i++) v.b[t] |= (uint64_t)(i < sq.queries ? row[i] : 0) << (8 * i);
      }
    }
    return v;
  }
  // -inf in the logits where a row does not see
  __device__ __forceinline__ void hide(const TreeArgs& a, const TreeSeq& sq, f32x4 (*s)[NA], const Seen& v, int tok, int g) {
    const int from = tok + PT * g, d0 = from - (sq.ctx - sq.queries);
    const int inside = sq.ctx - from;  // places of this lane within the context
    const uint32_t in_context = inside >= PT ? 0xffffffffu : (inside <= 0 ? 0u : (1u << inside) - 1u);
    const uint32_t open = d0 >= 0 ? 0u : (d0 <= -PT ? 0xffffffffu : (1u << -d0) - 1u);  // places that all see
#pragma unroll
    for (int t = 0; t < RT; t++) {
      uint32_t sees = 0;
      if (a.mask == nullptr) {
        const int n = query[t] - d0 + 1;
        sees = n >= PT ? 0xffffffffu : (n <= 0 ? 0u : (1u << n) - 1u);
      } else {
        const int last = a.max_query >= 8 ? a.max_query - 8 : 0, read = d0 < 0 ? 0 : (d0 < last ? d0 : last), by = d0 - read;
        uint64_t b = by >= 8 || by <= -8 ? 0 : (by >= 0 ? v.b[t] >> (8 * by) : v.b[t] << (-8 * by));
        b |= b >> 4;  // a truth value to its lowest bit
        b |= b >> 2;
        b |= b >> 1;
        sees = (uint32_t)(((b & 0x0101010101010101ull) * 0x0102040810204080ull) >> 56);  // bit i: byte i's
      }
      sees = (sees | open) & in_context;
#pragma unroll
      for (int i = 0; i < PT; i++) s[t][i >> 2][i & 3] = (sees >> i) & 1u ? s[t][i >> 2][i & 3] : -__builtin_inff();
    }
  }

  // Raises the running maxima where a logit exceeds one by its slack.  A weight is then exp2(s * scale.c - scale.m)
  // with one rounding, of the difference; past 2^24 the product's own would show, and past 2^31 overflow: there the
  // logits are made differences first, of rounded products.
  struct Scale { float c, m[RT]; };
  __device__ __forceinline__ Scale raise(const TreeArgs& a, f32x4 (*s)[NA]) {
    float top[RT];
    bool over = false;
#pragma unroll
    for (int t = 0; t < RT; t++) {
      top[t] = s[t][0][0];
#pragma unroll
      for (int i = 1; i < PT; i++) top[t] = fmaxf(top[t], s[t][i >> 2][i & 3]);
      top[t] *= a.c;
      over |= top[t] > m[t] + (E::kBias + kMaxSlack);
    }
    Scale r;
    r.c = a.c;
    if (__builtin_amdgcn_ballot_w64(over) != 0) {
      bool big = false;
#pragma unroll
      for (int t = 0; t < RT; t++) {
        float high = fmaxf(m[t], top[t] - E::kBias);
        high = fmaxf(high, __shfl_xor(high, 16));
        high = fmaxf(high, __shfl_xor(high, 32));
        const float f = __builtin_amdgcn_exp2f(m[t] - high);
        m[t] = high;
        lx[t] *= f;
        l[t] *= f;
#pragma unroll
        for (int j = 0; j < NJ; j++) o[t][j] *= f;
        big |= fabsf(high) > 0x1p24f && high != kNoMax;
      }
      huge = __builtin_amdgcn_ballot_w64(big) != 0;
    }
#pragma unroll
    for (int t = 0; t < RT; t++) r.m[t] = m[t];
    if (huge) {
#pragma unroll
      for (int t = 0; t < RT; t++) {
#pragma unroll
        for (int i = 0; i < PT; i++) {
          float x = s[t][i >> 2][i & 3] * a.c;
          asm("" : "+v"(x));  // rounded before the difference
          s[t][i >> 2][i & 3] = x - m[t];
        }
        r.m[t] = 0.f;
      }
      r.c = 1.f;
    }
    return r;
  }

  // Logits to rounded weights, and their sum; EXACT: the sum before the rounding too
  template <bool EXACT>
  __device__ __forceinline__ u32x4 weigh(const Scale& scale, int t, const f32x4* s) {
    float x[PT];
#pragma unroll
    for (int i = 0; i < PT; i++) x[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i >> 2][i & 3], scale.c, -scale.m[t]));
    if (EXACT) {
#pragma unroll
      for (int i = 0; i < PT; i++) lx[t] += x[i];
    }
    const u32x4 p = E::pack(x);
    l[t] = E::mma(u32x4{E::kOnes, E::kOnes, E::kOnes, E::kOnes}, p, l[t]);
    return p;
  }

  // The values of a step that ends past what all rows see.  What lies behind the context is nobody's and may
  // be anything: it is taken as 0.  A drafted position may hold infinities or NaN that only the rows that see
  // it must show, and a product with a weight of 0 would hand them to all: such elements are taken out, and put
  // back where the weight is not 0.
  __device__ __forceinline__ void clean(const TreeSeq& sq, u32x4* v, const u32x4* pf, int tok, int g) {
    const int count = sq.ctx - (tok + PT * g);
    uint32_t odd = 0;
#pragma unroll
    for (int j = 0; j < NJ; j++) {
      v[j] = first_elements<E>(v[j], count);
#pragma unroll
      for (int i = 0; i < 4; i++) odd |= odd_signs<E>(v[j][i]);
    }
    if (__builtin_amdgcn_ballot_w64(odd != 0) == 0) return;
#pragma unroll 1
    for (int kind = 0; kind < 3; kind++) {  // +inf, -inf, NaN
      const float special = kind == 0 ? __builtin_inff() : (kind == 1 ? -__builtin_inff() : __builtin_nanf(""));
      const uint32_t nan = kind == 2 ? E::kSign : 0u, flip = kind == 0 ? 0xffffffffu : 0u;
#pragma unroll
      for (int j = 0; j < NJ; j++) {
        u32x4 is;
#pragma unroll
        for (int i = 0; i < 4; i++) {
          uint32_t w = v[j][i];
          asm volatile("" : "+v"(w));  // made anew each time: what could be kept for the next would fill the registers
          const uint32_t n = nan_signs<E>(w);
          is[i] = E::kOnes & whole<E>((n & nan) | (odd_signs<E>(w) & ~n & (w ^ flip) & ~nan));
        }
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
#pragma unroll
      for (int i = 0; i < 4; i++) {
        uint32_t w = v[j][i];
        asm volatile("" : "+v"(w));
        v[j][i] = w & ~whole<E>(odd_signs<E>(w));
      }
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
  if ((sq.parts > 1 || a.logits != nullptr) && d == 0)
    *reinterpret_cast<f32x4*>(a.ml + tree_row(a, it.seq, it.head, it.part, row) * 4) = f32x4{mx, sum, exact, 0.f};
}

// ---- few rows: the caches go straight into the operands ------------------------------------------------
//
// All 4 waves have the same RT tiles of rows; they take turns at the steps of the context and add up
// through LDS.  A wave holds the keys and the values of one step: the next keys are on their way while
// the weights are made, the next values while the next logits are.
// Bound by HBM where sequences are many (64 chains of five over up to 2048 tokens, 40 heads of 128, 16 bits: 256 us =
// 6.6 TB/s, of the 6.9 that bare reads reach), by its chain of loads where they are few (one sequence, 1024 tokens,
// 32 heads: 11 us, of which the 17 MB are 2.5: lengths, table, keys and values, then the join's launch).
// ACC: the weight cache is added to.  A partition's logits stay in LDS (which bounds its length).  Where it is
// the sequence's only one the weights are made of them here; else they go out together at the end, for the
// kernel that joins partitions.  Written out step by step, with the loop's reads, they cost three times as much
// (96 sequences of up to 4096 tokens, 4 query heads to a kv head: 48 us of 247, for 31 MB).
template <typename E, int D, int B, int RT, bool ACC>
__global__ void __launch_bounds__(256, (RT == 1 ? 3 : 2)) pa_tree_few_kernel(const TreeArgs a) {
  typedef typename E::storage T;
  typedef Rows<E, D, RT> R;
  constexpr int X = R::X, TS = R::TS, KS = R::KS, NA = R::NA, NJ = R::NJ, PT = R::PT, WK = 4, ROWS = 16 * RT;
  Item it = tree_item(a);
  if (!it.exists) return;
  if (a.sorted) {
    __shared__ __attribute__((aligned(16))) int sm_len[kTreeSorted];
    __shared__ int sm_found;
    it.seq = by_length(a, it.seq, sm_len, &sm_found);
  }
  const TreeSeq sq = tree_seq(a, it.seq);
  const int tid = threadIdx.x, lane = tid & 63, wk = __builtin_amdgcn_readfirstlane(tid >> 6);
  if (sq.bad) {
    if (it.part == 0 && it.tile == 0) fill_nan<E, D>(a, sq, it.head);
    return;
  }
  const int row0 = it.tile * ROWS;
  if (row0 >= sq.rows || it.part >= sq.parts) return;
  const int n = lane & 15, g = lane >> 4;
  const int p0 = it.part * sq.part_len;
  const int p1 = it.part == sq.parts - 1 ? sq.ctx : p0 + sq.part_len;
  const Span span = tree_span<ACC>(a, sq, row0, ROWS, p0, p1, TS);
  const int steps = span.steps, open_steps = span.open_steps;
  R r;
  __shared__ float sm_m[WK][ROWS], sm_l[WK][ROWS], sm_x[WK][ROWS];
  constexpr int ST = D + 4;  // rows of LDS start 4 banks apart
  extern __shared__ __attribute__((aligned(16))) float sm[];  // tree_few_floats()
  const int logit_row = sq.part_len + 4;

  const int32_t* table = a.tables + (int64_t)it.seq * a.table_width;
  const int last_entry = (sq.ctx - 1) / B;
  const uint32_t block_bytes = (uint32_t)a.num_kv_heads * (uint32_t)(D * B * (int)sizeof(T));  // under 2^32: checked on the host
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
    const char* base = kc + (uint64_t)(uint32_t)checked(b) * block_bytes + (((p0 + step * TS + ktok) & (B - 1)) + g * B) * 16;
#pragma unroll
    for (int i = 0; i < NA; i++)
#pragma unroll
      for (int ks = 0; ks < KS; ks++) {
        if (KS * 4 * X == D || ks < KS - 1 || ks * 4 + g < D / X) kf[i][ks] = load16<true>(base + (i * 4 + ks * 4 * B) * 16);
        else kf[i][ks] = u32x4{0, 0, 0, 0};
      }
  };
  const auto load_v = [&](int b, int step) {
    const char* base = vc + (uint64_t)(uint32_t)checked(b) * block_bytes + (((p0 + step * TS + vtok) & (B - 1)) + n * B) * (int)sizeof(T);
#pragma unroll
    for (int j = 0; j < NJ; j++) vf[j] = load16<true>(base + j * 16 * B * (int)sizeof(T));
  };

  int step = wk;
  if (step >= steps) {
    r.init(a, sq, it.head, row0, lane);
  } else {
    const Ids now = load_ids(step);
    Ids next = load_ids(step + WK < steps ? step + WK : step);
    r.init(a, sq, it.head, row0, lane);
    __builtin_amdgcn_sched_barrier(0);  // in this order, as in the loop: a wait for them must not wait for the blocks
    load_k(now.k, step);
    load_v(now.v, step);
    __builtin_amdgcn_sched_barrier(0);
    r.set(a, g);
    // INNER: a step that all rows see, with another behind it.  Its loads are under no condition: a wait can
    // count on what was issued after the load that it is for only where that is certain.
    const auto turn = [&](auto inner) {
      constexpr bool kInner = decltype(inner)::value;
      const bool more = kInner || step + WK < steps, masked = !kInner && step >= open_steps;
      const int tok = p0 + step * TS;
      typename R::Seen seen;
      if (masked) seen = r.look(a, sq, tok, g);
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
      __builtin_amdgcn_sched_barrier(0);  // the loads where they stand: earlier, they would take registers twice
      if (!kInner) settle<E>();
      if (more) load_k(next.k, step + WK);
      __builtin_amdgcn_sched_barrier(0);
      if (masked) r.hide(a, sq, s, seen, tok, g);
      if (ACC) {
#pragma unroll
        for (int t = 0; t < RT; t++)
          if (r.valid[t]) {
#pragma unroll
            for (int i = 0; i < NA; i++)
              *reinterpret_cast<f32x4*>(sm + (t * 16 + n) * logit_row + step * TS + vtok + 4 * i) = s[t][i] * a.c;
          }
      }
      const typename R::Scale scale = r.raise(a, s);
      u32x4 pf[RT];
#pragma unroll
      for (int t = 0; t < RT; t++) pf[t] = r.template weigh<ACC>(scale, t, s[t]);
      if (masked) r.clean(sq, vf, pf, tok, g);
#pragma unroll
      for (int t = 0; t < RT; t++)
#pragma unroll
        for (int j = 0; j < NJ; j++) r.o[t][j] = E::mma(vf[j], pf[t], r.o[t][j]);
      __builtin_amdgcn_sched_barrier(0);
      if (more) load_v(next.v, step + WK);
      __builtin_amdgcn_sched_barrier(0);
      next = after;
    };
    for (; step < open_steps && step + WK < steps; step += WK) turn(std::true_type{});
    for (; step < steps; step += WK) turn(std::false_type{});
  }
  // a block number outside the cache: the rows must not pass for a result
  const bool any_bad = __builtin_amdgcn_ballot_w64(bad_block) != 0;
  if (ACC) r.finish_exact();

  // the waves' shares of a row: their maxima first, then the sums at the common scale
  if (g == 0) {
#pragma unroll
    for (int t = 0; t < RT; t++) sm_m[wk][t * 16 + n] = r.m[t];
  }
  __syncthreads();
  float share[RT];
#pragma unroll
  for (int t = 0; t < RT; t++) {
    const int row = t * 16 + n;
    float high = sm_m[0][row];
#pragma unroll
    for (int w = 1; w < WK; w++) high = fmaxf(high, sm_m[w][row]);
    share[t] = any_bad ? __builtin_nanf("") : __builtin_amdgcn_exp2f(r.m[t] - high);
    if (g == 0) {
      sm_l[wk][row] = r.l[t][0] * share[t];
      sm_x[wk][row] = r.lx[t] * share[t];
    }
  }
  if (ACC) {
    __syncthreads();
    const int rows = sq.rows - row0 < ROWS ? sq.rows - row0 : ROWS;
    if (tree_whole(sq, ROWS)) {
      for (int pos = tid * 4; pos < sq.ctx; pos += 1024) {
        f32x4 w = {0, 0, 0, 0};
        for (int row = 0; row < rows; row++) {
          float high = sm_m[0][row], sum = sm_x[0][row];
#pragma unroll
          for (int k = 1; k < WK; k++) {
            high = fmaxf(high, sm_m[k][row]);
            sum += sm_x[k][row];
          }
          const float inv = sum == 0.f ? 0.f : 1.0f / sum;
          const f32x4 x = *reinterpret_cast<const f32x4*>(sm + row * logit_row + pos);
#pragma unroll
          for (int i = 0; i < 4; i++) w[i] = __builtin_fmaf(__builtin_amdgcn_exp2f(x[i] - high), inv, w[i]);
        }
        add_weights(a, sq, it.seq, it.head, pos, w);
      }
    } else {
      float* to = a.logits + (((int64_t)it.seq * a.num_kv_heads + it.head) * a.max_rows + row0) * a.logit_stride + p0;
      const int len = (p1 - p0 + TS - 1) / TS * TS;
      for (int row = 0; row < rows; row++)
        for (int pos = tid * 4; pos < len; pos += 1024)
          *reinterpret_cast<f32x4*>(to + row * a.logit_stride + pos) = *reinterpret_cast<const f32x4*>(sm + row * logit_row + pos);
    }
    __syncthreads();
  }
  float (*sm_o)[ROWS][ST] = reinterpret_cast<float (*)[ROWS][ST]>(sm);
#pragma unroll
  for (int t = 0; t < RT; t++)
#pragma unroll
    for (int j = 0; j < NJ; j++) *reinterpret_cast<f32x4*>(&sm_o[wk][t * 16 + n][16 * j + 4 * g]) = r.o[t][j] * share[t];
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
// from the caches at the addresses that the few-rows kernel would use.  Two buffers of each kind, filled from
// registers that were loaded two turns before.  Step i's turn reads keys i + 1 and values i, and fills the other
// buffer of each kind with keys i + 2 and values i + 1: between two barriers a buffer is either read or filled.  One
// barrier a step keeps to that, and one more behind the reads of keys 0, which no turn makes.
//
// Bound by the matrix and vector units, which one wave of each SIMD feeds in turn: 32 sequences of 8192 tokens, 64
// queries each, 8 kv heads of 32: 348 us = 790 TFLOP/s of the 1150 that a large library product reaches (matrix units
// 41 % busy, vector units 47 %); with a quarter of the rows, 200 us, HBM at 5.4 TB/s.  All 256 rows of a head in one
// workgroup halve the reads from L2, but leave fewer workgroups to balance (24 ragged trees of 64, before the longest
// went first: 141 us against 126).
template <typename E, int D, int RT>
__global__ void __launch_bounds__(256, 2) pa_tree_many_kernel(const TreeArgs a) {
  constexpr int NW = 4;
  typedef typename E::storage T;
  typedef Rows<E, D, RT> R;
  constexpr int X = R::X, TS = R::TS, KS = R::KS, NA = R::NA, NJ = R::NJ, PT = R::PT, ROWS = 16 * RT * NW;
  constexpr int NK = NA * KS, FK = (NK + NW - 1) / NW, FV = (NJ + NW - 1) / NW;
  __shared__ __attribute__((aligned(16))) u32x4 sm_k[2][NK * 64], sm_v[2][NJ * 64];
  __shared__ int sm_bad;
  Item it = tree_item(a);
  if (!it.exists) return;
  if (a.sorted) {
    __shared__ __attribute__((aligned(16))) int sm_len[kTreeSorted];
    __shared__ int sm_found;
    it.seq = by_length(a, it.seq, sm_len, &sm_found);
  }
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
  const int p0 = it.part * sq.part_len;
  const int p1 = it.part == sq.parts - 1 ? sq.ctx : p0 + sq.part_len;
  const Span span = tree_span<false>(a, sq, row0, ROWS, p0, p1, TS);
  const int steps = span.steps, open_steps = span.open_steps;
  const bool has_rows = row0 + wave * 16 * RT < sq.rows;
  if (tid == 0) sm_bad = 0;

  R r;

  const int32_t* table = a.tables + (int64_t)it.seq * a.table_width;
  const int last_entry = (sq.ctx - 1) >> bits;
  const uint32_t block_bytes = (uint32_t)a.num_kv_heads * (uint32_t)(D * B * (int)sizeof(T));  // under 2^32: checked on the host
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
  // this wave's pieces; a wave beyond their number fetches the last again
  int k_at[FK], v_at[FV];
  bool k_in[FK];  // whether this lane's chunk is within the head
  const auto k_piece = [&](int f) { return wave + f * NW < NK ? wave + f * NW : NK - 1; };
  const auto v_piece = [&](int f) { return wave + f * NW < NJ ? wave + f * NW : NJ - 1; };
#pragma unroll
  for (int f = 0; f < FK; f++) {
    const int i = k_piece(f) / KS, ks = k_piece(f) - i * KS;
    k_in[f] = ks * 4 + g < D / X;
    k_at[f] = k_in[f] ? (i * 4 + ks * 4 * B) * 16 : 0;
  }
#pragma unroll
  for (int f = 0; f < FV; f++) v_at[f] = v_piece(f) * 16 * B * (int)sizeof(T);
  const auto fetch_k = [&](u32x4* v, int id, int step) {
    const char* kb = kc + (uint64_t)(uint32_t)checked(id) * block_bytes + (((p0 + step * TS + ktok) & (B - 1)) + g * B) * 16;
#pragma unroll
    for (int f = 0; f < FK; f++) v[f] = load16<false>(kb + k_at[f]);
  };
  const auto fetch_v = [&](u32x4* v, int id, int step) {
    const char* vb = vc + (uint64_t)(uint32_t)checked(id) * block_bytes + (((p0 + step * TS + vtok) & (B - 1)) + n * B) * (int)sizeof(T);
#pragma unroll
    for (int f = 0; f < FV; f++) v[f] = load16<false>(vb + v_at[f]);
  };
  const auto put_k = [&](const u32x4* v, u32x4* buf) {
#pragma unroll
    for (int f = 0; f < FK; f++) buf[k_piece(f) * 64 + lane] = KS * 4 * X == D || k_in[f] ? v[f] : u32x4{0, 0, 0, 0};
  };
  const auto put_v = [&](const u32x4* v, u32x4* buf) {
#pragma unroll
    for (int f = 0; f < FV; f++) buf[v_piece(f) * 64 + lane] = v[f];
  };
  const auto take = [&](u32x4 (*k)[KS], const u32x4* buf) {
#pragma unroll
    for (int ks = 0; ks < KS; ks++)
#pragma unroll
      for (int i = 0; i < NA; i++) k[i][ks] = buf[(i * KS + ks) * 64 + lane];
  };
  const auto multiply = [&](f32x4 (*s)[NA], const u32x4 (*k)[KS]) {
#pragma unroll
    for (int t = 0; t < RT; t++)
#pragma unroll
      for (int i = 0; i < NA; i++) s[t][i] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int ks = 0; ks < KS; ks++)
#pragma unroll
      for (int i = 0; i < NA; i++)
#pragma unroll
        for (int t = 0; t < RT; t++) s[t][i] = E::mma(k[i][ks], r.qf[t][ks], s[t][i]);
  };

  // A step past the last is the last again.  Keys run one step ahead of values: when step i's turn comes its
  // logits are there, and the products of step i + 1's keys have no part in what is made of them, so the
  // matrix and the vector units work side by side in every wave.
  const auto clamp = [&](int step) { return step < steps ? step : (steps > 0 ? steps - 1 : 0); };
  u32x4 k_held[2][FK], v_held[2][FV];  // step i's pieces pass through set i % 2; no copies, which would wait for the loads
  f32x4 s[RT][NA];
  {
    const Ids i0 = load_ids(0), i1 = load_ids(clamp(1)), i2 = load_ids(clamp(2));
    r.init(a, sq, it.head, row0 + wave * 16 * RT, lane);
    __builtin_amdgcn_sched_barrier(0);
    fetch_k(k_held[0], i0.k, 0);
    fetch_k(k_held[1], i1.k, clamp(1));
    fetch_v(v_held[0], i0.v, 0);
    fetch_v(v_held[1], i1.v, clamp(1));
    r.set(a, g);
    put_k(k_held[0], sm_k[0]);
    fetch_k(k_held[0], i2.k, clamp(2));
    put_k(k_held[1], sm_k[1]);
    put_v(v_held[0], sm_v[0]);
  }
  __syncthreads();
  {
    u32x4 k[NA][KS];
    take(k, sm_k[0]);
    lds_barrier();  // the first turn fills this buffer anew
    multiply(s, k);
  }
  int next_k = load_ids(clamp(3)).k, next_v = load_ids(clamp(2)).v;
  const auto turn = [&](auto masked, auto odd, int step) {
    constexpr bool kMasked = decltype(masked)::value;
    constexpr int kOdd = decltype(odd)::value;  // step % 2
    const int id_k = next_k, id_v = next_v;
    const int tok = p0 + step * TS;
    typename R::Seen seen;
    if (kMasked) seen = r.look(a, sq, tok, g);
    next_k = load_ids(clamp(step + 4)).k;
    next_v = load_ids(clamp(step + 3)).v;
    fetch_k(k_held[1 - kOdd], id_k, clamp(step + 3));
    fetch_v(v_held[kOdd], id_v, clamp(step + 2));
    if (has_rows) {
      u32x4 k[NA][KS], v[NJ];
      take(k, sm_k[1 - kOdd]);  // on their way while the maxima are looked at
      __builtin_amdgcn_sched_barrier(0);
      if (kMasked) r.hide(a, sq, s, seen, tok, g);
      const typename R::Scale scale = r.raise(a, s);
      f32x4 ahead[RT][NA];
      multiply(ahead, k);
#pragma unroll
      for (int j = 0; j < NJ; j++) v[j] = sm_v[kOdd][j * 64 + lane];
      u32x4 pf[RT];
#pragma unroll
      for (int t = 0; t < RT; t++) pf[t] = r.template weigh<false>(scale, t, s[t]);
      if (kMasked) r.clean(sq, v, pf, tok, g);
#pragma unroll
      for (int j = 0; j < NJ; j++)
#pragma unroll
        for (int t = 0; t < RT; t++) r.o[t][j] = E::mma(v[j], pf[t], r.o[t][j]);
#pragma unroll
      for (int t = 0; t < RT; t++)
#pragma unroll
        for (int i = 0; i < NA; i++) s[t][i] = ahead[t][i];
    }
    put_k(k_held[kOdd], sm_k[kOdd]);
    put_v(v_held[1 - kOdd], sm_v[1 - kOdd]);
    lds_barrier();
  };
  int step = 0;
  constexpr std::integral_constant<int, 0> even{};
  constexpr std::integral_constant<int, 1> odd{};
  for (; step + 1 < open_steps; step += 2) {
    turn(std::false_type{}, even, step);
    turn(std::false_type{}, odd, step + 1);
  }
  for (; step < steps; step += 2) {  // an open step among them is looked at like the others
    turn(std::true_type{}, even, step);
    if (step + 1 < steps) turn(std::true_type{}, odd, step + 1);
  }
  if (bad_block) sm_bad = 1;
  __syncthreads();
  const bool any_bad = sm_bad != 0;
#pragma unroll
  for (int t = 0; t < RT; t++)
    if (r.valid[t]) {
      const float sum = any_bad ? __builtin_nanf("") : r.l[t][0];
#pragma unroll
      for (int j = 0; j < NJ; j++) store_row<E, D>(a, sq, it, r.row[t], 16 * j + 4 * g, r.o[t][j], r.m[t], sum, 0.f);
    }
}

template <typename E, int D, int B, int RT, bool ACC>
static int tree_few_launch(const TreeArgs& a, unsigned grid, hipStream_t st) {
  // as much LDS as this launch's logits take: short contexts leave room for a third workgroup on a CU
  // (108 sequences of up to 176 tokens, 16 heads of 64: 16.4 us, with 76 KiB for all 22.3)
  const int floats = tree_few_floats(D, RT, ACC ? (a.max_rows < 16 * RT ? a.max_rows : 16 * RT) : 0, a.part_len);
  const void* kernel = reinterpret_cast<const void*>(&pa_tree_few_kernel<E, D, B, RT, ACC>);
  if (floats * 4 > 65536) {
    // the most of any launch: two threads that set what their own take could lower it before the other's launch
    const hipError_t e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, kTreeLogitFloats * 4);
    if (e != hipSuccess) return fail(PA_ERR_HIP, "cached attention of several queries: hipFuncSetAttribute: %s", hipGetErrorString(e));
  }
  hipLaunchKernelGGL((pa_tree_few_kernel<E, D, B, RT, ACC>), dim3(grid), dim3(256), floats * 4, st, a);
  return PA_OK;
}

template <typename E, int D, int B>
static int tree_few(const TreeArgs& a, int form, unsigned grid, hipStream_t st) {
  if (a.weights != nullptr)
    return form == kTreeFew16 ? tree_few_launch<E, D, B, 1, true>(a, grid, st) : tree_few_launch<E, D, B, 2, true>(a, grid, st);
  return form == kTreeFew16 ? tree_few_launch<E, D, B, 1, false>(a, grid, st) : tree_few_launch<E, D, B, 2, false>(a, grid, st);
}

template <typename E, int D>
static int tree_pick_form(const TreeArgs& a, unsigned grid, hipStream_t st) {
  const int form = a.form;
  if (form == kTreeMany64) hipLaunchKernelGGL((pa_tree_many_kernel<E, D, 1>), dim3(grid), dim3(256), 0, st, a);
  else if (form == kTreeMany128) {
    if constexpr (E::kX == 8) hipLaunchKernelGGL((pa_tree_many_kernel<E, D, 2>), dim3(grid), dim3(256), 0, st, a);
  } else {
    if (a.block_bits == 3) return tree_few<E, D, 8>(a, form, grid, st);
    if (a.block_bits == 4) return tree_few<E, D, 16>(a, form, grid, st);
    return tree_few<E, D, 32>(a, form, grid, st);
  }
  return PA_OK;
}

template <typename E>
static int tree_launch(const TreeArgs& a, int head_size, unsigned grid, hipStream_t st) {
  int rc;
  switch (head_size) {
    case 64: rc = tree_pick_form<E, 64>(a, grid, st); break;
    case 80: rc = tree_pick_form<E, 80>(a, grid, st); break;
    case 96: rc = tree_pick_form<E, 96>(a, grid, st); break;
    default: rc = tree_pick_form<E, 128>(a, grid, st); break;
  }
  if (rc != PA_OK) return rc;
  PA_CHECK_LAUNCH("cached attention of several queries");
  return PA_OK;
}

}  // namespace tree
}  // namespace pa
