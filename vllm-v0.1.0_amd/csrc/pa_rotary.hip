// Rotary embedding in both pair layouts, over all or the first part of every
// head, and the same with an RMS norm of every query and key head in front, for
// gfx950 (MI355X).  No counterpart in the reference, whose only rotation is
// rotary_embedding_neox (csrc/pos_encoding_kernels.cu:7-83; pa_elementwise.hip).
//
//   pair i of a head:  half layout (v[i], v[i + rot_dim/2]), interleaved (v[2i], v[2i+1])
//   (a, b) -> (a cos - b sin, b cos + a sin),  cos / sin = the position's table row
//   with the norm, v = x * rsqrt(mean(x^2) + epsilon) * weight before the rotation;
//   elements from rot_dim on are normed and not rotated.
//
// Everything between the load and the store is fp32 and rounded once: a 16-bit
// result is off by half a step of its type.  The table is fp32 (or the rows'
// type): a 16-bit table would put an error of 2^-9 on every angle's cosine,
// which is as much as the result's own rounding.
//
// One pass over the rows, bound by HBM for prompts (8192 tokens of 40 + 40 heads
// of 128 with norms, fp16: 70 us = 4.9 TB/s of the 5.9 that an in-place pass over
// plain memory reaches) and by the launch for the steps of a small batch (8 tokens
// 2.8 us, 256 tokens with norms 4.0).  2^k lanes own a head (k such that a lane holds
// two vectors of the rotated part, and one of the rest): a head's sum of squares is
// then k exchanges between lanes, and both elements of a pair are in one lane in both
// layouts.  A lane keeps its table entries for all the heads of a token that it
// visits: the row is fetched once per wave, not once per head.  Two heads in a lane's
// hand at once were slower (84 us), streaming loads and stores too where a part of
// every head is rotated (43 us against 37).
#include "pa_common.h"
#include "pa_exact_math.h"

namespace pa {

struct RotaryArgs {
  const int64_t* positions;
  void* rows[2];             // query, key
  int64_t stride[2];         // elements between token rows
  const void* weight[2];     // [head_size], of the rows' type (norm only)
  const void* table;         // [max_position, rot_dim]: cos half, sin half
  int64_t max_position;
  int num_heads[2];
  int head_size, rot_dim;
  int lane_bits;             // log2 of the lanes that own a head
  float epsilon;
};

template <typename T, int N>
struct alignas(sizeof(T) * N) Vec {
  T v[N];
};

template <typename T, int N>
__device__ __forceinline__ void load_f32(const T* p, float* f) {
  const Vec<T, N> x = *reinterpret_cast<const Vec<T, N>*>(p);
#pragma unroll
  for (int e = 0; e < N; e++) f[e] = Num<T>::to(x.v[e]);
}

// the table's row may be less aligned than a lane's share of it: 16 bytes at most
template <typename T, int N>
__device__ __forceinline__ void load_table(const T* p, float* f) {
  constexpr int M = N * (int)sizeof(T) > 16 ? 16 / (int)sizeof(T) : N;
#pragma unroll
  for (int i = 0; i < N / M; i++) load_f32<T, M>(p + i * M, f + i * M);
}

template <typename T, int N>
__device__ __forceinline__ void store_rounded(T* p, const float* f) {
  Vec<T, N> x;
#pragma unroll
  for (int e = 0; e < N; e++) x.v[e] = Num<T>::from(f[e]);
  *reinterpret_cast<Vec<T, N>*>(p) = x;
}

// the W / 2 pairs of one vector
template <int W>
__device__ __forceinline__ void turn_inside(float* v, const float* c, const float* s) {
#pragma unroll
  for (int e = 0; e < W / 2; e++) {
    const float p = v[2 * e], q = v[2 * e + 1];
    v[2 * e] = __builtin_fmaf(p, c[e], -(q * s[e]));
    v[2 * e + 1] = __builtin_fmaf(q, c[e], p * s[e]);
  }
}

// W: elements of a vector.  A lane's two vectors are W * i and rot_dim / 2 + W * i in both layouts, so that
// neighbouring lanes read neighbouring memory: W pairs across them in the half layout, W / 2 pairs within each in
// the interleaved one (W = 1: the two elements of one pair).  The chain of loads is kept short: a token's first
// heads are on their way before its position is known, its next ones while the last are worked on, and the
// weights while a sum is exchanged.  grid = (tokens, slices of the heads).
template <typename T, typename TT, int W, bool INTERLEAVED, bool NORM>
__global__ void __launch_bounds__(256)
pa_rotary_kernel(const RotaryArgs a) {
  const int token = blockIdx.x;
  constexpr bool INSIDE = INTERLEAVED && W > 1;  // pairs within a vector
  const int half = a.rot_dim >> 1;
  const int lane = threadIdx.x & ((1 << a.lane_bits) - 1);
  const int slot = (int)((blockIdx.y * blockDim.x + threadIdx.x) >> a.lane_bits);
  const int slots = (int)((gridDim.y * blockDim.x) >> a.lane_bits);
  const int heads = a.num_heads[0] + a.num_heads[1];
  if (slot >= heads) return;
  const bool has_pair = W * lane < half;
  const int ia = INTERLEAVED && !INSIDE ? 2 * lane : W * lane;
  const int ib = INTERLEAVED && !INSIDE ? ia + 1 : half + ia;
  const int it = a.rot_dim + W * lane;
  const bool has_tail = NORM && it < a.head_size;
  typedef Vec<T, W> V;

  struct Head { T* base; const T* weight; V x, y, t; };
  const auto fetch = [&](int h) {
    Head r;
    const int w = h >= a.num_heads[0];
    r.base = static_cast<T*>(a.rows[w]) + (int64_t)token * a.stride[w] + (int64_t)(h - (w ? a.num_heads[0] : 0)) * a.head_size;
    r.weight = static_cast<const T*>(a.weight[w]);
    // lanes without a part of the head read its first elements
    r.x = *reinterpret_cast<const V*>(r.base + (has_pair ? ia : 0));
    r.y = *reinterpret_cast<const V*>(r.base + (has_pair ? ib : 0));
    if (NORM) r.t = *reinterpret_cast<const V*>(r.base + (has_tail ? it : 0));
    return r;
  };
  Head next = fetch(slot);
  const int64_t pos = a.positions[token];
  if (pos < 0) return;  // a padded row

  // INSIDE: the first vector's W / 2 pairs, then the second's
  float c[W], s[W];
#pragma unroll
  for (int e = 0; e < W; e++) c[e] = s[e] = 0.f;
  if (has_pair) {
    if (pos < a.max_position) {
      const TT* row = static_cast<const TT*>(a.table) + pos * a.rot_dim;
      if constexpr (INSIDE) {
        load_table<TT, W / 2>(row + ia / 2, c);
        load_table<TT, W / 2>(row + ib / 2, c + W / 2);
        load_table<TT, W / 2>(row + half + ia / 2, s);
        load_table<TT, W / 2>(row + half + ib / 2, s + W / 2);
      } else {
        load_table<TT, W>(row + W * lane, c);
        load_table<TT, W>(row + half + W * lane, s);
      }
    } else {  // no such row: the caller's mistake must not pass for a result
#pragma unroll
      for (int e = 0; e < W; e++) c[e] = s[e] = __builtin_nanf("");
    }
  }
  for (int h = slot; h < heads; h += slots) {
    const Head now = next;
    next = fetch(h + slots < heads ? h + slots : h);  // behind the last, the last again
    float x[W], y[W], t[W];
#pragma unroll
    for (int e = 0; e < W; e++) {
      x[e] = has_pair ? Num<T>::to(now.x.v[e]) : 0.f;
      y[e] = has_pair ? Num<T>::to(now.y.v[e]) : 0.f;
      if (NORM) t[e] = has_tail ? Num<T>::to(now.t.v[e]) : 0.f;
    }
    if (NORM) {
      float gx[W], gy[W], gt[W];
      load_f32<T, W>(now.weight + (has_pair ? ia : 0), gx);
      load_f32<T, W>(now.weight + (has_pair ? ib : 0), gy);
      load_f32<T, W>(now.weight + (has_tail ? it : 0), gt);
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < W; e++) ss = __builtin_fmaf(x[e], x[e], __builtin_fmaf(y[e], y[e], __builtin_fmaf(t[e], t[e], ss)));
      for (int off = (1 << a.lane_bits) >> 1; off >= 1; off >>= 1) ss += __shfl_xor(ss, off);
      const float r = 1.0f / sqrtf(ss / (float)a.head_size + a.epsilon);
#pragma unroll
      for (int e = 0; e < W; e++) {
        x[e] *= r * gx[e];
        y[e] *= r * gy[e];
        t[e] *= r * gt[e];
      }
      if (has_tail) store_rounded<T, W>(now.base + it, t);
    }
    if (has_pair) {
      if constexpr (INSIDE) {
        turn_inside<W>(x, c, s);
        turn_inside<W>(y, c + W / 2, s + W / 2);
      } else {
#pragma unroll
        for (int e = 0; e < W; e++) {
          const float p = x[e], q = y[e];
          x[e] = __builtin_fmaf(p, c[e], -(q * s[e]));
          y[e] = __builtin_fmaf(q, c[e], p * s[e]);
        }
      }
      store_rounded<T, W>(now.base + ia, x);
      store_rounded<T, W>(now.base + ib, y);
    }
  }
}

// Heads of more vectors than a wave has lanes (long heads at addresses that allow only narrow
// vectors): one wave to a head, element by element.  Every element is read for the sum before any
// is written, and each pair is read again by the lane that writes it.
template <typename T, typename TT, bool INTERLEAVED, bool NORM>
__global__ void __launch_bounds__(256)
pa_rotary_long_kernel(const RotaryArgs a) {
  const int token = blockIdx.x;
  const int64_t pos = a.positions[token];
  if (pos < 0) return;
  const int half = a.rot_dim >> 1;
  const int lane = threadIdx.x & 63;
  const int waves = (int)(gridDim.y * blockDim.x) >> 6;
  const TT* row = static_cast<const TT*>(a.table) + (pos < a.max_position ? pos : 0) * a.rot_dim;
  const float bad = pos < a.max_position ? 0.f : __builtin_nanf("");
  for (int h = (int)(blockIdx.y * blockDim.x + threadIdx.x) >> 6; h < a.num_heads[0] + a.num_heads[1]; h += waves) {
    const int w = h >= a.num_heads[0];
    T* base = static_cast<T*>(a.rows[w]) + (int64_t)token * a.stride[w] +
              (int64_t)(h - (w ? a.num_heads[0] : 0)) * a.head_size;
    const T* weight = static_cast<const T*>(a.weight[w]);
    float r = 1.f;
    if (NORM) {
      float ss = 0.f;
      for (int i = lane; i < a.head_size; i += 64) {
        const float x = Num<T>::to(base[i]);
        ss = __builtin_fmaf(x, x, ss);
      }
#pragma unroll
      for (int off = 32; off >= 1; off >>= 1) ss += __shfl_xor(ss, off);
      r = 1.0f / sqrtf(ss / (float)a.head_size + a.epsilon);
      for (int i = a.rot_dim + lane; i < a.head_size; i += 64) base[i] = Num<T>::from(Num<T>::to(base[i]) * (r * Num<T>::to(weight[i])));
    }
    for (int i = lane; i < half; i += 64) {
      const int ia = INTERLEAVED ? 2 * i : i, ib = INTERLEAVED ? ia + 1 : half + i;
      const float c = Num<TT>::to(row[i]) + bad, s = Num<TT>::to(row[half + i]) + bad;
      float x = Num<T>::to(base[ia]), y = Num<T>::to(base[ib]);
      if (NORM) {
        x *= r * Num<T>::to(weight[ia]);
        y *= r * Num<T>::to(weight[ib]);
      }
      base[ia] = Num<T>::from(__builtin_fmaf(x, c, -(y * s)));
      base[ib] = Num<T>::from(__builtin_fmaf(y, c, x * s));
    }
  }
}

template <typename T, typename TT>
static void rotary_pick_long(const RotaryArgs& a, bool interleaved, bool norm, dim3 grid, hipStream_t st) {
  if (interleaved) {
    if (norm) hipLaunchKernelGGL((pa_rotary_long_kernel<T, TT, true, true>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((pa_rotary_long_kernel<T, TT, true, false>), grid, dim3(256), 0, st, a);
  } else {
    if (norm) hipLaunchKernelGGL((pa_rotary_long_kernel<T, TT, false, true>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((pa_rotary_long_kernel<T, TT, false, false>), grid, dim3(256), 0, st, a);
  }
}

template <typename T, typename TT, int W>
static void rotary_pick(const RotaryArgs& a, bool interleaved, bool norm, dim3 grid, int threads, hipStream_t st) {
  if (interleaved) {
    if (norm) hipLaunchKernelGGL((pa_rotary_kernel<T, TT, W, true, true>), grid, dim3(threads), 0, st, a);
    else hipLaunchKernelGGL((pa_rotary_kernel<T, TT, W, true, false>), grid, dim3(threads), 0, st, a);
  } else {
    if (norm) hipLaunchKernelGGL((pa_rotary_kernel<T, TT, W, false, true>), grid, dim3(threads), 0, st, a);
    else hipLaunchKernelGGL((pa_rotary_kernel<T, TT, W, false, false>), grid, dim3(threads), 0, st, a);
  }
}

template <typename T, typename TT>
static int rotary_launch_any(const char* what, RotaryArgs a, int num_tokens, bool interleaved, bool norm, hipStream_t st) {
  // The widest vector that every address a lane forms is a multiple of: 16 bytes, or less where
  // a part's length, a stride or a pointer asks for it.
  int w = 16 / (int)sizeof(T);
  const int half = a.rot_dim / 2;
  const auto fits = [&](int n) {
    bool ok = half % n == 0 && a.head_size % n == 0 && reinterpret_cast<uintptr_t>(a.table) % (n * sizeof(TT) > 16 ? 16 : n * sizeof(TT)) == 0;
    if (norm) ok = ok && (a.head_size - a.rot_dim) % n == 0;
    for (int i = 0; i < 2; i++) {
      if (a.num_heads[i] == 0) continue;
      ok = ok && reinterpret_cast<uintptr_t>(a.rows[i]) % (n * sizeof(T)) == 0 && a.stride[i] % n == 0;
      if (norm) ok = ok && reinterpret_cast<uintptr_t>(a.weight[i]) % (n * sizeof(T)) == 0;
    }
    return ok;
  };
  while (w > 1 && !fits(w)) w >>= 1;
  int items = half / w;
  if (norm && (a.head_size - a.rot_dim) / w > items) items = (a.head_size - a.rot_dim) / w;
  a.lane_bits = 0;
  while ((1 << a.lane_bits) < items) a.lane_bits++;
  if (a.lane_bits > 6) {
    const int heads = a.num_heads[0] + a.num_heads[1], want = (2048 + num_tokens - 1) / num_tokens;
    const dim3 grid(num_tokens, (heads + 3) / 4 < want ? (heads + 3) / 4 : want);
    rotary_pick_long<T, TT>(a, interleaved, norm, grid, st);
    PA_CHECK_LAUNCH(what);
    return PA_OK;
  }
  const int work = (a.num_heads[0] + a.num_heads[1]) << a.lane_bits;
  const int threads = work <= 64 ? 64 : (work <= 128 ? 128 : 256);
  int slices = (work + threads - 1) / threads;
  const int want = (2048 + num_tokens - 1) / num_tokens;  // small batches still fill the chip
  if (slices > want) slices = want;
  const dim3 grid(num_tokens, slices);
  switch (w) {
    case 8: rotary_pick<T, TT, (sizeof(T) == 2 ? 8 : 4)>(a, interleaved, norm, grid, threads, st); break;
    case 4: rotary_pick<T, TT, 4>(a, interleaved, norm, grid, threads, st); break;
    case 2: rotary_pick<T, TT, 2>(a, interleaved, norm, grid, threads, st); break;
    default: rotary_pick<T, TT, 1>(a, interleaved, norm, grid, threads, st); break;
  }
  PA_CHECK_LAUNCH(what);
  return PA_OK;
}

// Whether two sets of token rows share an element.  Rows of one stride (columns of one projection) are
// told apart by their columns; others by their extents.
static bool rows_overlap(const void* pa, int64_t sa, int64_t la, const void* pb, int64_t sb, int64_t lb, int64_t n, int es) {
  const int64_t a = static_cast<int64_t>(reinterpret_cast<uintptr_t>(pa)), b = static_cast<int64_t>(reinterpret_cast<uintptr_t>(pb));
  const int64_t ea = a + ((n - 1) * sa + la) * es, eb = b + ((n - 1) * sb + lb) * es;
  if (ea <= b || eb <= a) return false;
  if (n == 1 || sa != sb) return true;
  int64_t d = (b - a) % (sa * es);
  if (d < 0) d += sa * es;
  return d < la * es || d + lb * es > sa * es;
}

static int rotary_entry(const char* what, const int64_t* positions, void* query, void* key, const void* query_weight,
                        const void* key_weight, float epsilon, const void* cos_sin_cache, int num_tokens, int num_heads,
                        int num_kv_heads, int head_size, int rot_dim, int64_t max_position, int64_t query_stride,
                        int64_t key_stride, int interleaved, bool norm, int dtype, int table_dtype, void* stream) {
  clear_error();
  if (dtype != PA_DTYPE_F32 && dtype != PA_DTYPE_F16 && dtype != PA_DTYPE_BF16)
    return fail(PA_ERR_UNSUPPORTED, "%s: unsupported data type code: %d", what, dtype);
  if (table_dtype != PA_DTYPE_F32 && table_dtype != dtype)
    return fail(PA_ERR_UNSUPPORTED, "%s: cos_sin_cache must be float32 or of query's data type", what);
  PA_REQUIRE(num_tokens >= 0 && num_heads >= 0 && num_kv_heads >= 0 && head_size >= 0 && rot_dim >= 0 && max_position >= 0,
             "%s: negative size", what);
  PA_REQUIRE(rot_dim % 2 == 0 && rot_dim <= head_size, "%s: rot_dim %d must be even and <= head_size %d", what, rot_dim, head_size);
  PA_REQUIRE(num_heads <= (1 << 20) && num_kv_heads <= (1 << 20), "%s: too many heads", what);
  if (num_tokens == 0 || num_heads + num_kv_heads == 0 || head_size == 0 || (rot_dim == 0 && !norm)) return PA_OK;
  PA_REQUIRE(positions && (query || num_heads == 0) && (key || num_kv_heads == 0) && (cos_sin_cache || rot_dim == 0),
             "%s: null pointer argument", what);
  PA_REQUIRE(!norm || ((query_weight || num_heads == 0) && (key_weight || num_kv_heads == 0)), "%s: null weight", what);
  const int64_t ql = (int64_t)num_heads * head_size, kl = (int64_t)num_kv_heads * head_size;
  PA_REQUIRE(num_tokens == 1 || (query_stride >= ql && key_stride >= kl), "%s: row stride is shorter than a token row", what);
  PA_REQUIRE(num_heads == 0 || num_kv_heads == 0 ||
                 !rows_overlap(query, query_stride, ql, key, key_stride, kl, num_tokens, elem_size(dtype)),
             "%s: query and key rows overlap", what);
  RotaryArgs a;
  a.positions = positions;
  a.rows[0] = query, a.rows[1] = key;
  a.stride[0] = query_stride, a.stride[1] = key_stride;
  a.weight[0] = query_weight, a.weight[1] = key_weight;
  a.table = cos_sin_cache;
  a.max_position = max_position;
  a.num_heads[0] = num_heads, a.num_heads[1] = num_kv_heads;
  a.head_size = head_size, a.rot_dim = rot_dim;
  a.epsilon = epsilon;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const bool il = interleaved != 0;
  switch (dtype) {
    case PA_DTYPE_F32: return rotary_launch_any<float, float>(what, a, num_tokens, il, norm, st);
    case PA_DTYPE_F16:
      return table_dtype == PA_DTYPE_F32 ? rotary_launch_any<_Float16, float>(what, a, num_tokens, il, norm, st)
                                         : rotary_launch_any<_Float16, _Float16>(what, a, num_tokens, il, norm, st);
    default:
      return table_dtype == PA_DTYPE_F32 ? rotary_launch_any<__bf16, float>(what, a, num_tokens, il, norm, st)
                                         : rotary_launch_any<__bf16, __bf16>(what, a, num_tokens, il, norm, st);
  }
}

}  // namespace pa

extern "C" int pa_rotary_embedding(const int64_t* positions, void* query, void* key, const void* cos_sin_cache,
                                   int num_tokens, int num_heads, int num_kv_heads, int head_size, int rot_dim,
                                   int64_t max_position, int64_t query_stride, int64_t key_stride, int interleaved,
                                   int dtype, int table_dtype, void* stream) {
  return pa::rotary_entry("pa_rotary_embedding", positions, query, key, nullptr, nullptr, 0.f, cos_sin_cache, num_tokens,
                          num_heads, num_kv_heads, head_size, rot_dim, max_position, query_stride, key_stride, interleaved,
                          false, dtype, table_dtype, stream);
}

extern "C" int pa_qk_norm_rotary_embedding(const int64_t* positions, void* query, void* key, const void* query_weight,
                                           const void* key_weight, float epsilon, const void* cos_sin_cache,
                                           int num_tokens, int num_heads, int num_kv_heads, int head_size, int rot_dim,
                                           int64_t max_position, int64_t query_stride, int64_t key_stride,
                                           int interleaved, int dtype, int table_dtype, void* stream) {
  return pa::rotary_entry("pa_qk_norm_rotary_embedding", positions, query, key, query_weight, key_weight, epsilon,
                          cos_sin_cache, num_tokens, num_heads, num_kv_heads, head_size, rot_dim, max_position,
                          query_stride, key_stride, interleaved, true, dtype, table_dtype, stream);
}
