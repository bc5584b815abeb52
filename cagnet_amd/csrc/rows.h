// Typed row access and the counter-based generator shared by the row-wise training operators (dropout, embedding,
// rms_norm, norm_residual).  Activations are float32, bfloat16 or float16 in memory and float32 in registers.
#pragma once
#include "common.h"

namespace cg {

template <int DTYPE>
struct Elem;
template <>
struct Elem<CG_F32> {
  typedef float type;
};
template <>
struct Elem<CG_BF16> {
  typedef __bf16 type;
};
template <>
struct Elem<CG_F16> {
  typedef _Float16 type;
};

// The rounding at a store.  A product that is rounded to float16 right away would be compiled to one instruction that
// rounds the exact product once, in some kernels and not in others; held in a register in between, it is float32
// arithmetic and then a rounding everywhere, for every type.
template <typename T>
__device__ __forceinline__ T rounded(float v) {
  if (sizeof(T) == 2) asm("" : "+v"(v));
  return (T)v;
}

// N consecutive elements that are only aligned as single elements are: rows of 602 floats start 8 bytes apart from a
// 16-byte boundary, rows of 41 start anywhere.  The memory pipeline takes wide accesses at any element address, so
// such rows are moved 16 bytes per lane like aligned ones.
template <typename T, int N>
struct Pack {
  typedef T type __attribute__((ext_vector_type(N), aligned(alignof(T))));
};

template <typename T, int N>
__device__ __forceinline__ void load_pack(const T *__restrict__ p, float (&out)[N]) {
  const typename Pack<T, N>::type q = *reinterpret_cast<const typename Pack<T, N>::type *>(p);
#pragma unroll
  for (int i = 0; i < N; ++i) out[i] = (float)q[i];
}
template <typename T, int N>
__device__ __forceinline__ void store_pack(T *__restrict__ p, const float (&in)[N]) {
  typename Pack<T, N>::type q;
#pragma unroll
  for (int i = 0; i < N; ++i) q[i] = rounded<T>(in[i]);
  *reinterpret_cast<typename Pack<T, N>::type *>(p) = q;
}
// the first `live` (0..N) of N elements; the others read as zero and are not written
template <typename T, int N>
__device__ __forceinline__ void load_some(const T *__restrict__ p, int live, float (&out)[N]) {
  if (live >= N) {
    load_pack<T, N>(p, out);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = i < live ? (float)p[i] : 0.f;
  }
}
template <typename T, int N>
__device__ __forceinline__ void store_some(T *__restrict__ p, int live, const float (&in)[N]) {
  if (live >= N) {
    store_pack<T, N>(p, in);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < live) p[i] = rounded<T>(in[i]);
  }
}

// ---------------------------------------------------------------------------------------------
// A row as 16-byte chunks, one per lane and step.  Every load is unconditional: a load behind a branch would make the
// compiler wait for it inside the branch.  Lanes behind the row's end read its start and are zeroed.  RAGGED: rows whose
// length is not a whole number of chunks; the last chunk is then read as the row's last 16 bytes and shifted into place,
// which costs up to 20 instructions a load, so that rows of whole chunks have kernels of their own.
// ---------------------------------------------------------------------------------------------
typedef uint32_t Raw __attribute__((ext_vector_type(4)));

template <typename T, bool RAGGED>
struct Chunk {
  static constexpr int V = 16 / (int)sizeof(T);  // elements of a chunk
  typedef typename Pack<T, V>::type vec;

  int32_t at;    // element of the row the load starts at
  int32_t live;  // elements of the row in this chunk: V, fewer in the last one, 0 behind the end
  int32_t d;

  __device__ __forceinline__ void place(int32_t j, int32_t d_) {
    d = d_;
    const int32_t left = d - j;
    live = left >= V ? V : (left > 0 ? left : 0);
    at = left >= V ? j : (left > 0 && d >= V ? d - V : 0);
  }
  __device__ __forceinline__ Raw load(const T *row) const {
    if (!RAGGED || d >= V) return __builtin_bit_cast(Raw, *reinterpret_cast<const vec *>(row + at));
    vec q = {};  // rows shorter than a chunk (uniform branch)
#pragma unroll
    for (int i = 0; i < V; ++i) q[i] = row[i < d ? i : d - 1];
    return __builtin_bit_cast(Raw, q);
  }
  // the chunk's elements as floats; those that are not live are zero
  __device__ __forceinline__ void floats(Raw r, float (&out)[V]) const {
    if (!RAGGED) {
      r = live ? r : Raw{0u, 0u, 0u, 0u};
    } else if (d >= V) {  // uniform
      const int32_t drop = V - live;  // elements of the chunk before that this load repeats; all V behind the end
      if (sizeof(T) == 4) {
        r = (drop & 1) ? Raw{r.y, r.z, r.w, 0u} : r;
        r = (drop & 2) ? Raw{r.z, r.w, 0u, 0u} : r;
        r = (drop & 4) ? Raw{0u, 0u, 0u, 0u} : r;
      } else {
        r = (drop & 1) ? Raw{(r.x >> 16) | (r.y << 16), (r.y >> 16) | (r.z << 16), (r.z >> 16) | (r.w << 16), r.w >> 16} : r;
        r = (drop & 2) ? Raw{r.y, r.z, r.w, 0u} : r;
        r = (drop & 4) ? Raw{r.z, r.w, 0u, 0u} : r;
        r = (drop & 8) ? Raw{0u, 0u, 0u, 0u} : r;
      }
    }
    const vec q = __builtin_bit_cast(vec, r);
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = (float)q[i];
    if (RAGGED && d < V) {
#pragma unroll
      for (int i = 0; i < V; ++i) out[i] = i < live ? out[i] : 0.f;
    }
  }
  __device__ __forceinline__ void write(T *row, const float (&in)[V]) const {
    vec q = {};
#pragma unroll
    for (int i = 0; i < V; ++i) q[i] = rounded<T>(in[i]);
    if (live == V) {
      *reinterpret_cast<vec *>(row + at) = q;
    } else if (RAGGED && live > 0) {
      T *p = row + d - live;
#pragma unroll
      for (int i = 0; i < V - 1; ++i)
        if (i < live) p[i] = q[i];
    }
  }
};

// Sum over teams of LANES consecutive lanes of a wavefront, the same bits in every lane, without a trip through LDS: data
// parallel primitives inside 16 lanes (swap in pairs, in quads, mirror 8, mirror 16: sums of equal groups, so a mirror
// does what an exclusive-or of the lane number would), then the exchanges of halves between rows of 16 and of 32.
template <int LANES>
__device__ __forceinline__ float team_sum_of(float v) {
#define CG_DPP(ctrl) __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), ctrl, 0xf, 0xf, true))
  if (LANES >= 2) v += CG_DPP(0xB1);
  if (LANES >= 4) v += CG_DPP(0x4E);
  if (LANES >= 8) v += CG_DPP(0x141);
  if (LANES >= 16) v += CG_DPP(0x140);
#undef CG_DPP
  if (LANES >= 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
    v = __builtin_bit_cast(float, (uint32_t)r[0]) + __builtin_bit_cast(float, (uint32_t)r[1]);
  }
  if (LANES >= 64) {
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
    v = __builtin_bit_cast(float, (uint32_t)r[0]) + __builtin_bit_cast(float, (uint32_t)r[1]);
  }
  return v;
}

// A weight vector: float32, or the type of the activations; a null pointer stands for ones.
template <typename T>
__device__ __forceinline__ float weight_at(const void *w, int w_f32, int32_t j) {
  if (!w) return 1.f;
  return w_f32 ? static_cast<const float *>(w)[j] : (float)static_cast<const T *>(w)[j];
}
template <typename T>
__device__ __forceinline__ void weight_put(void *w, int w_f32, int32_t j, float v) {
  if (w_f32)
    static_cast<float *>(w)[j] = v;
  else
    static_cast<T *>(w)[j] = rounded<T>(v);
}

// ---------------------------------------------------------------------------------------------
// Masks.  Philox 4x32 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3",
// 2011): a keyed bijection of a 128-bit counter, each round two 32 x 32 -> 64 bit products.  Seven
// rounds are the fewest for which the paper reports no failure in its statistical test batteries;
// its default of ten adds a margin that a mask of kept elements has no use for
// (65,537 x 1027 bf16 in both directions: 106 us with seven, 115 with ten).
//   key = the seed; counter = (column / 4, row, offset low, offset high); word column % 4 of the
// result decides element (row, column), whatever the strides, the type or the kernel that asks.
// ---------------------------------------------------------------------------------------------
constexpr int kPhiloxRounds = 7;

struct Mask {  // what the host knows of a dropout: `last` is the largest word that still drops
  const int64_t *rng;  // device {seed, offset}; nullptr: nothing is dropped
  uint32_t last;
  float inv_keep;  // 1 / (1 - p)
};

// p = 0: nothing to drop (no mask at all).  p = 1: every word drops.
static inline Mask make_mask(double p, const int64_t *d_rng) {
  const double t = p * 4294967296.0 + 0.5;
  const uint64_t threshold = t >= 4294967296.0 ? (1ull << 32) : (uint64_t)t;
  Mask m;
  m.rng = threshold > 0 ? d_rng : nullptr;
  m.last = threshold > 0 ? (uint32_t)(threshold - 1) : 0u;
  m.inv_keep = p < 1.0 ? (float)(1.0 / (1.0 - p)) : 0.f;
  return m;
}

struct MaskKey {
  uint32_t seed_lo, seed_hi, off_lo, off_hi;
};
__device__ __forceinline__ MaskKey mask_key(const int64_t *__restrict__ rng) {
  const uint64_t seed = (uint64_t)rng[0], off = (uint64_t)rng[1];
  return MaskKey{(uint32_t)seed, (uint32_t)(seed >> 32), (uint32_t)off, (uint32_t)(off >> 32)};
}

// one instruction with the truth table of a ^ b ^ c
__device__ __forceinline__ uint32_t xor3(uint32_t a, uint32_t b, uint32_t c) {
  return __builtin_amdgcn_bitop3_b32(a, b, c, 0x96);
}

// the four words of columns 4 * block .. 4 * block + 3 of `row`
__device__ __forceinline__ void mask_words(const MaskKey &k, uint32_t row, uint32_t block, uint32_t (&w)[4]) {
  uint32_t c0 = block, c1 = row, c2 = k.off_lo, c3 = k.off_hi, k0 = k.seed_lo, k1 = k.seed_hi;
#pragma unroll
  for (int r = 0; r < kPhiloxRounds; ++r) {
    const uint64_t a = (uint64_t)0xD2511F53u * c0, b = (uint64_t)0xCD9E8D57u * c2;
    c0 = xor3((uint32_t)(b >> 32), c1, k0);
    c2 = xor3((uint32_t)(a >> 32), c3, k1);
    c1 = (uint32_t)b;
    c3 = (uint32_t)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  w[0] = c0;
  w[1] = c1;
  w[2] = c2;
  w[3] = c3;
}
// bit i: the element in column j + i is kept (j a multiple of four)
template <int V>
__device__ __forceinline__ uint32_t keep_bits(const MaskKey &k, const Mask &m, int64_t row, int32_t j) {
  uint32_t bits = 0;
#pragma unroll
  for (int b = 0; b < V / 4; ++b) {
    uint32_t w[4];
    mask_words(k, (uint32_t)row, (uint32_t)(j / 4 + b), w);
#pragma unroll
    for (int i = 0; i < 4; ++i) bits |= w[i] > m.last ? 1u << (4 * b + i) : 0u;
  }
  return bits;
}

// v / (1 - p) for the kept elements of the chunk that starts at column j (a multiple of four), 0 for the others
template <int V>
__device__ __forceinline__ void drop_chunk(const MaskKey &k, const Mask &m, int64_t row, int32_t j, float (&v)[V]) {
#pragma unroll
  for (int b = 0; b < V / 4; ++b) {
    uint32_t w[4];
    mask_words(k, (uint32_t)row, (uint32_t)(j / 4 + b), w);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[4 * b + i] = w[i] > m.last ? v[4 * b + i] * m.inv_keep : 0.f;
  }
}

// ---------------------------------------------------------------------------------------------
// A lane's 16 bytes of a row.  Where the row ends inside them, or before them, the lane takes the row's last 16 bytes
// instead: the elements it repeats from the lane before (the first `dup`) are computed again, to the same bits, but
// count in no sum.  So every load and store is whole and none needs shifting into place.
// ---------------------------------------------------------------------------------------------
enum RowFit {
  kWholeChunks,  // rows of a whole number of chunks: a lane's elements count all or none (dup 0 or V)
  kPartChunk,    // others of at least one chunk
  kShortRow      // rows shorter than a chunk, moved element by element
};

template <typename T, int FIT>
struct Span {
  static constexpr int V = 16 / (int)sizeof(T);
  typedef typename Pack<T, V>::type vec;

  int32_t at, dup, d;

  __device__ __forceinline__ void place(int32_t j, int32_t d_) {
    d = d_;
    at = FIT == kShortRow ? 0 : (j < d - V ? j : d - V);
    dup = j - at < V ? j - at : V;
  }
  __device__ __forceinline__ bool any() const { return dup < V; }
  // all V elements lie in the row, repeated ones among them
  __device__ __forceinline__ bool whole() const { return FIT != kShortRow; }
  // element i of the lane counts
  __device__ __forceinline__ bool counts(int i) const {
    return FIT == kWholeChunks ? dup == 0 : FIT == kPartChunk ? i >= dup : dup == 0 && i < d;
  }
  __device__ __forceinline__ Raw load(const T *row) const {
    if (FIT != kShortRow) return __builtin_bit_cast(Raw, *reinterpret_cast<const vec *>(row + at));
    vec q = {};
#pragma unroll
    for (int i = 0; i < V; ++i) q[i] = row[i < d ? i : d - 1];
    return __builtin_bit_cast(Raw, q);
  }
  __device__ __forceinline__ void floats(Raw r, float (&out)[V]) const {
    const vec q = __builtin_bit_cast(vec, r);
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = (float)q[i];
  }
  __device__ __forceinline__ void write(T *row, const float (&in)[V]) const {
    vec q = {};
#pragma unroll
    for (int i = 0; i < V; ++i) q[i] = rounded<T>(in[i]);
    if (!any()) return;
    if (FIT != kShortRow) {
      *reinterpret_cast<vec *>(row + at) = q;
    } else {
#pragma unroll
      for (int i = 0; i < V - 1; ++i)
        if (i < d) row[i] = q[i];
    }
  }
  // sum of a * b over the elements that count
  __device__ __forceinline__ float dot(const float (&a)[V], const float (&b)[V]) const {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) s += FIT == kWholeChunks || counts(i) ? a[i] * b[i] : 0.f;
    return FIT != kWholeChunks || dup == 0 ? s : 0.f;
  }
  // a weight vector's elements, ones for a null pointer
  __device__ __forceinline__ void weights(const void *w, int w_f32, float (&out)[V]) const {
    if (!w) {
#pragma unroll
      for (int i = 0; i < V; ++i) out[i] = 1.f;
    } else if (FIT == kShortRow) {
#pragma unroll
      for (int i = 0; i < V; ++i) out[i] = weight_at<T>(w, w_f32, i < d ? i : d - 1);
    } else if (w_f32) {
      load_pack<float, V>(static_cast<const float *>(w) + at, out);
    } else {
      load_pack<T, V>(static_cast<const T *>(w) + at, out);
    }
  }
  // v / (1 - p) for kept elements, 0 for dropped ones.  The generator decides aligned groups of four columns; where the
  // lane's columns are not aligned, the decisions of its own V columns and of the V before are shifted together.
  __device__ __forceinline__ void drop(const MaskKey &key, const Mask &m, int64_t row, float (&v)[V]) const {
    if (FIT != kPartChunk) {
      drop_chunk<V>(key, m, row, at, v);
      return;
    }
    const int32_t j = at + dup;  // the aligned columns the lane would have without the row's end (dup < V)
    uint32_t bits = keep_bits<V>(key, m, row, j);
    if (dup > 0 && dup < V) bits = ((bits << V) | keep_bits<V>(key, m, row, j - V)) >> (V - dup);
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = (bits >> i) & 1u ? v[i] * m.inv_keep : 0.f;
  }
};

// ---- argument checks shared by the entry points ---------------------------------------------------
static inline int check_dtype(const char *who, int dtype) {
  if (dtype != CG_F32 && dtype != CG_BF16 && dtype != CG_F16)
    CG_FAIL(CG_ERR_UNSUPPORTED, "%s: dtype %d is none of CG_F32, CG_BF16, CG_F16", who, dtype);
  return CG_OK;
}
static inline int check_row_shape(const char *who, int64_t n, int32_t d) {
  if (n < 0 || d <= 0) CG_FAIL(CG_ERR_SIZE, "%s: n=%lld rows of d=%d elements", who, (long long)n, d);
  if (n > 0xffffffffLL) CG_FAIL(CG_ERR_OVERFLOW, "%s: n=%lld rows (at most 2^32 - 1)", who, (long long)n);
  return CG_OK;
}
static inline int check_work(const char *who, const void *d_work, int64_t have, int64_t need) {
  if (have < need) CG_FAIL(CG_ERR_SIZE, "%s: workspace of %lld bytes, %lld needed", who, (long long)have, (long long)need);
  if ((uintptr_t)d_work % 16 != 0) CG_FAIL(CG_ERR_UNSUPPORTED, "%s: the workspace is not 16-byte aligned", who);
  return CG_OK;
}
static inline int check_p(const char *who, double p, const int64_t *d_rng) {
  if (!(p >= 0.0 && p <= 1.0)) CG_FAIL(CG_ERR_SIZE, "%s: dropout probability %g outside [0, 1]", who, p);
  if (p > 0.0 && !d_rng) CG_FAIL(CG_ERR_NULL, "%s: p > 0 without generator state", who);
  return CG_OK;
}
static inline size_t elem_size(int dtype) { return dtype == CG_F32 ? 4 : 2; }

// calls F<dtype constant>
#define CG_BY_DTYPE(dtype, CALL)          \
  switch (dtype) {                        \
    case CG_F32: CALL(CG_F32); break;     \
    case CG_BF16: CALL(CG_BF16); break;   \
    default: CALL(CG_F16); break;         \
  }

}  // namespace cg
