// Arguments, reductions and the choice of lanes per row of the norm kernels (norm.hip, norm_fwd.hip, norm_bwd.hip).
#pragma once
#include "rows.h"

namespace cg {

constexpr int kNormThreads = 256;
constexpr int kNormWaves = kNormThreads / kWave;

// Arguments of either operator, forward and backward; rms_norm uses the z side as its input x and leaves the rest
// at its defaults.
struct NormArgs {
  const void *z, *x, *gate, *dr, *dh, *r_in;
  void *r, *h, *dz, *dx, *dgate;
  int64_t ldz, ldx, ldgate, lddr, lddh, ldr_in, ldr, ldh, lddz, lddx, lddgate;
  const void *w_post, *w_pre, *scale;
  int w_f32, gate_kind;
  float alpha, eps;
  float *rstd_z, *rstd_r;  // written forward, read backward
  float *partial;          // backward: one slice per workgroup, [d] of q and for the residual block [d] of dw_pre
  Mask mask;
  int64_t n;
  int32_t d;
};

// Lanes that share a row and 16-byte chunks each of them holds.  Rows of up to 64 chunks are taken by the smallest
// power of two of lanes (at least 4) that covers them with one chunk each, several rows per wavefront; longer rows by a
// whole wavefront with up to 16 elements a lane; then by a workgroup of as many wavefronts as the row fills, at most 8,
// with 16 elements a lane.  The gradient of the residual block keeps five operands of a row and four column vectors in
// registers: 8 elements a lane let three or four wavefronts run on a SIMD instead of two, and it takes 16 only where 8
// wavefronts of 8 are too few.  lanes == 0: the row does not fit and is read again for every pass over it.
constexpr int kNormMaxWaves = 8;

struct NormShape {
  int lanes, chunks;
  int threads;  // of a workgroup
  bool whole;   // the workgroup holds one row at a time
};
static inline NormShape norm_shape(int32_t d, int dtype, bool residual_bwd) {
  const int v = dtype == CG_F32 ? 4 : 8;
  const int64_t c = ceil_div64(d, v);
  if (c <= kWave) {
    int lanes = 4;
    while (lanes < c) lanes *= 2;
    return NormShape{lanes, 1, kNormThreads, false};
  }
  const int most = 16 / v;  // chunks of 16 elements a lane
  if (c <= (int64_t)kWave * most) return NormShape{kWave, (int)ceil_div64(c, kWave), kNormThreads, false};
  for (int chunks = residual_bwd ? most / 2 : most; chunks <= most; chunks *= 2) {
    const int64_t waves = ceil_div64(c, (int64_t)kWave * chunks);
    if (waves <= kNormMaxWaves) return NormShape{kWave, chunks, (int)waves * kWave, true};
  }
  return NormShape{0, 0, 512, true};
}
static inline int norm_rows_at_once(const NormShape &s) { return s.whole ? 1 : s.threads / s.lanes; }

int launch_norm_fwd(const NormArgs &a, bool residual, int dtype, hipStream_t s);
int launch_norm_bwd(const NormArgs &a, bool residual, int dtype, int64_t groups, hipStream_t s);

// Sum over the lanes of a row.  Teams inside a wavefront exchange registers; a whole workgroup goes through `slots`,
// whose halves alternate from one reduction to the next, so that one barrier a reduction is enough: a half is written
// again only after everybody has passed the barrier of the reduction in between, hence has read it.
typedef float NormSlots[2][kNormMaxWaves];

template <int LANES, bool WHOLE>
__device__ __forceinline__ float row_sum(float v, NormSlots &slots, int &turn) {
  v = team_sum_of<LANES>(v);
  if (!WHOLE) return v;
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave, waves = blockDim.x / kWave;
  if (lane == 0) slots[turn][wave] = v;
  __syncthreads();
  float s = 0.f;
  for (int w = 0; w < waves; ++w) s += slots[turn][w];
  turn ^= 1;
  return s;
}

// 1 / (1 + 2^(-a log2 e)).  The hardware's exponential and reciprocal are within one unit of the last place; the
// rounding of the exponent adds |a| roundings to e^-a, which for a > 0 is the small term of the sum and for a < 0 leaves
// a result below e^a off by |a| e^a units.
__device__ __forceinline__ float sigmoid(float a) {
  return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(a * -1.44269504f));
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

}  // namespace cg
