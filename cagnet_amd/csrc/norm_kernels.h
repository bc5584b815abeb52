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
// The same with its derivative s (1 - s).  With s rounded to 24 bits, 1 - s has lost its leading digits where s is near 1
// (at a = 10 about a thousandth of it is wrong, from 17 on it is 0); there e^-a s is the same number without a difference.
// Up to a half 1 - s is exact to a rounding, and e^-a can be infinite.
__device__ __forceinline__ float sigmoid(float a, float &slope) {
  const float e = __builtin_amdgcn_exp2f(a * -1.44269504f), s = __builtin_amdgcn_rcpf(1.f + e);
  slope = s * (s > 0.5f ? e * s : 1.f - s);
  return s;
}

}  // namespace cg
