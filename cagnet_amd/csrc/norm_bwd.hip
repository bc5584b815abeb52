// Gradients of rms_norm and norm_residual with the row in registers: every operand is read once and every result
// written once.  The gradients of the weights are sums over all rows: each lane adds its columns up over the rows its
// team takes, the teams and wavefronts of a workgroup are added at the end, and one slice per workgroup goes to memory
// (norm_weight_grads_kernel adds the slices).
#include "norm_kernels.h"

namespace cg {

// the workgroup's columns of one sum, added over its teams in a fixed order, to dst[0..d)
template <typename C, int LANES, int K, bool WHOLE>
__device__ __forceinline__ void fold_columns(float (&acc)[K][C::V], const C (&c)[K], float *lds, float *__restrict__ dst,
                                             int32_t d) {
  constexpr int V = C::V;
  if (WHOLE) {  // every column belongs to one lane
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (c[k].counts(i)) dst[c[k].at + i] = acc[k][i];
    return;
  }
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < V; ++i) {
#pragma unroll
      for (int off = LANES; off < kWave; off <<= 1) acc[k][i] += __shfl_xor(acc[k][i], off, kWave);
      if (lane < LANES && c[k].counts(i)) lds[wave * (LANES * K * V) + c[k].at + i] = acc[k][i];
    }
  __syncthreads();
  for (int j = threadIdx.x; j < d; j += kNormThreads) {
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < kNormWaves; ++w) s += lds[w * (LANES * K * V) + j];
    dst[j] = s;
  }
  __syncthreads();
}

// The bound on registers, where 8 elements of 16 bits a lane miss it by a few: four wavefronts a SIMD for rows of whole
// chunks (2,343,750 x 64 bf16: 420 us without, 353 with), three for others, which would have to spill for the fourth
// (3,658,536 x 41 bf16 with row gates and dropout: 872 us with four, 705 with three).  In float32 the
// bounds only keep the compiler from taking a register or two too many for them (nothing is spilled).
template <int DT, int K, bool WHOLE, int FIT, bool RESIDUAL>
constexpr int bwd_waves() {
  if (!RESIDUAL || WHOLE) return 1;
  if (DT == CG_F32) return K == 1 ? 5 : FIT != kWholeChunks ? 1 : K == 2 ? 4 : 2;
  return K > 1 ? 1 : FIT == kPartChunk ? 3 : 4;
}

template <int DT, int LANES, int K, bool WHOLE, int FIT, bool RESIDUAL>
__global__ __launch_bounds__(WHOLE ? kWave * kNormMaxWaves : kNormThreads,
                             (bwd_waves<DT, K, WHOLE, FIT, RESIDUAL>())) void norm_bwd_kernel(NormArgs a) {
  typedef typename Elem<DT>::type T;
  typedef Span<T, FIT> C;
  constexpr int V = C::V, TEAMS = WHOLE ? 1 : kNormThreads / LANES;
  __shared__ NormSlots slots;
  __shared__ float lds[WHOLE ? 1 : kNormWaves * LANES * K * V];
  int turn = 0;
  // Where a wavefront holds one row its number is made uniform, which moves the row's addresses to the scalar unit:
  // 250,000 x 300 float32 with row gates and dropout 432 -> 365 us.  With 16 elements a lane the scalar registers run
  // out and it costs instead (249,169 x 602 bf16: 417 -> 457 us).
  constexpr bool UNIFORM = !WHOLE && LANES == kWave && K * V < 16;
  const int lane = WHOLE ? threadIdx.x : threadIdx.x % LANES;
  const int team = WHOLE ? 0 : UNIFORM ? __builtin_amdgcn_readfirstlane(threadIdx.x / kWave) : threadIdx.x / LANES;
  const int lanes = WHOLE ? blockDim.x : LANES;
  C c[K];
  float wz[K][V], wr[K][V], q[K][V], p[K][V];  // alpha scale w_post (w_post alone for rms_norm), w_pre, column sums
#pragma unroll
  for (int k = 0; k < K; ++k) {
    c[k].place((lane + k * lanes) * V, a.d);
    c[k].weights(a.w_post, a.w_f32, wz[k]);
    if (RESIDUAL) {
      float s[V];
      c[k].weights(a.scale, a.w_f32, s);
      c[k].weights(a.w_pre, a.w_f32, wr[k]);
#pragma unroll
      for (int i = 0; i < V; ++i) wz[k][i] *= a.alpha * s[i];
    }
#pragma unroll
    for (int i = 0; i < V; ++i) q[k][i] = p[k][i] = 0.f;
  }
  const float inv_d = 1.f / (float)a.d;
  MaskKey key = {0, 0, 0, 0};
  if (RESIDUAL && a.mask.rng) key = mask_key(a.mask.rng);
  const int64_t step = (int64_t)gridDim.x * TEAMS;
  for (int64_t row = (int64_t)blockIdx.x * TEAMS + team; row < a.n; row += step) {
    Raw rz[K], rdh[K], rr[K], rdr[K], rg[K];
#pragma unroll
    for (int k = 0; k < K; ++k) rz[k] = c[k].load((const T *)a.z + row * a.ldz);
    if (!RESIDUAL || a.dh) {
#pragma unroll
      for (int k = 0; k < K; ++k) rdh[k] = c[k].load((const T *)a.dh + row * a.lddh);
    }
    const float rho_z = a.rstd_z[row];
    if (!RESIDUAL) {
      float zh[K][V], t[K][V], s = 0.f;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        c[k].floats(rz[k], zh[k]);
        c[k].floats(rdh[k], t[k]);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          zh[k][i] *= rho_z;
          q[k][i] += t[k][i] * zh[k][i];
          t[k][i] *= wz[k][i];
        }
        s += c[k].dot(t[k], zh[k]);
      }
      const float m = row_sum<LANES, WHOLE>(s, slots, turn) * inv_d;
#pragma unroll
      for (int k = 0; k < K; ++k) {
#pragma unroll
        for (int i = 0; i < V; ++i) t[k][i] = rho_z * (t[k][i] - zh[k][i] * m);
        c[k].write((T *)a.dz + row * a.lddz, t[k]);
      }
      continue;
    }
    if (a.dh) {
#pragma unroll
      for (int k = 0; k < K; ++k) rr[k] = c[k].load((const T *)a.r_in + row * a.ldr_in);
    }
    if (a.dr) {
#pragma unroll
      for (int k = 0; k < K; ++k) rdr[k] = c[k].load((const T *)a.dr + row * a.lddr);
    }
    float row_gate = 0.f;
    if (a.gate_kind == CG_GATE_FULL) {
#pragma unroll
      for (int k = 0; k < K; ++k) rg[k] = c[k].load((const T *)a.gate + row * a.ldgate);
    } else if (a.gate_kind == CG_GATE_ROW) {
      row_gate = (float)((const T *)a.gate)[row * a.ldgate];
    }
    float D[K][V], zh[K][V];  // gradient of the residual sum; the normalised block output
    if (a.dh) {
      const float rho_r = a.rstd_r[row];
      float rh[K][V], s = 0.f;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        c[k].floats(rdh[k], D[k]);
        c[k].floats(rr[k], rh[k]);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          rh[k][i] *= rho_r;
          p[k][i] += D[k][i] * rh[k][i];
          D[k][i] *= wr[k][i];
        }
        s += c[k].dot(D[k], rh[k]);
      }
      const float m = row_sum<LANES, WHOLE>(s, slots, turn) * inv_d;
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) D[k][i] = rho_r * (D[k][i] - rh[k][i] * m);
    } else {
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) D[k][i] = 0.f;
    }
    if (a.dr) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        float g[V];
        c[k].floats(rdr[k], g);
#pragma unroll
        for (int i = 0; i < V; ++i) D[k][i] += g[i];
      }
    }
    float row_slope = 0.f;
    const float row_sig = a.gate_kind == CG_GATE_ROW ? sigmoid(row_gate, row_slope) : 1.f;
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      c[k].write((T *)a.dx + row * a.lddx, D[k]);
      c[k].floats(rz[k], zh[k]);
      if (a.mask.rng)
        c[k].drop(key, a.mask, row, D[k]);
#pragma unroll
      for (int i = 0; i < V; ++i) zh[k][i] *= rho_z;
      if (a.gate_kind == CG_GATE_FULL) {
        float g[V];
        c[k].floats(rg[k], g);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          float slope;
          const float sig = sigmoid(g[i], slope), e = D[k][i] * wz[k][i];
          q[k][i] += D[k][i] * sig * zh[k][i];
          g[i] = e * zh[k][i] * slope;
          D[k][i] = e * sig;
        }
        c[k].write((T *)a.dgate + row * a.lddgate, g);
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          q[k][i] += D[k][i] * row_sig * zh[k][i];
          D[k][i] *= wz[k][i];
        }
      }
      s += c[k].dot(D[k], zh[k]);
    }
    s = row_sum<LANES, WHOLE>(s, slots, turn);
    if (a.gate_kind == CG_GATE_ROW && lane == 0) ((T *)a.dgate)[row * a.lddgate] = rounded<T>(s * row_slope);
    const float m = s * inv_d, rho_s = rho_z * row_sig;
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
      for (int i = 0; i < V; ++i) D[k][i] = rho_s * (D[k][i] - zh[k][i] * m);
      c[k].write((T *)a.dz + row * a.lddz, D[k]);
    }
  }
  float *slice = a.partial + (int64_t)blockIdx.x * (RESIDUAL ? 2 : 1) * a.d;
  fold_columns<C, LANES, K, WHOLE>(q, c, lds, slice, a.d);
  if (RESIDUAL) fold_columns<C, LANES, K, WHOLE>(p, c, lds, slice + a.d, a.d);
}

template <int DT, int LANES, int K, bool WHOLE, int FIT>
static int go_fit(const NormArgs &a, bool residual, const NormShape &sh, int64_t groups, hipStream_t s) {
  if (residual)
    norm_bwd_kernel<DT, LANES, K, WHOLE, FIT, true><<<(unsigned)groups, sh.threads, 0, s>>>(a);
  else
    norm_bwd_kernel<DT, LANES, K, WHOLE, FIT, false><<<(unsigned)groups, sh.threads, 0, s>>>(a);
  CG_LAUNCH_CHECK();
  return CG_OK;
}

template <int DT, int LANES, int K, bool WHOLE>
static int go(const NormArgs &a, bool residual, const NormShape &sh, int64_t groups, hipStream_t s) {
  constexpr int V = DT == CG_F32 ? 4 : 8;
  if (a.d % V == 0) return go_fit<DT, LANES, K, WHOLE, kWholeChunks>(a, residual, sh, groups, s);
  if (LANES == 4 && a.d < V) return go_fit<DT, 4, 1, false, kShortRow>(a, residual, sh, groups, s);
  return go_fit<DT, LANES, K, WHOLE, kPartChunk>(a, residual, sh, groups, s);
}

template <int DT>
static int go_shape(const NormArgs &a, bool residual, int64_t groups, hipStream_t s) {
  constexpr int MOST = DT == CG_F32 ? 4 : 2;  // chunks of 16 elements
  const NormShape sh = norm_shape(a.d, DT, residual);
  if (sh.whole && sh.chunks < MOST) return go<DT, kWave, MOST / 2, true>(a, residual, sh, groups, s);
  if (sh.whole) return go<DT, kWave, MOST, true>(a, residual, sh, groups, s);
  if (sh.lanes == 4) return go<DT, 4, 1, false>(a, residual, sh, groups, s);
  if (sh.lanes == 8) return go<DT, 8, 1, false>(a, residual, sh, groups, s);
  if (sh.lanes == 16) return go<DT, 16, 1, false>(a, residual, sh, groups, s);
  if (sh.lanes == 32) return go<DT, 32, 1, false>(a, residual, sh, groups, s);
  if (sh.chunks == 1) return go<DT, kWave, 1, false>(a, residual, sh, groups, s);
  if (sh.chunks == 2) return go<DT, kWave, 2, false>(a, residual, sh, groups, s);
  if (MOST > 2 && sh.chunks == 3) return go<DT, kWave, MOST - 1, false>(a, residual, sh, groups, s);
  return go<DT, kWave, MOST, false>(a, residual, sh, groups, s);
}

int launch_norm_bwd(const NormArgs &a, bool residual, int dtype, int64_t groups, hipStream_t s) {
  if (dtype == CG_F32) return go_shape<CG_F32>(a, residual, groups, s);
  if (dtype == CG_BF16) return go_shape<CG_BF16>(a, residual, groups, s);
  return go_shape<CG_F16>(a, residual, groups, s);
}

}  // namespace cg
