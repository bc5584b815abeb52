// Forward pass of rms_norm and norm_residual with the row in registers: every operand is read once and every result
// written once, the statistics come from the registers in between.  Lanes and chunks per row: norm_shape.  The waves
// loop over rows (all of them side by side through memory) and keep their columns' weights in registers.
#include "norm_kernels.h"

namespace cg {

template <int DT, int LANES, int K, bool RESIDUAL>
__global__ __launch_bounds__(kNormThreads) void norm_fwd_kernel(NormArgs a) {
  typedef typename Elem<DT>::type T;
  typedef Chunk<T> C;
  constexpr int V = C::V, TEAMS = kNormThreads / LANES;
  __shared__ float slots[2][kNormWaves];
  int turn = 0;
  const int lane = threadIdx.x % LANES, team = threadIdx.x / LANES;
  C c[K];
  float wz[K][V], wr[K][V];  // alpha scale w_post (w_post alone for rms_norm) and w_pre
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int32_t j = (lane + k * LANES) * V;
    c[k].place(j, a.d);
    weight_chunk<T>(a.w_post, a.w_f32, j, c[k].live, wz[k]);
    if (RESIDUAL) {
      float s[V];
      weight_chunk<T>(a.scale, a.w_f32, j, c[k].live, s);
      weight_chunk<T>(a.w_pre, a.w_f32, j, c[k].live, wr[k]);
#pragma unroll
      for (int i = 0; i < V; ++i) wz[k][i] *= a.alpha * s[i];
    }
  }
  const float inv_d = 1.f / (float)a.d;
  MaskKey key = {0, 0, 0, 0};
  if (RESIDUAL && a.mask.rng) key = mask_key(a.mask.rng);
  const int64_t step = (int64_t)gridDim.x * TEAMS;
  for (int64_t row = (int64_t)blockIdx.x * TEAMS + team; row < a.n; row += step) {
    Raw rz[K], rx[K], rg[K];
#pragma unroll
    for (int k = 0; k < K; ++k) rz[k] = c[k].load((const T *)a.z + row * a.ldz);
    float row_gate = 1.f;
    if (RESIDUAL) {
#pragma unroll
      for (int k = 0; k < K; ++k) rx[k] = c[k].load((const T *)a.x + row * a.ldx);
      if (a.gate_kind == CG_GATE_FULL) {
#pragma unroll
        for (int k = 0; k < K; ++k) rg[k] = c[k].load((const T *)a.gate + row * a.ldgate);
      } else if (a.gate_kind == CG_GATE_ROW) {
        row_gate = (float)((const T *)a.gate)[row * a.ldgate];
      }
    }
    float v[K][V], s = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      c[k].floats(rz[k], v[k]);
#pragma unroll
      for (int i = 0; i < V; ++i) s += v[k][i] * v[k][i];
    }
    const float rho_z = rsqrtf(row_sum<LANES>(s, slots, turn) * inv_d + a.eps);
    if (lane == 0) a.rstd_z[row] = rho_z;
    if (!RESIDUAL) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
#pragma unroll
        for (int i = 0; i < V; ++i) v[k][i] *= rho_z * wz[k][i];
        c[k].write((T *)a.h + row * a.ldh, v[k]);
      }
      continue;
    }
    const float rho_s = a.gate_kind == CG_GATE_ROW ? rho_z * sigmoid(row_gate) : rho_z;
    s = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float x[V];
#pragma unroll
      for (int i = 0; i < V; ++i) v[k][i] *= rho_s * wz[k][i];
      if (a.gate_kind == CG_GATE_FULL) {
        float g[V];
        c[k].floats(rg[k], g);
#pragma unroll
        for (int i = 0; i < V; ++i) v[k][i] *= sigmoid(g[i]);
      }
      if (a.mask.rng) {
        float m[V];
        mask_chunk<V>(key, a.mask, row, (lane + k * LANES) * V, m);
#pragma unroll
        for (int i = 0; i < V; ++i) v[k][i] = m[i] > 0.f ? v[k][i] * m[i] : 0.f;
      }
      c[k].floats(rx[k], x);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        v[k][i] += x[i];
        s += v[k][i] * v[k][i];
      }
      c[k].write((T *)a.r + row * a.ldr, v[k]);
    }
    const float rho_r = rsqrtf(row_sum<LANES>(s, slots, turn) * inv_d + a.eps);
    if (lane == 0) a.rstd_r[row] = rho_r;
#pragma unroll
    for (int k = 0; k < K; ++k) {  // h comes from the sum before its rounding to the stored type
#pragma unroll
      for (int i = 0; i < V; ++i) v[k][i] *= rho_r * wr[k][i];
      c[k].write((T *)a.h + row * a.ldh, v[k]);
    }
  }
}

template <int DT, int LANES, int K>
static int go(const NormArgs &a, bool residual, hipStream_t s) {
  const int64_t want = ceil_div64(a.n, kNormThreads / LANES);
  const unsigned groups = (unsigned)(want < 256 * 8 ? want : 256 * 8);
  if (residual)
    norm_fwd_kernel<DT, LANES, K, true><<<groups, kNormThreads, 0, s>>>(a);
  else
    norm_fwd_kernel<DT, LANES, K, false><<<groups, kNormThreads, 0, s>>>(a);
  CG_LAUNCH_CHECK();
  return CG_OK;
}

template <int DT>
static int go_shape(const NormArgs &a, bool residual, const NormShape &sh, hipStream_t s) {
  constexpr bool F32 = DT == CG_F32;
  switch (sh.lanes * 16 + sh.chunks) {
    case 4 * 16 + 1: return go<DT, 4, 1>(a, residual, s);
    case 8 * 16 + 1: return go<DT, 8, 1>(a, residual, s);
    case 16 * 16 + 1: return go<DT, 16, 1>(a, residual, s);
    case 32 * 16 + 1: return go<DT, 32, 1>(a, residual, s);
    case 64 * 16 + 1: return go<DT, 64, 1>(a, residual, s);
    case 64 * 16 + 2: return go<DT, 64, 2>(a, residual, s);
    case 64 * 16 + 3: if (F32) return go<DT, 64, F32 ? 3 : 1>(a, residual, s); break;
    case 64 * 16 + 4: if (F32) return go<DT, 64, F32 ? 4 : 1>(a, residual, s); break;
    case 256 * 16 + 1: if (!F32) return go<DT, 256, 1>(a, residual, s); break;
    case 256 * 16 + 2: return go<DT, 256, 2>(a, residual, s);
    case 256 * 16 + 3: return go<DT, 256, 3>(a, residual, s);
    case 256 * 16 + 4: return go<DT, 256, 4>(a, residual, s);
    case 256 * 16 + 5: if (F32) return go<DT, 256, F32 ? 5 : 2>(a, residual, s); break;
    case 256 * 16 + 6: if (F32) return go<DT, 256, F32 ? 6 : 2>(a, residual, s); break;
    case 256 * 16 + 7: if (F32) return go<DT, 256, F32 ? 7 : 2>(a, residual, s); break;
    case 256 * 16 + 8: if (F32) return go<DT, 256, F32 ? 8 : 2>(a, residual, s); break;
  }
  CG_FAIL(CG_ERR_UNSUPPORTED, "norm: no kernel for %d lanes of %d chunks", sh.lanes, sh.chunks);
}

int launch_norm_fwd(const NormArgs &a, bool residual, int dtype, hipStream_t s) {
  const NormShape sh = norm_shape(a.d, dtype);
  if (dtype == CG_F32) return go_shape<CG_F32>(a, residual, sh, s);
  if (dtype == CG_BF16) return go_shape<CG_BF16>(a, residual, sh, s);
  return go_shape<CG_F16>(a, residual, sh, s);
}

}  // namespace cg
