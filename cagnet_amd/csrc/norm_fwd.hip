// Forward pass of rms_norm and norm_residual with the row in registers: every operand is read once and every result
// written once, the statistics come from the registers in between.  Lanes and chunks per row: norm_shape.  The waves
// loop over rows, all of them side by side through memory, with their columns' weights in registers.
#include "norm_kernels.h"

namespace cg {

// 128 registers or fewer let four wavefronts run on a SIMD, 168 three: the bounds hold the compiler to what it misses by
// a few registers otherwise.
template <int DT, int LANES, int K, bool WHOLE, int FIT, bool RESIDUAL>
__global__ __launch_bounds__(WHOLE ? kWave * kNormMaxWaves : kNormThreads, !RESIDUAL ? 1 : (DT != CG_F32 && K == 2) || K == 3 ? 4 : 3) void norm_fwd_kernel(NormArgs a) {
  typedef typename Elem<DT>::type T;
  typedef Span<T, FIT> C;
  constexpr int V = C::V, TEAMS = WHOLE ? 1 : kNormThreads / LANES;
  __shared__ NormSlots slots;
  int turn = 0;
  const int lane = WHOLE ? threadIdx.x : threadIdx.x % LANES, team = WHOLE ? 0 : threadIdx.x / LANES;
  const int lanes = WHOLE ? blockDim.x : LANES;
  C c[K];
  float wz[K][V], wr[K][V];  // alpha scale w_post (w_post alone for rms_norm) and w_pre
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
      s += c[k].dot(v[k], v[k]);
    }
    const float rho_z = rsqrtf(row_sum<LANES, WHOLE>(s, slots, turn) * inv_d + a.eps);
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
      if (a.mask.rng)
        c[k].drop(key, a.mask, row, v[k]);
      c[k].floats(rx[k], x);
#pragma unroll
      for (int i = 0; i < V; ++i) v[k][i] += x[i];
      s += c[k].dot(v[k], v[k]);
      c[k].write((T *)a.r + row * a.ldr, v[k]);
    }
    const float rho_r = rsqrtf(row_sum<LANES, WHOLE>(s, slots, turn) * inv_d + a.eps);
    if (lane == 0) a.rstd_r[row] = rho_r;
#pragma unroll
    for (int k = 0; k < K; ++k) {  // h comes from the sum before its rounding to the stored type
#pragma unroll
      for (int i = 0; i < V; ++i) v[k][i] *= rho_r * wr[k][i];
      c[k].write((T *)a.h + row * a.ldh, v[k]);
    }
  }
}

template <int DT, int LANES, int K, bool WHOLE, int FIT>
static int go_fit(const NormArgs &a, bool residual, const NormShape &sh, int64_t groups, hipStream_t s) {
  if (residual)
    norm_fwd_kernel<DT, LANES, K, WHOLE, FIT, true><<<(unsigned)groups, sh.threads, 0, s>>>(a);
  else
    norm_fwd_kernel<DT, LANES, K, WHOLE, FIT, false><<<(unsigned)groups, sh.threads, 0, s>>>(a);
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
static int go_shape(const NormArgs &a, bool residual, hipStream_t s) {
  constexpr int MOST = DT == CG_F32 ? 4 : 2;  // chunks of 16 elements
  const NormShape sh = norm_shape(a.d, DT, false);
  // Few rows a wave: the loads of a wave's next row would wait for the stores of the row before (they are counted
  // together and in order), those of a new wave do not.  124,584 x 602 float32: 242 us with 8 workgroups per compute unit
  // in all, 228 with 32, 210 with 128.  Partial chunks of 16-bit elements pay more per wave for their weights and
  // addresses: 249,169 x 602 bf16 with dropout 328 us with 8 or 32, 397 with 128.
  const bool costly = residual && DT != CG_F32 && !sh.whole && a.d % 8 != 0;
  const int64_t want = ceil_div64(a.n, norm_rows_at_once(sh));
  const int64_t most = sh.whole ? 256 * 256 / (sh.threads / kWave) : costly ? 256 * 32 : 256 * 128;
  const int64_t groups = want < most ? want : most;
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

int launch_norm_fwd(const NormArgs &a, bool residual, int dtype, hipStream_t s) {
  if (dtype == CG_F32) return go_shape<CG_F32>(a, residual, s);
  if (dtype == CG_BF16) return go_shape<CG_BF16>(a, residual, s);
  return go_shape<CG_F16>(a, residual, s);
}

}  // namespace cg
