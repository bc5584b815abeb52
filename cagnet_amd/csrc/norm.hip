// Root-mean-square norms of rows, alone (rms_norm) and on both sides of a residual block (norm_residual):
//   rms_norm       y = x rho w,                                        rho = 1 / sqrt(mean(x^2) + eps)
//   norm_residual  u = alpha scale keep(sigmoid(gate) z rho_z w_post),  r = x + u,  h = r rho_r w_pre
// and their gradients.  With t = g w and xh = x rho, dx = rho (t - xh mean(t xh)) and dw = sum over rows of g xh.
// Statistics, sums and everything between a load and the one rounding at a store are float32.
#include "norm_kernels.h"

namespace cg {

// ---------------------------------------------------------------------------------------------
// Rows too long for registers: one workgroup per row, 16 bytes a lane and step, the row read again for every pass over it
// (it comes from the L2 cache then).
// ---------------------------------------------------------------------------------------------
constexpr int kLongThreads = 512;

template <int DT, bool RESIDUAL>
__global__ __launch_bounds__(kLongThreads) void norm_fwd_rows_kernel(NormArgs a) {
  typedef typename Elem<DT>::type T;
  typedef Span<T, kPartChunk> C;
  constexpr int V = C::V;
  __shared__ NormSlots slots;
  int turn = 0;
  const int32_t step = kLongThreads * V, start = threadIdx.x * V;
  MaskKey key = {0, 0, 0, 0};
  if (RESIDUAL && a.mask.rng) key = mask_key(a.mask.rng);
  for (int64_t row = blockIdx.x; row < a.n; row += gridDim.x) {
    const T *z = (const T *)a.z + row * a.ldz, *x = (const T *)a.x + row * a.ldx, *gate = (const T *)a.gate + row * a.ldgate;
    C c;
    float s = 0.f;
    for (int32_t j = start; j < a.d; j += step) {
      float v[V];
      c.place(j, a.d);
      c.floats(c.load(z), v);
      s += c.dot(v, v);
    }
    const float rho_z = rsqrtf(row_sum<kWave, true>(s, slots, turn) / (float)a.d + a.eps);
    if (threadIdx.x == 0) a.rstd_z[row] = rho_z;
    if (!RESIDUAL) {
      for (int32_t j = start; j < a.d; j += step) {
        float v[V], w[V];
        c.place(j, a.d);
        c.floats(c.load(z), v);
        c.weights(a.w_post, a.w_f32, w);
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] *= rho_z * w[i];
        c.write((T *)a.h + row * a.ldh, v);
      }
      continue;
    }
    const float row_sig = a.gate_kind == CG_GATE_ROW ? sigmoid((float)gate[0]) : 1.f;
    auto sum_at = [&](float (&v)[V]) {  // x + u in the columns of c
      float w[V], t[V];
      c.floats(c.load(z), v);
      c.weights(a.w_post, a.w_f32, w);
      c.weights(a.scale, a.w_f32, t);
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] *= rho_z * row_sig * (w[i] * (a.alpha * t[i]));
      if (a.gate_kind == CG_GATE_FULL) {
        c.floats(c.load(gate), t);
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] *= sigmoid(t[i]);
      }
      if (a.mask.rng) c.drop(key, a.mask, row, v);
      c.floats(c.load(x), t);
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] += t[i];
    };
    s = 0.f;
    for (int32_t j = start; j < a.d; j += step) {
      float v[V];
      c.place(j, a.d);
      sum_at(v);
      s += c.dot(v, v);
      c.write((T *)a.r + row * a.ldr, v);
    }
    const float rho_r = rsqrtf(row_sum<kWave, true>(s, slots, turn) / (float)a.d + a.eps);
    if (threadIdx.x == 0) a.rstd_r[row] = rho_r;
    for (int32_t j = start; j < a.d; j += step) {  // h comes from the sum before its rounding to the stored type
      float v[V], w[V];
      c.place(j, a.d);
      sum_at(v);
      c.weights(a.w_pre, a.w_f32, w);
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] *= rho_r * w[i];
      c.write((T *)a.h + row * a.ldh, v);
    }
  }
}

// The gradients of the weights are sums over rows: every workgroup adds its rows up in its own slice of `partial`
// (each column belongs to one thread), and a second kernel adds the slices in order.
template <int DT, bool RESIDUAL>
__global__ __launch_bounds__(kLongThreads) void norm_bwd_rows_kernel(NormArgs a) {
  typedef typename Elem<DT>::type T;
  typedef Span<T, kPartChunk> C;
  constexpr int V = C::V;
  __shared__ NormSlots slots;
  int turn = 0;
  const int32_t step = kLongThreads * V, start = threadIdx.x * V;
  MaskKey key = {0, 0, 0, 0};
  if (RESIDUAL && a.mask.rng) key = mask_key(a.mask.rng);
  float *q = a.partial + (int64_t)blockIdx.x * (RESIDUAL ? 2 : 1) * a.d, *p = q + a.d;
  C c;
  bool first = true;
  auto add_to = [&](float *sums, const float (&v)[V]) {  // the workgroup's first row writes
    float old[V];
    if (c.dup == 0) {
#pragma unroll
      for (int i = 0; i < V; ++i) old[i] = 0.f;
      if (!first) load_pack<float, V>(sums + c.at, old);
#pragma unroll
      for (int i = 0; i < V; ++i) old[i] += v[i];
      store_pack<float, V>(sums + c.at, old);
      return;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) old[i] = !first && c.counts(i) ? sums[c.at + i] : 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (c.counts(i)) sums[c.at + i] = old[i] + v[i];
  };
  for (int64_t row = blockIdx.x; row < a.n; row += gridDim.x, first = false) {
    const T *z = (const T *)a.z + row * a.ldz, *dh = (const T *)a.dh + row * a.lddh, *r = (const T *)a.r_in + row * a.ldr_in;
    const T *dr = (const T *)a.dr + row * a.lddr, *gate = (const T *)a.gate + row * a.ldgate;
    T *dz = (T *)a.dz + row * a.lddz;
    const float rho_z = a.rstd_z[row], rho_r = RESIDUAL ? a.rstd_r[row] : 0.f;
    const T *g = dh, *unit = RESIDUAL ? r : z;  // the norm whose output's gradient is given
    const void *weight = RESIDUAL ? a.w_pre : a.w_post;
    const float rho = RESIDUAL ? rho_r : rho_z;
    float mean = 0.f;
    if (a.dh) {
      float s = 0.f;
      for (int32_t j = start; j < a.d; j += step) {
        float t[V], h[V], w[V];
        c.place(j, a.d);
        c.floats(c.load(g), t);
        c.floats(c.load(unit), h);
        c.weights(weight, a.w_f32, w);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          h[i] *= rho;
          w[i] *= t[i];
          t[i] *= h[i];
        }
        add_to(RESIDUAL ? p : q, t);
        s += c.dot(w, h);
      }
      mean = row_sum<kWave, true>(s, slots, turn) / (float)a.d;
    }
    auto into = [&](float (&v)[V]) {  // gradient of that norm's input, of the residual sum with dr
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = 0.f;
      if (a.dh) {
        float h[V], w[V];
        c.floats(c.load(g), v);
        c.floats(c.load(unit), h);
        c.weights(weight, a.w_f32, w);
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = rho * (v[i] * w[i] - h[i] * rho * mean);
      }
      if (RESIDUAL && a.dr) {
        float t[V];
        c.floats(c.load(dr), t);
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] += t[i];
      }
    };
    if (!RESIDUAL) {
      for (int32_t j = start; j < a.d; j += step) {
        float v[V];
        c.place(j, a.d);
        into(v);
        c.write(dz, v);
      }
      continue;
    }
    float row_slope = 0.f;
    const float row_sig = a.gate_kind == CG_GATE_ROW ? sigmoid((float)gate[0], row_slope) : 1.f;
    auto through = [&](float (&D)[V], float (&zh)[V], float (&f)[V], bool outputs) {  // f: gradient of the normalised z
      float w[V], t[V], sig[V];
      into(D);
      if (outputs) c.write((T *)a.dx + row * a.lddx, D);
      if (a.mask.rng) c.drop(key, a.mask, row, D);
      c.floats(c.load(z), zh);
      c.weights(a.w_post, a.w_f32, w);
      c.weights(a.scale, a.w_f32, t);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        zh[i] *= rho_z;
        f[i] = D[i] * (w[i] * (a.alpha * t[i]));
        sig[i] = row_sig;
      }
      if (a.gate_kind == CG_GATE_FULL) {
        c.floats(c.load(gate), t);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          float slope;
          sig[i] = sigmoid(t[i], slope);
          t[i] = f[i] * zh[i] * slope;
        }
        if (outputs) c.write((T *)a.dgate + row * a.lddgate, t);
      }
#pragma unroll
      for (int i = 0; i < V; ++i) {
        D[i] *= sig[i] * zh[i];
        f[i] *= a.gate_kind == CG_GATE_FULL ? sig[i] : 1.f;
      }
    };
    float s = 0.f;
    for (int32_t j = start; j < a.d; j += step) {
      float D[V], zh[V], f[V];
      c.place(j, a.d);
      through(D, zh, f, true);
      add_to(q, D);
      if (!a.dh && first) {
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (c.counts(i)) p[c.at + i] = 0.f;
      }
      s += c.dot(f, zh);
    }
    s = row_sum<kWave, true>(s, slots, turn);
    if (a.gate_kind == CG_GATE_ROW && threadIdx.x == 0) ((T *)a.dgate)[row * a.lddgate] = rounded<T>(s * row_slope);
    const float mean_z = s / (float)a.d;
    for (int32_t j = start; j < a.d; j += step) {
      float D[V], zh[V], f[V];
      c.place(j, a.d);
      through(D, zh, f, false);
#pragma unroll
      for (int i = 0; i < V; ++i) f[i] = rho_z * row_sig * (f[i] - zh[i] * mean_z);
      c.write(dz, f);
    }
  }
}

// dw_post = alpha scale q, dscale = alpha w_post q, dw_pre: the slices of `partial` added up.  One workgroup per 16
// columns; 64 threads share a column, each adds every 64th slice in order, then the 64 sums are added in order.  A launch
// holds fewer than 2^32 threads, so that the workgroups of very long rows take more than one stretch of columns each.
constexpr int kFoldCols = 16, kFoldTeams = 64;
constexpr int64_t kFoldGroups = 1 << 20;

template <int DT, bool RESIDUAL>
__global__ __launch_bounds__(kFoldCols *kFoldTeams) void norm_weight_grads_kernel(NormArgs a, int32_t slices, void *dw_post,
                                                                                  void *dw_pre, void *dscale) {
  typedef typename Elem<DT>::type T;
  __shared__ float sq[kFoldTeams][kFoldCols + 1], sp[kFoldTeams][kFoldCols + 1];
  const int col = threadIdx.x % kFoldCols, team = threadIdx.x / kFoldCols;
  const int64_t step = (int64_t)(RESIDUAL ? 2 : 1) * a.d;
  for (int32_t j0 = blockIdx.x * kFoldCols; j0 < a.d; j0 += gridDim.x * kFoldCols) {  // once for rows of up to 2^24 columns
    const int32_t j = j0 + col;
    float q = 0.f, p = 0.f;
    if (j < a.d) {
#pragma unroll 8
      for (int32_t k = team; k < slices; k += kFoldTeams) {
        const float *at = a.partial + k * step + j;
        q += at[0];
        if (RESIDUAL) p += at[a.d];
      }
    }
    sq[team][col] = q;
    if (RESIDUAL) sp[team][col] = p;
    __syncthreads();
    if (team == 0 && j < a.d) {
      q = p = 0.f;
#pragma unroll 8
      for (int t = 0; t < kFoldTeams; ++t) {
        q += sq[t][col];
        if (RESIDUAL) p += sp[t][col];
      }
      if (dw_post) weight_put<T>(dw_post, a.w_f32, j, a.alpha * weight_at<T>(a.scale, a.w_f32, j) * q);
      if (dscale) weight_put<T>(dscale, a.w_f32, j, a.alpha * weight_at<T>(a.w_post, a.w_f32, j) * q);
      if (dw_pre) weight_put<T>(dw_pre, a.w_f32, j, p);
    }
    __syncthreads();  // the sums have been read
  }
}

// ---- host side ------------------------------------------------------------------------------------
// Workgroups of a gradient = slices of partial sums: enough for 16 wavefronts per compute unit; where a workgroup
// holds one row at a time (its slices are as long as its rows) for 12 of the residual block's and 8 of rms_norm's.
static int64_t norm_groups(int64_t n, int32_t d, int dtype, bool residual) {
  const NormShape sh = norm_shape(d, dtype, residual);
  const int waves = sh.threads / kWave, per_cu = (!sh.whole ? 16 : residual ? 12 : 8) / waves;
  const int64_t most = 256 * (per_cu > 0 ? per_cu : 1);
  const int64_t want = ceil_div64(n, norm_rows_at_once(sh));
  return want < most ? want : most;
}
// an upper bound for every type and both operators
static size_t norm_workspace(int64_t n, int32_t d) {
  int64_t slices = 0;  // of d floats
  for (int dtype : {CG_F32, CG_BF16})
    for (int residual : {0, 1}) {
      const int64_t g = norm_groups(n, d, dtype, residual) * (residual ? 2 : 1);
      slices = g > slices ? g : slices;
    }
  return (size_t)slices * (size_t)d * sizeof(float);
}

// columns are stepped through in int32, a workgroup's width at a time
static int check_norm_shape(const char *who, int64_t n, int32_t d) {
  CG_TRY(check_row_shape(who, n, d));
  if (d > (1 << 30)) CG_FAIL(CG_ERR_OVERFLOW, "%s: rows of d=%d elements (at most 2^30)", who, d);
  return CG_OK;
}

static int check_weights(const char *who, int dtype, int wdtype) {
  if (wdtype != CG_F32 && wdtype != dtype)
    CG_FAIL(CG_ERR_UNSUPPORTED, "%s: weights of dtype %d beside activations of dtype %d (CG_F32 or the same)", who, wdtype, dtype);
  return CG_OK;
}
static int check_float(const char *who, const char *what, float v, bool positive) {
  if (!(v - v == 0.f) || (positive && !(v > 0.f)))
    CG_FAIL(CG_ERR_SIZE, "%s: %s=%g has to be finite%s", who, what, (double)v, positive ? " and above zero" : "");
  return CG_OK;
}

template <bool RESIDUAL>
static int norm_fwd(const NormArgs &a, int dtype, hipStream_t s) {
  if (norm_shape(a.d, dtype, false).lanes > 0) return launch_norm_fwd(a, RESIDUAL, dtype, s);
  const int64_t groups = a.n < 256 * 32 ? a.n : 256 * 32;
#define CG_CALL(DT) norm_fwd_rows_kernel<DT, RESIDUAL><<<(unsigned)groups, kLongThreads, 0, s>>>(a)
  CG_BY_DTYPE(dtype, CG_CALL)
#undef CG_CALL
  CG_LAUNCH_CHECK();
  return CG_OK;
}

template <bool RESIDUAL>
static int norm_bwd(const NormArgs &a, int dtype, void *dw_post, void *dw_pre, void *dscale, hipStream_t s) {
  const int64_t groups = norm_groups(a.n, a.d, dtype, RESIDUAL);
  if (groups > 0 && norm_shape(a.d, dtype, RESIDUAL).lanes > 0) {
    CG_TRY(launch_norm_bwd(a, RESIDUAL, dtype, groups, s));
  } else if (groups > 0) {
#define CG_CALL(DT) norm_bwd_rows_kernel<DT, RESIDUAL><<<(unsigned)groups, kLongThreads, 0, s>>>(a)
    CG_BY_DTYPE(dtype, CG_CALL)
#undef CG_CALL
    CG_LAUNCH_CHECK();
  }
  if (dw_post || dw_pre || dscale) {
    const int64_t stretches = ceil_div64(a.d, kFoldCols);
    const unsigned cols = (unsigned)(stretches < kFoldGroups ? stretches : kFoldGroups);
#define CG_CALL(DT)                                                                                            \
  norm_weight_grads_kernel<DT, RESIDUAL><<<cols, kFoldCols * kFoldTeams, 0, s>>>(a, (int32_t)groups, dw_post, \
                                                                                 dw_pre, dscale)
    CG_BY_DTYPE(dtype, CG_CALL)
#undef CG_CALL
    CG_LAUNCH_CHECK();
  }
  return CG_OK;
}

}  // namespace cg

extern "C" {

int cg_norm_bwd_workspace(int64_t n, int32_t d, int64_t *bytes) {
  using namespace cg;
  if (!bytes) CG_FAIL(CG_ERR_NULL, "cg_norm_bwd_workspace: null pointer");
  CG_TRY(check_norm_shape("cg_norm_bwd_workspace", n, d));
  *bytes = (int64_t)norm_workspace(n, d);
  return CG_OK;
}

int cg_rms_norm_fwd(const void *d_x, int64_t ldx, const void *d_w, int wdtype, void *d_y, int64_t ldy, float *d_rstd,
                    int64_t n, int32_t d, int dtype, float eps, cg_stream_t stream) {
  using namespace cg;
  const char *who = "cg_rms_norm_fwd";
  CG_TRY(check_dtype(who, dtype));
  CG_TRY(check_weights(who, dtype, wdtype));
  CG_TRY(check_norm_shape(who, n, d));
  CG_TRY(check_float(who, "eps", eps, true));
  if (n == 0) return CG_OK;
  if (!d_x || !d_y || !d_rstd) CG_FAIL(CG_ERR_NULL, "%s: null pointer", who);
  if (ldx < d || ldy < d) CG_FAIL(CG_ERR_SIZE, "%s: leading dimension smaller than d", who);
  if (d_x == d_y) CG_FAIL(CG_ERR_ALIAS, "%s: the output may not be the input", who);
  NormArgs a = {};
  a.z = d_x, a.ldz = ldx, a.w_post = d_w, a.w_f32 = wdtype == CG_F32, a.h = d_y, a.ldh = ldy, a.rstd_z = d_rstd;
  a.n = n, a.d = d, a.eps = eps, a.alpha = 1.f;
  ProfScope prof("rms_norm_fwd", d, (hipStream_t)stream);
  return norm_fwd<false>(a, dtype, (hipStream_t)stream);
}

int cg_rms_norm_bwd(const void *d_g, int64_t ldg, const void *d_x, int64_t ldx, const void *d_w, int wdtype,
                    const float *d_rstd, void *d_dx, int64_t lddx, void *d_dw, int64_t n, int32_t d, int dtype,
                    void *d_work, int64_t work_bytes, cg_stream_t stream) {
  using namespace cg;
  const char *who = "cg_rms_norm_bwd";
  CG_TRY(check_dtype(who, dtype));
  CG_TRY(check_weights(who, dtype, wdtype));
  CG_TRY(check_norm_shape(who, n, d));
  if (n > 0) {
    if (!d_g || !d_x || !d_rstd || !d_dx || !d_work) CG_FAIL(CG_ERR_NULL, "%s: null pointer", who);
    if (ldg < d || ldx < d || lddx < d) CG_FAIL(CG_ERR_SIZE, "%s: leading dimension smaller than d", who);
    if (d_dx == d_g || d_dx == d_x) CG_FAIL(CG_ERR_ALIAS, "%s: the output may not be an input", who);
    CG_TRY(check_work(who, d_work, work_bytes, (int64_t)norm_workspace(n, d)));
  }
  NormArgs a = {};
  a.dh = d_g, a.lddh = ldg, a.z = d_x, a.ldz = ldx, a.w_post = d_w, a.w_f32 = wdtype == CG_F32;
  a.rstd_z = const_cast<float *>(d_rstd), a.dz = d_dx, a.lddz = lddx, a.partial = (float *)d_work;
  a.n = n, a.d = d, a.alpha = 1.f;
  ProfScope prof("rms_norm_bwd", d, (hipStream_t)stream);
  return norm_bwd<false>(a, dtype, d_dw, nullptr, nullptr, (hipStream_t)stream);
}

int cg_norm_residual_fwd(const void *d_z, int64_t ldz, const void *d_x, int64_t ldx, const void *d_gate, int64_t ldgate,
                         int gate_kind, const void *d_w_post, const void *d_w_pre, const void *d_scale, int wdtype,
                         float alpha, double p, const int64_t *d_rng, float eps, void *d_r, int64_t ldr, void *d_h,
                         int64_t ldh, float *d_rstd_z, float *d_rstd_r, int64_t n, int32_t d, int dtype,
                         cg_stream_t stream) {
  using namespace cg;
  const char *who = "cg_norm_residual_fwd";
  CG_TRY(check_dtype(who, dtype));
  CG_TRY(check_weights(who, dtype, wdtype));
  CG_TRY(check_norm_shape(who, n, d));
  CG_TRY(check_float(who, "eps", eps, true));
  CG_TRY(check_float(who, "alpha", alpha, false));
  CG_TRY(check_p(who, p, d_rng));
  if (gate_kind < CG_GATE_NONE || gate_kind > CG_GATE_FULL) CG_FAIL(CG_ERR_UNSUPPORTED, "%s: gate kind %d", who, gate_kind);
  if (n == 0) return CG_OK;
  if (!d_z || !d_x || !d_r || !d_h || !d_rstd_z || !d_rstd_r || (gate_kind != CG_GATE_NONE && !d_gate))
    CG_FAIL(CG_ERR_NULL, "%s: null pointer", who);
  if (ldz < d || ldx < d || ldr < d || ldh < d || (gate_kind == CG_GATE_FULL && ldgate < d) || (gate_kind == CG_GATE_ROW && ldgate < 1))
    CG_FAIL(CG_ERR_SIZE, "%s: leading dimension smaller than d", who);
  if (d_r == d_z || d_r == d_x || d_h == d_z || d_h == d_x || d_r == d_h || (gate_kind != CG_GATE_NONE && (d_r == d_gate || d_h == d_gate)))
    CG_FAIL(CG_ERR_ALIAS, "%s: an output may not be an input or the other output", who);
  NormArgs a = {};
  a.z = d_z, a.ldz = ldz, a.x = d_x, a.ldx = ldx, a.gate = d_gate, a.ldgate = ldgate, a.gate_kind = gate_kind;
  a.w_post = d_w_post, a.w_pre = d_w_pre, a.scale = d_scale, a.w_f32 = wdtype == CG_F32, a.alpha = alpha, a.eps = eps;
  a.r = d_r, a.ldr = ldr, a.h = d_h, a.ldh = ldh, a.rstd_z = d_rstd_z, a.rstd_r = d_rstd_r, a.mask = make_mask(p, d_rng);
  a.n = n, a.d = d;
  ProfScope prof("norm_residual_fwd", d, (hipStream_t)stream);
  return norm_fwd<true>(a, dtype, (hipStream_t)stream);
}

int cg_norm_residual_bwd(const void *d_dr, int64_t lddr, const void *d_dh, int64_t lddh, const void *d_z, int64_t ldz,
                         const void *d_r, int64_t ldr, const void *d_gate, int64_t ldgate, int gate_kind,
                         const void *d_w_post, const void *d_w_pre, const void *d_scale, int wdtype, float alpha,
                         double p, const int64_t *d_rng, const float *d_rstd_z, const float *d_rstd_r, void *d_dz,
                         int64_t lddz, void *d_dx, int64_t lddx, void *d_dgate, int64_t lddgate, void *d_dw_post,
                         void *d_dw_pre, void *d_dscale, int64_t n, int32_t d, int dtype, void *d_work,
                         int64_t work_bytes, cg_stream_t stream) {
  using namespace cg;
  const char *who = "cg_norm_residual_bwd";
  CG_TRY(check_dtype(who, dtype));
  CG_TRY(check_weights(who, dtype, wdtype));
  CG_TRY(check_norm_shape(who, n, d));
  CG_TRY(check_float(who, "alpha", alpha, false));
  CG_TRY(check_p(who, p, d_rng));
  if (gate_kind < CG_GATE_NONE || gate_kind > CG_GATE_FULL) CG_FAIL(CG_ERR_UNSUPPORTED, "%s: gate kind %d", who, gate_kind);
  if (n > 0) {
    if ((!d_dr && !d_dh) || !d_z || !d_r || !d_rstd_z || !d_rstd_r || !d_dz || !d_dx || !d_work ||
        (gate_kind != CG_GATE_NONE && (!d_gate || !d_dgate)))
      CG_FAIL(CG_ERR_NULL, "%s: null pointer", who);
    if ((d_dr && lddr < d) || (d_dh && lddh < d) || ldz < d || ldr < d || lddz < d || lddx < d ||
        (gate_kind == CG_GATE_FULL && (ldgate < d || lddgate < d)) || (gate_kind == CG_GATE_ROW && (ldgate < 1 || lddgate < 1)))
      CG_FAIL(CG_ERR_SIZE, "%s: leading dimension smaller than d", who);
    const void *ins[5] = {d_dr, d_dh, d_z, d_r, gate_kind != CG_GATE_NONE ? d_gate : nullptr};
    const void *outs[3] = {d_dz, d_dx, gate_kind != CG_GATE_NONE ? d_dgate : nullptr};
    for (int o = 0; o < 3; ++o) {
      for (const void *i : ins)
        if (outs[o] && outs[o] == i) CG_FAIL(CG_ERR_ALIAS, "%s: an output may not be an input", who);
      if (outs[o] && outs[o] == outs[(o + 1) % 3]) CG_FAIL(CG_ERR_ALIAS, "%s: two outputs are the same", who);
    }
    CG_TRY(check_work(who, d_work, work_bytes, (int64_t)norm_workspace(n, d)));
  }
  NormArgs a = {};
  a.dr = d_dr, a.lddr = lddr, a.dh = d_dh, a.lddh = lddh, a.z = d_z, a.ldz = ldz, a.r_in = d_r, a.ldr_in = ldr;
  a.gate = d_gate, a.ldgate = ldgate, a.gate_kind = gate_kind, a.w_post = d_w_post, a.w_pre = d_w_pre, a.scale = d_scale;
  a.w_f32 = wdtype == CG_F32, a.alpha = alpha, a.mask = make_mask(p, d_rng);
  a.rstd_z = const_cast<float *>(d_rstd_z), a.rstd_r = const_cast<float *>(d_rstd_r);
  a.dz = d_dz, a.lddz = lddz, a.dx = d_dx, a.lddx = lddx, a.dgate = d_dgate, a.lddgate = lddgate;
  a.partial = (float *)d_work, a.n = n, a.d = d;
  ProfScope prof("norm_residual_bwd", d, (hipStream_t)stream);
  return norm_bwd<true>(a, dtype, d_dw_post, d_dw_pre, d_dscale, (hipStream_t)stream);
}

}  // extern "C"
