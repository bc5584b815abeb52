// Dropout with masks that are recomputed instead of stored: forward and gradient are the same kernel,
//   out = keep ? x / (1 - p) : 0,  keep decided by the counter-based generator of rows.h.
#include "rows.h"

namespace cg {

constexpr int kDropThreads = 256;

__global__ void rng_next_kernel(int64_t *__restrict__ state, int64_t *__restrict__ out) {
  const int64_t seed = state[0], off = state[1];
  out[0] = seed;
  out[1] = off;
  state[1] = (int64_t)((uint64_t)off + 1ull);
}

// One thread per four consecutive columns: one generator call decides them.
template <int DT>
__global__ __launch_bounds__(kDropThreads) void dropout_kernel(const typename Elem<DT>::type *x, int64_t ldx,
                                                               typename Elem<DT>::type *out, int64_t ldo, int64_t n,
                                                               int32_t d, Mask m) {
  const int32_t blocks = (d + 3) / 4;
  const int64_t total = n * blocks, step = (int64_t)gridDim.x * kDropThreads;
  MaskKey key = {0, 0, 0, 0};
  if (m.rng) key = mask_key(m.rng);
  for (int64_t i = (int64_t)blockIdx.x * kDropThreads + threadIdx.x; i < total; i += step) {
    const int64_t row = i / blocks;
    const int32_t block = (int32_t)(i - row * blocks), j = block * 4;
    const int live = d - j < 4 ? d - j : 4;
    float v[4];
    load_some(x + row * ldx + j, live, v);
    if (m.rng) {
      uint32_t w[4];
      mask_words(key, (uint32_t)row, (uint32_t)block, w);
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = w[k] > m.last ? v[k] * m.inv_keep : 0.f;
    }
    store_some(out + row * ldo + j, live, v);
  }
}

}  // namespace cg

extern "C" {

int cg_rng_next(int64_t *d_state, int64_t *d_out, cg_stream_t stream) {
  using namespace cg;
  if (!d_state || !d_out) CG_FAIL(CG_ERR_NULL, "cg_rng_next: null pointer");
  if (d_state == d_out) CG_FAIL(CG_ERR_ALIAS, "cg_rng_next: the snapshot may not be the state itself");
  rng_next_kernel<<<1, 1, 0, (hipStream_t)stream>>>(d_state, d_out);
  CG_LAUNCH_CHECK();
  return CG_OK;
}

int cg_dropout(const void *d_x, int64_t ldx, void *d_out, int64_t ldo, int64_t n, int32_t d, int dtype, double p,
               const int64_t *d_rng, cg_stream_t stream) {
  using namespace cg;
  CG_TRY(check_dtype("cg_dropout", dtype));
  CG_TRY(check_row_shape("cg_dropout", n, d));
  CG_TRY(check_p("cg_dropout", p, d_rng));
  if (n == 0) return CG_OK;
  if (!d_x || !d_out) CG_FAIL(CG_ERR_NULL, "cg_dropout: null pointer");
  if (ldx < d || ldo < d) CG_FAIL(CG_ERR_SIZE, "cg_dropout: leading dimension smaller than d");
  if (d_x == d_out && ldx != ldo) CG_FAIL(CG_ERR_ALIAS, "cg_dropout: in place needs equal leading dimensions");
  const Mask m = make_mask(p, d_rng);
  hipStream_t s = (hipStream_t)stream;
  ProfScope prof("dropout", d, s);
  int64_t groups = ceil_div64(n * ((d + 3) / 4), kDropThreads);
  if (groups > 256 * 64) groups = 256 * 64;
#define CG_CALL(DT)                                                                                                    \
  dropout_kernel<DT><<<(unsigned)groups, kDropThreads, 0, s>>>((const Elem<DT>::type *)d_x, ldx, (Elem<DT>::type *)d_out, \
                                                               ldo, n, d, m)
  CG_BY_DTYPE(dtype, CG_CALL)
#undef CG_CALL
  CG_LAUNCH_CHECK();
  return CG_OK;
}

}  // extern "C"
