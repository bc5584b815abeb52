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

// 16 bytes a thread and step: one generator call for four float32 columns, two for eight 16-bit ones.  Threads walk the
// chunks of the whole array in order, `rows_on` rows and `chunks_on` chunks further at every step.  kSteps chunks are
// loaded before the first is decided: their generator calls run while the loads are on their way.
constexpr int kSteps = 2;

template <int DT, bool RAGGED>
__global__ __launch_bounds__(kDropThreads) void dropout_kernel(const typename Elem<DT>::type *x, int64_t ldx,
                                                               typename Elem<DT>::type *out, int64_t ldo, int64_t n,
                                                               int32_t d, int32_t chunks, int64_t rows_on,
                                                               int32_t chunks_on, Mask m) {
  typedef typename Elem<DT>::type T;
  typedef Chunk<T, RAGGED> C;
  MaskKey key = {0, 0, 0, 0};
  if (m.rng) key = mask_key(m.rng);
  const int64_t first = (int64_t)blockIdx.x * kDropThreads + threadIdx.x;
  int64_t row = first / chunks;
  int32_t at = (int32_t)(first - row * chunks);
  while (row < n) {
    C c[kSteps];
    Raw r[kSteps];
    int64_t rows[kSteps];
    int32_t cols[kSteps];
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
      rows[k] = row;
      cols[k] = at;
      c[k].place(at * C::V, d);
      r[k] = c[k].load(x + (row < n ? row : n - 1) * ldx);
      row += rows_on;
      at += chunks_on;
      if (at >= chunks) at -= chunks, ++row;
    }
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
      float v[C::V];
      c[k].floats(r[k], v);
      if (m.rng) drop_chunk<C::V>(key, m, rows[k], cols[k] * C::V, v);
      if (rows[k] < n) c[k].write(out + rows[k] * ldo, v);
    }
  }
}

template <int DT>
static void launch_dropout(const void *x, int64_t ldx, void *out, int64_t ldo, int64_t n, int32_t d, const Mask &m,
                           hipStream_t s) {
  typedef typename Elem<DT>::type T;
  const int v = Chunk<T, false>::V;
  const int32_t chunks = (int32_t)ceil_div64(d, v);
  int64_t groups = ceil_div64(n * chunks, kDropThreads * kSteps);
  if (groups > 256 * 128) groups = 256 * 128;
  const int64_t step = groups * kDropThreads;
  if (d % v == 0)
    dropout_kernel<DT, false><<<(unsigned)groups, kDropThreads, 0, s>>>((const T *)x, ldx, (T *)out, ldo, n, d, chunks,
                                                                        step / chunks, (int32_t)(step % chunks), m);
  else
    dropout_kernel<DT, true><<<(unsigned)groups, kDropThreads, 0, s>>>((const T *)x, ldx, (T *)out, ldo, n, d, chunks,
                                                                       step / chunks, (int32_t)(step % chunks), m);
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
#define CG_CALL(DT) launch_dropout<DT>(d_x, ldx, d_out, ldo, n, d, m, s)
  CG_BY_DTYPE(dtype, CG_CALL)
#undef CG_CALL
  CG_LAUNCH_CHECK();
  return CG_OK;
}

}  // extern "C"
