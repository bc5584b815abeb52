// Embedding lookup and its gradient.
//   forward   out_i = scale * table[idx_i]          (an index outside [0, rows) reads a row of zeros)
//   gradient  dtable_v = scale * sum_{i: idx_i = v} g_i + beta * dtable_v
// The gradient sorts (index, position) stably, so that the positions of one table row lie side by side in their
// original order, and adds them up in that order: no floating-point atomics, the same bits on every call.  Every
// buffer it needs comes from the caller's workspace.
#include "rows.h"

namespace cg {

constexpr int kEmbThreads = 256;
constexpr int kEmbWaves = kEmbThreads / kWave;

struct IndexView {
  const void *idx;
  int wide;  // int64 indices
};
__device__ __forceinline__ int64_t index_at(const IndexView &v, int64_t i) {
  return v.wide ? static_cast<const int64_t *>(v.idx)[i] : (int64_t) static_cast<const int32_t *>(v.idx)[i];
}

// Lanes that share a row: a power of two that covers its 16-byte chunks, at most a workgroup (longer rows are taken in
// strides of it); lanes beyond the row's end have nothing to do.
static inline int lanes_log2(int32_t d, int per_chunk) {
  const int64_t c = ceil_div64(d, per_chunk);
  int log2 = 0;
  while (((int64_t)1 << log2) < c && log2 < 8) ++log2;
  return log2;
}

// ---------------------------------------------------------------------------------------------
// lookup: kLookups rows a team at once, all indices loaded before the first row and all rows before the first store
// ---------------------------------------------------------------------------------------------
constexpr int kLookups = 4;

template <int DT>
__global__ __launch_bounds__(kEmbThreads) void embedding_fwd_kernel(const typename Elem<DT>::type *__restrict__ table,
                                                                    int64_t ldt, int64_t rows, IndexView idx, int64_t n,
                                                                    int32_t d, float scale, int lanes_log,
                                                                    typename Elem<DT>::type *__restrict__ out,
                                                                    int64_t ldo) {
  typedef typename Elem<DT>::type T;
  typedef Chunk<T, true> C;
  const int lanes = 1 << lanes_log, lane = threadIdx.x & (lanes - 1), teams = kEmbThreads >> lanes_log;
  const int64_t step = (int64_t)gridDim.x * teams * kLookups;
  for (int64_t i0 = ((int64_t)blockIdx.x * teams + (threadIdx.x >> lanes_log)) * kLookups; i0 < n; i0 += step) {
    int64_t v[kLookups];
#pragma unroll
    for (int k = 0; k < kLookups; ++k) v[k] = index_at(idx, i0 + k < n ? i0 + k : n - 1);
    for (int32_t j = lane * C::V; j < d; j += lanes * C::V) {
      C c;
      c.place(j, d);
      Raw r[kLookups];
#pragma unroll
      for (int k = 0; k < kLookups; ++k) r[k] = c.load(table + (v[k] >= 0 && v[k] < rows ? v[k] : 0) * ldt);
#pragma unroll
      for (int k = 0; k < kLookups; ++k) {
        float f[C::V];
        c.floats(r[k], f);
        const bool in = v[k] >= 0 && v[k] < rows;
#pragma unroll
        for (int i = 0; i < C::V; ++i) f[i] = in ? f[i] * scale : 0.f;
        if (i0 + k < n) c.write(out + (i0 + k) * ldo, f);
      }
    }
  }
}

// ---------------------------------------------------------------------------------------------
// stable radix sort of (key, position), digits of up to 9 bits: 16 to 18 bit tables take two passes
// ---------------------------------------------------------------------------------------------
constexpr int kMaxDigit = 9;
constexpr int kMaxRadix = 1 << kMaxDigit;
constexpr int kKeysPerLane = 4;
constexpr int kEmbTile = kEmbThreads * kKeysPerLane;  // 1024 keys a workgroup
constexpr int kWaveKeys = kWave * kKeysPerLane;

// Where a pass reads its keys from: the caller's indices (an index outside the table becomes `rows`, which sorts
// behind every table row) or the arrays of the pass before.
struct KeySource {
  IndexView idx;
  const int32_t *key, *pos;
  int64_t rows;
};
__device__ __forceinline__ int32_t key_at(const KeySource &s, int64_t i) {
  if (s.key) return s.key[i];
  const int64_t v = index_at(s.idx, i);
  return (int32_t)(v >= 0 && v < s.rows ? v : s.rows);
}

// hist[digit * tiles + tile]
__global__ __launch_bounds__(kEmbThreads) void emb_hist_kernel(KeySource src, int64_t n, int shift, int dbits,
                                                               uint32_t *__restrict__ hist, int64_t tiles) {
  __shared__ uint32_t count[kMaxRadix];
  const int radix = 1 << dbits;
  for (int i = threadIdx.x; i < radix; i += kEmbThreads) count[i] = 0;
  __syncthreads();
  const int64_t base = (int64_t)blockIdx.x * kEmbTile;
  int32_t k[kKeysPerLane];
#pragma unroll
  for (int r = 0; r < kKeysPerLane; ++r) {
    const int64_t i = base + r * kEmbThreads + threadIdx.x;
    k[r] = key_at(src, i < n ? i : n - 1);
  }
#pragma unroll
  for (int r = 0; r < kKeysPerLane; ++r)
    if (base + r * kEmbThreads + threadIdx.x < n) atomicAdd(&count[((uint32_t)k[r] >> shift) & (radix - 1)], 1u);
  __syncthreads();
  for (int i = threadIdx.x; i < radix; i += kEmbThreads) hist[(int64_t)i * tiles + blockIdx.x] = count[i];
}

// one wave per digit: exclusive prefix of its counts over the tiles, in place, and their total
__global__ __launch_bounds__(kEmbThreads) void emb_scan_kernel(uint32_t *__restrict__ hist, int64_t tiles, int radix,
                                                               uint32_t *__restrict__ totals) {
  const int digit = blockIdx.x * kEmbWaves + threadIdx.x / kWave, lane = threadIdx.x & (kWave - 1);
  if (digit >= radix) return;
  uint32_t *h = hist + (int64_t)digit * tiles;
  uint32_t run = 0;
  for (int64_t t0 = 0; t0 < tiles; t0 += kWave) {
    const int64_t t = t0 + lane;
    const uint32_t v = t < tiles ? h[t] : 0u;
    uint32_t inc = v;
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1) {
      const uint32_t up = __shfl_up(inc, off, kWave);
      if (lane >= off) inc += up;
    }
    if (t < tiles) h[t] = run + inc - v;
    run += __shfl(inc, kWave - 1, kWave);
  }
  if (lane == 0) totals[digit] = run;
}

// Exclusive prefix over the workgroup's threads of one value each.
__device__ __forceinline__ uint32_t group_exclusive(uint32_t v, uint32_t *wave_sums) {
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  uint32_t inc = v;
#pragma unroll
  for (int off = 1; off < kWave; off <<= 1) {
    const uint32_t up = __shfl_up(inc, off, kWave);
    if (lane >= off) inc += up;
  }
  __syncthreads();
  if (lane == kWave - 1) wave_sums[wave] = inc;
  __syncthreads();
  uint32_t before = 0;
  for (int w = 0; w < wave; ++w) before += wave_sums[w];
  return before + inc - v;
}

// Wave w of a workgroup owns keys [tile + 256 w, tile + 256 (w + 1)), 64 at a time in order.  Lanes with equal digits
// find each other by ballots; a key's rank is the wave's running count of its digit plus the equal lanes below it.
__global__ __launch_bounds__(kEmbThreads) void emb_scatter_kernel(KeySource src, int64_t n, int shift, int dbits,
                                                                  const uint32_t *__restrict__ hist, int64_t tiles,
                                                                  const uint32_t *__restrict__ totals,
                                                                  int32_t *__restrict__ out_key,
                                                                  int32_t *__restrict__ out_pos) {
  __shared__ uint32_t count[kEmbWaves][kMaxRadix];
  __shared__ uint32_t first[kMaxRadix];  // global position of a record = first[digit] + its position in the tile
  __shared__ uint32_t wave_sums[kEmbWaves];
  __shared__ int32_t skey[kEmbTile], spos[kEmbTile];
  const int radix = 1 << dbits, lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  for (int i = threadIdx.x; i < kEmbWaves * kMaxRadix; i += kEmbThreads) (&count[0][0])[i] = 0;
  const int64_t tile_base = (int64_t)blockIdx.x * kEmbTile, base = tile_base + wave * kWaveKeys;
  int32_t key[kKeysPerLane], pos[kKeysPerLane];
#pragma unroll
  for (int r = 0; r < kKeysPerLane; ++r) {
    const int64_t i = base + r * kWave + lane, at = i < n ? i : n - 1;
    key[r] = key_at(src, at);
    pos[r] = src.pos ? src.pos[at] : (int32_t)at;
  }
  __syncthreads();
  uint32_t rank[kKeysPerLane];
  const uint64_t below = (1ull << lane) - 1ull;
#pragma unroll
  for (int r = 0; r < kKeysPerLane; ++r) {
    const bool valid = base + r * kWave + lane < n;
    const uint32_t digit = ((uint32_t)key[r] >> shift) & (uint32_t)(radix - 1);
    uint64_t peers = __ballot(valid);
#pragma unroll
    for (int b = 0; b < kMaxDigit; ++b)
      if (b < dbits) {
        const bool one = (digit >> b) & 1u;
        const uint64_t with = __ballot(one);
        peers &= one ? with : ~with;
      }
    const uint32_t before = (uint32_t)__popcll(peers & below);
    uint32_t had = 0;
    if (valid) had = count[wave][digit];
    // the lowest lane of the set writes the new count; it depends on `had`, so the read above comes first
    if (valid && before == 0) count[wave][digit] = had + (uint32_t)__popcll(peers);
    rank[r] = had + before;
  }
  __syncthreads();
  // digit offsets: two digits a thread; in the tile (for the order in LDS) and in the whole array
  const int d0 = threadIdx.x * 2;
  uint32_t here[2] = {0, 0}, all[2] = {0, 0};
#pragma unroll
  for (int k = 0; k < 2; ++k)
    if (d0 + k < radix) {
      for (int w = 0; w < kEmbWaves; ++w) here[k] += count[w][d0 + k];
      all[k] = totals[d0 + k];
    }
  uint32_t in_tile = group_exclusive(here[0] + here[1], wave_sums);
  uint32_t in_all = group_exclusive(all[0] + all[1], wave_sums);
#pragma unroll
  for (int k = 0; k < 2; ++k)
    if (d0 + k < radix) {
      first[d0 + k] = in_all + hist[(int64_t)(d0 + k) * tiles + blockIdx.x] - in_tile;  // modulo 2^32, undone below
      uint32_t run = in_tile;
      for (int w = 0; w < kEmbWaves; ++w) {
        const uint32_t c = count[w][d0 + k];
        count[w][d0 + k] = run;
        run += c;
      }
      in_tile += here[k];
      in_all += all[k];
    }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kKeysPerLane; ++r)
    if (base + r * kWave + lane < n) {
      const uint32_t digit = ((uint32_t)key[r] >> shift) & (uint32_t)(radix - 1);
      const uint32_t at = count[wave][digit] + rank[r];
      skey[at] = key[r];
      spos[at] = pos[r];
    }
  __syncthreads();
  const int64_t left = n - tile_base;
  const int here_n = (int)(left < kEmbTile ? left : kEmbTile);
  for (int i = threadIdx.x; i < here_n; i += kEmbThreads) {
    const uint32_t to = first[((uint32_t)skey[i] >> shift) & (uint32_t)(radix - 1)] + (uint32_t)i;
    out_key[to] = skey[i];
    out_pos[to] = spos[i];
  }
}

// ---------------------------------------------------------------------------------------------
// Sums.  rowptr[v] .. rowptr[v + 1] are the sorted positions of table row v.  A row with up to `span` of them is added
// up by one team of lanes.  The sorted array is also cut into chunks of `span` positions: a row with more than `span`
// ("hot": with popular indices one row can hold a tenth of all) covers the end of at least one chunk, so a chunk holds a
// part of at most two hot rows, the one it begins in and the one it ends in.  A team adds up each part into a partial
// row, and a second kernel adds a hot row's partial rows in order.
// ---------------------------------------------------------------------------------------------
struct SumArgs {
  const void *g;
  int64_t ldg;
  const int32_t *rowptr, *key, *pos;
  int64_t rows;
  int32_t n, d, span;
  float scale, beta;
  void *out;
  int64_t ldo;
  float *partial;  // [2 * chunks][d], float32
  unsigned chunk_groups, chunk_teams;
};

constexpr int kAhead = 8;  // rows of g in flight per lane

// The chunk's columns of g's rows pos[from .. to), added in order.  The positions of the next kAhead rows are loaded
// while those before them are on their way, so that a long segment pays one memory latency a step and not two.
template <typename T>
__device__ __forceinline__ void add_rows(const SumArgs &a, const Chunk<T, true> &c, int32_t from, int32_t to,
                                         float (&sum)[Chunk<T, true>::V]) {
  constexpr int V = Chunk<T, true>::V;
#pragma unroll
  for (int i = 0; i < V; ++i) sum[i] = 0.f;
  if (from >= to) return;
  int32_t p[kAhead];
#pragma unroll
  for (int k = 0; k < kAhead; ++k) p[k] = a.pos[from + k < to ? from + k : to - 1];
  for (int32_t at = from; at < to; at += kAhead) {
    Raw r[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      r[k] = Raw{0u, 0u, 0u, 0u};
      if (k == 0 || at + k < to) r[k] = c.load((const T *)a.g + (int64_t)p[k] * a.ldg);
    }
    if (at + kAhead < to) {
#pragma unroll
      for (int k = 0; k < kAhead; ++k) p[k] = a.pos[at + kAhead + k < to ? at + kAhead + k : to - 1];
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      float f[V];
      c.floats(r[k], f);
#pragma unroll
      for (int i = 0; i < V; ++i) sum[i] += f[i];
    }
  }
}

template <int DT, bool OUT_F32>
__global__ __launch_bounds__(kEmbThreads) void emb_sum_kernel(SumArgs a, int lanes_log) {
  typedef typename Elem<DT>::type T;
  typedef typename Elem<OUT_F32 ? CG_F32 : DT>::type O;
  constexpr int V = Chunk<T, true>::V;
  const int lanes = 1 << lanes_log, lane = threadIdx.x & (lanes - 1), teams = kEmbThreads >> lanes_log;
  const int team = threadIdx.x >> lanes_log;
  if (blockIdx.x < a.chunk_groups) {  // parts of hot rows
    const int32_t chunk = (int32_t)blockIdx.x * teams + team;
    if (chunk >= (int32_t)a.chunk_teams) return;
    const int32_t all = a.rowptr[a.rows], begin = chunk * a.span;
    if (begin >= all) return;
    const int32_t end = all - begin < a.span ? all : begin + a.span;
    const int32_t first = a.key[begin], last = a.key[end - 1];
#pragma unroll
    for (int part = 0; part < 2; ++part) {
      const int32_t v = part == 0 ? first : last, from = a.rowptr[v], to = a.rowptr[v + 1];
      if (to - from <= a.span || (part == 1 && first == last)) continue;
      float *dst = a.partial + ((int64_t)chunk * 2 + part) * a.d;
      for (int32_t j = lane * V; j < a.d; j += lanes * V) {
        Chunk<T, true> c;
        c.place(j, a.d);
        float sum[V];
        add_rows<T>(a, c, from > begin ? from : begin, to < end ? to : end, sum);
        store_some<float, V>(dst + j, c.live, sum);
      }
    }
    return;
  }
  const int64_t step = (int64_t)(gridDim.x - a.chunk_groups) * teams;
  for (int64_t v = (int64_t)(blockIdx.x - a.chunk_groups) * teams + team; v < a.rows; v += step) {
    const int32_t from = a.rowptr[v], to = a.rowptr[v + 1];
    if (to - from > a.span || (from == to && a.beta == 1.f)) continue;
    O *out = (O *)a.out + v * a.ldo;
    for (int32_t j = lane * V; j < a.d; j += lanes * V) {
      Chunk<T, true> c;
      c.place(j, a.d);
      float sum[V];
      add_rows<T>(a, c, from, to, sum);
#pragma unroll
      for (int i = 0; i < V; ++i) sum[i] *= a.scale;
      if (a.beta != 0.f) {
        float old[V];
        load_some<O, V>(out + j, c.live, old);
#pragma unroll
        for (int i = 0; i < V; ++i) sum[i] += a.beta * old[i];
      }
      store_some<O, V>(out + j, c.live, sum);
    }
  }
}

// One workgroup per chunk and 256 columns; it has work if a hot row begins in its chunk (at most one does: it covers
// the chunk's end).  Its 16 waves take every 16th partial row each, their sums are added in order.
constexpr int kFoldWaves = 16, kFoldColumns = kWave * 4;

template <int OT>
__global__ __launch_bounds__(kWave *kFoldWaves) void emb_fold_kernel(SumArgs a) {
  typedef typename Elem<OT>::type O;
  __shared__ float lds[kFoldWaves][kFoldColumns];
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const int32_t j = blockIdx.y * kFoldColumns + lane * 4, all = a.rowptr[a.rows];
  Chunk<float, true> c;
  c.place(j, a.d);
  for (int32_t chunk = blockIdx.x; chunk < (int32_t)a.chunk_teams; chunk += gridDim.x) {  // uniform in the workgroup
    const int32_t begin = chunk * a.span;
    if (begin >= all) return;
    const int32_t end = all - begin < a.span ? all : begin + a.span;
    const int32_t v = a.key[end - 1], from = a.rowptr[v], to = a.rowptr[v + 1];
    if (to - from <= a.span || from < begin) continue;
    const int32_t chunks = (to - 1) / a.span - chunk + 1;
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
    if (c.live > 0) {
#pragma unroll 8
      for (int32_t k = wave; k < chunks; k += kFoldWaves) {
        // the row's part in its first chunk is that chunk's last part unless the chunk begins with it
        const int64_t slot = (int64_t)(chunk + k) * 2 + (k == 0 && from > begin ? 1 : 0);
        float f[4];
        load_some<float, 4>(a.partial + slot * a.d + j, c.live, f);
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[i] += f[i];
      }
    }
    __syncthreads();  // the sums of the chunk before have been read
#pragma unroll
    for (int i = 0; i < 4; ++i) lds[wave][lane * 4 + i] = sum[i];
    __syncthreads();
    if (wave != 0 || c.live <= 0) continue;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      sum[i] = 0.f;
      for (int w = 0; w < kFoldWaves; ++w) sum[i] += lds[w][lane * 4 + i];
      sum[i] *= a.scale;
    }
    O *out = (O *)a.out + v * a.ldo;
    if (a.beta != 0.f) {
      float old[4];
      load_some<O, 4>(out + j, c.live, old);
#pragma unroll
      for (int i = 0; i < 4; ++i) sum[i] += a.beta * old[i];
    }
    store_some<O, 4>(out + j, c.live, sum);
  }
}

// ---- host side ------------------------------------------------------------------------------------
struct EmbPlan {
  int passes, dbits;
  int64_t tiles, chunks;
  int32_t span;
  size_t key[2], pos[2], hist, totals, rowptr, partial, bytes;  // offsets into the workspace
};
static EmbPlan emb_plan(int64_t n, int64_t rows, int32_t d) {
  EmbPlan p = {};
  int bits = bits_for((int32_t)(rows + 1));
  p.passes = bits > 0 ? (bits + kMaxDigit - 1) / kMaxDigit : 1;
  p.dbits = bits > 0 ? (bits + p.passes - 1) / p.passes : 1;
  p.tiles = ceil_div64(n, kEmbTile);
  // about sqrt(n / 128): the longest chain of additions in a team and the longest list of partial rows grow alike
  p.span = 32;
  while (p.span < 512 && (int64_t)p.span * p.span * 128 < n) p.span *= 2;
  p.chunks = ceil_div64(n, p.span);
  size_t at = 0;
  auto take = [&at](size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) & ~(size_t)255;
    return here;
  };
  for (int k = 0; k < 2; ++k) p.key[k] = take((size_t)n * 4), p.pos[k] = take((size_t)n * 4);
  p.hist = take((size_t)p.tiles * ((size_t)1 << p.dbits) * 4);
  p.totals = take((size_t)kMaxRadix * 4);
  p.rowptr = take((size_t)(rows + 2) * 4);
  p.partial = take((size_t)p.chunks * 2 * (size_t)d * 4);
  p.bytes = at;
  return p;
}

static int check_lookup(const char *who, int64_t n, int64_t rows, int32_t d) {
  if (n < 0 || rows <= 0 || d <= 0)
    CG_FAIL(CG_ERR_SIZE, "%s: n=%lld indices into rows=%lld of d=%d elements", who, (long long)n, (long long)rows, d);
  if (n > 0x7fff0000LL || rows > 0x7ffffffdLL)
    CG_FAIL(CG_ERR_OVERFLOW, "%s: n=%lld, rows=%lld overflow int32 positions", who, (long long)n, (long long)rows);
  return CG_OK;
}

}  // namespace cg

extern "C" {

int cg_embedding_fwd(const void *d_table, int64_t ldt, int64_t rows, const void *d_idx, int idx64, int64_t n, int32_t d,
                     int dtype, float scale, void *d_out, int64_t ldo, cg_stream_t stream) {
  using namespace cg;
  const char *who = "cg_embedding_fwd";
  CG_TRY(check_dtype(who, dtype));
  CG_TRY(check_lookup(who, n, rows, d));
  if (n == 0) return CG_OK;
  if (!d_table || !d_idx || !d_out) CG_FAIL(CG_ERR_NULL, "%s: null pointer", who);
  if (ldt < d || ldo < d) CG_FAIL(CG_ERR_SIZE, "%s: leading dimension smaller than d", who);
  if (d_out == d_table) CG_FAIL(CG_ERR_ALIAS, "%s: the output may not be the table", who);
  hipStream_t s = (hipStream_t)stream;
  ProfScope prof("embedding_fwd", d, s);
  const int lanes_log = lanes_log2(d, dtype == CG_F32 ? 4 : 8);
  int64_t groups = ceil_div64(n, (int64_t)(kEmbThreads >> lanes_log) * kLookups);
  if (groups > 256 * 64) groups = 256 * 64;
  const IndexView view = {d_idx, idx64 != 0};
#define CG_CALL(DT)                                                                                              \
  embedding_fwd_kernel<DT><<<(unsigned)groups, kEmbThreads, 0, s>>>((const Elem<DT>::type *)d_table, ldt, rows, view, n, \
                                                                     d, scale, lanes_log, (Elem<DT>::type *)d_out, ldo)
  CG_BY_DTYPE(dtype, CG_CALL)
#undef CG_CALL
  CG_LAUNCH_CHECK();
  return CG_OK;
}

int cg_embedding_bwd_workspace(int64_t n, int64_t rows, int32_t d, int64_t *bytes) {
  using namespace cg;
  if (!bytes) CG_FAIL(CG_ERR_NULL, "cg_embedding_bwd_workspace: null pointer");
  CG_TRY(check_lookup("cg_embedding_bwd_workspace", n, rows, d));
  *bytes = (int64_t)emb_plan(n, rows, d).bytes;
  return CG_OK;
}

int cg_embedding_bwd(const void *d_g, int64_t ldg, const void *d_idx, int idx64, int64_t n, int64_t rows, int32_t d,
                     int dtype, int out_dtype, float scale, float beta, void *d_out, int64_t ldo, void *d_work,
                     int64_t work_bytes, cg_stream_t stream) {
  using namespace cg;
  const char *who = "cg_embedding_bwd";
  CG_TRY(check_dtype(who, dtype));
  if (out_dtype != dtype && out_dtype != CG_F32)
    CG_FAIL(CG_ERR_UNSUPPORTED, "%s: output dtype %d for gradients of dtype %d (the same or CG_F32)", who, out_dtype, dtype);
  CG_TRY(check_lookup(who, n, rows, d));
  if (!d_out || !d_work || (n > 0 && (!d_g || !d_idx))) CG_FAIL(CG_ERR_NULL, "%s: null pointer", who);
  if (ldo < d || (n > 0 && ldg < d)) CG_FAIL(CG_ERR_SIZE, "%s: leading dimension smaller than d", who);
  if (d_out == d_g) CG_FAIL(CG_ERR_ALIAS, "%s: the output may not be the input", who);
  const EmbPlan p = emb_plan(n, rows, d);
  if (work_bytes < (int64_t)p.bytes) CG_FAIL(CG_ERR_SIZE, "%s: workspace of %lld bytes, %lld needed", who, (long long)work_bytes, (long long)p.bytes);
  hipStream_t s = (hipStream_t)stream;
  ProfScope prof("embedding_bwd", d, s);
  char *w = static_cast<char *>(d_work);
  int32_t *key[2] = {(int32_t *)(w + p.key[0]), (int32_t *)(w + p.key[1])};
  int32_t *pos[2] = {(int32_t *)(w + p.pos[0]), (int32_t *)(w + p.pos[1])};
  uint32_t *hist = (uint32_t *)(w + p.hist), *totals = (uint32_t *)(w + p.totals);
  int32_t *rowptr = (int32_t *)(w + p.rowptr);
  int last = 0;
  if (n > 0) {
    KeySource src = {{d_idx, idx64 != 0}, nullptr, nullptr, rows};
    for (int pass = 0; pass < p.passes; ++pass) {
      const int to = pass & 1, shift = pass * p.dbits, radix = 1 << p.dbits;
      emb_hist_kernel<<<(unsigned)p.tiles, kEmbThreads, 0, s>>>(src, n, shift, p.dbits, hist, p.tiles);
      CG_LAUNCH_CHECK();
      emb_scan_kernel<<<(unsigned)ceil_div64(radix, kEmbWaves), kEmbThreads, 0, s>>>(hist, p.tiles, radix, totals);
      CG_LAUNCH_CHECK();
      emb_scatter_kernel<<<(unsigned)p.tiles, kEmbThreads, 0, s>>>(src, n, shift, p.dbits, hist, p.tiles, totals, key[to], pos[to]);
      CG_LAUNCH_CHECK();
      src.key = key[to], src.pos = pos[to];
      last = to;
    }
  }
  CG_TRY(launch_rowptr(key[last], n, (int32_t)(rows + 1), rowptr, s));
  const int lanes_log = lanes_log2(d, dtype == CG_F32 ? 4 : 8), teams = kEmbThreads >> lanes_log;
  SumArgs a = {};
  a.g = d_g, a.ldg = ldg, a.rowptr = rowptr, a.key = key[last], a.pos = pos[last], a.rows = rows, a.n = (int32_t)n, a.d = d;
  a.span = p.span, a.scale = scale, a.beta = beta, a.out = d_out, a.ldo = ldo, a.partial = (float *)(w + p.partial);
  a.chunk_teams = (unsigned)p.chunks, a.chunk_groups = (unsigned)ceil_div64(p.chunks, teams);
  int64_t groups = ceil_div64(rows, teams);
  if (groups > 256 * 64) groups = 256 * 64;
  groups += a.chunk_groups;
#define CG_CALL(DT)                                                                  \
  if (out_dtype == CG_F32)                                                           \
    emb_sum_kernel<DT, true><<<(unsigned)groups, kEmbThreads, 0, s>>>(a, lanes_log); \
  else                                                                               \
    emb_sum_kernel<DT, false><<<(unsigned)groups, kEmbThreads, 0, s>>>(a, lanes_log)
  CG_BY_DTYPE(dtype, CG_CALL)
#undef CG_CALL
  CG_LAUNCH_CHECK();
  if (n <= p.span) return CG_OK;  // no row can be hot
  const dim3 fold((unsigned)(p.chunks < 65536 ? p.chunks : 65536), (unsigned)ceil_div64(d, kFoldColumns));
#define CG_CALL(OT) emb_fold_kernel<OT><<<fold, kWave * kFoldWaves, 0, s>>>(a)
  CG_BY_DTYPE(out_dtype, CG_CALL)
#undef CG_CALL
  CG_LAUNCH_CHECK();
  return CG_OK;
}

}  // extern "C"
