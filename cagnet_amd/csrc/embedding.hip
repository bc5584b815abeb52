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
// lookup: kLookups rows a team at once, all indices loaded before the first row and all rows before the first store.
// Bound by memory: 131,072 x 1024 float32 from 65,536 rows 173 us = 4.7 TB/s of rows read once and written (185 us with
// two rows at once, 173 with eight); 232,965 x 128 from 50,021 rows 28 us (28 and 29 us).  Rows that end inside 16 bytes
// take them whole too: 605,100 x 55 float16 22 us, 36 with the last ones shifted and stored one by one.
// ---------------------------------------------------------------------------------------------
constexpr int kLookups = 4;

template <int DT, int FIT>
__global__ __launch_bounds__(kEmbThreads) void embedding_fwd_kernel(const typename Elem<DT>::type *__restrict__ table,
                                                                    int64_t ldt, int64_t rows, IndexView idx, int64_t n,
                                                                    int32_t d, float scale, int lanes_log,
                                                                    typename Elem<DT>::type *__restrict__ out,
                                                                    int64_t ldo) {
  typedef typename Elem<DT>::type T;
  typedef Span<T, FIT> C;
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
// Stable radix sort of (key, position), digits of up to 10 bits: tables of up to a thousand rows take one pass, up to a
// million two.  A workgroup of 16 wavefronts holds a tile of 4096 keys.  One tile is sorted in LDS by one launch; up to kDirectTiles
// tiles take two launches a pass (count, scatter: every scatter workgroup adds the tiles' counts up itself, one row of
// counts a tile); more tiles take a third that scans the counts, one wavefront a digit.
// ---------------------------------------------------------------------------------------------
constexpr int kSortThreads = 1024, kSortWaves = kSortThreads / kWave;
constexpr int kMaxDigit = 10, kMaxRadix = 1 << kMaxDigit;
constexpr int kKeysPerLane = 4;
constexpr int kSortTile = kSortThreads * kKeysPerLane;
constexpr int kWaveKeys = kWave * kKeysPerLane;
constexpr int kDirectTiles = 64;

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

struct Segment {
  int32_t from, to;  // sorted positions of one table row; to == 0: none
};

// Hot rows are listed by one atomic each; kHotLists counters in cache lines of their own share them, because atomics on one
// address follow each other at 25 ns (1,000,000 x 60 float32 popular indices: 126 us with one counter, 116 with eight; in
// chunks of 8 434 and 139).
constexpr int kHotLists = 8, kHotStride = 64;

// Counts of a tile's digits, at hist[digit * digit_step + tile * tile_step].  Workgroups behind the tiles clear the table
// rows' segments meanwhile.
__global__ __launch_bounds__(kSortThreads) void emb_hist_kernel(KeySource src, int64_t n, int shift, int dbits,
                                                                uint32_t *__restrict__ hist, int64_t digit_step,
                                                                int64_t tile_step, int64_t tiles,
                                                                Segment *__restrict__ segments) {
  __shared__ uint32_t count[kMaxRadix];
  if ((int64_t)blockIdx.x >= tiles) {
    const int64_t step = (int64_t)(gridDim.x - tiles) * kSortThreads;
    for (int64_t v = ((int64_t)blockIdx.x - tiles) * kSortThreads + threadIdx.x; v < src.rows; v += step) segments[v] = Segment{0, 0};
    return;
  }
  const int radix = 1 << dbits;
  if ((int)threadIdx.x < radix) count[threadIdx.x] = 0;
  const int64_t base = (int64_t)blockIdx.x * kSortTile;
  int32_t k[kKeysPerLane];
#pragma unroll
  for (int r = 0; r < kKeysPerLane; ++r) {
    const int64_t i = base + r * kSortThreads + threadIdx.x;
    k[r] = key_at(src, i < n ? i : n - 1);
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kKeysPerLane; ++r)
    if (base + r * kSortThreads + threadIdx.x < n) atomicAdd(&count[((uint32_t)k[r] >> shift) & (radix - 1)], 1u);
  __syncthreads();
  if ((int)threadIdx.x < radix) hist[threadIdx.x * digit_step + blockIdx.x * tile_step] = count[threadIdx.x];
}

// one wavefront per digit: exclusive prefix of its counts over the tiles, in place, and their total
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

struct SortLds {
  uint32_t count[kSortWaves][kMaxRadix];  // of a wavefront's digits, then their offsets in the tile
  uint32_t before[kSortThreads], all[kSortThreads];
  uint32_t wave_sums[kSortWaves];
  int32_t key[kSortTile], pos[kSortTile];
};

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
#pragma unroll
  for (int w = 0; w < kSortWaves; ++w) before += w < wave ? wave_sums[w] : 0u;
  return before + inc - v;
}

// Orders the tile's `here` keys by one digit in LDS; thread t < radix gets the first place of digit t in the tile.
// Wave w owns keys [256 w, 256 (w + 1)) of the tile, 64 at a time in order.  Lanes with equal digits find each other
// by ballots; a key's rank is the wave's running count of its digit plus the equal lanes below it.
__device__ __forceinline__ uint32_t sort_tile(SortLds &s, const int32_t (&key)[kKeysPerLane], const int32_t (&pos)[kKeysPerLane],
                                              int here, int shift, int dbits) {
  const int radix = 1 << dbits, lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  for (int i = threadIdx.x; i < kSortWaves * radix; i += kSortThreads) s.count[i >> dbits][i & (radix - 1)] = 0;
  __syncthreads();
  uint32_t rank[kKeysPerLane];
  const uint64_t below = (1ull << lane) - 1ull;
#pragma unroll
  for (int r = 0; r < kKeysPerLane; ++r) {
    rank[r] = 0;
    if (wave * kWaveKeys + r * kWave >= here) continue;  // the whole wavefront is behind the last key
    const bool valid = wave * kWaveKeys + r * kWave + lane < here;
    const uint32_t digit = ((uint32_t)key[r] >> shift) & (uint32_t)(radix - 1);
    uint64_t peers = __ballot(valid);
#pragma unroll
    for (int b = 0; b < kMaxDigit; ++b)
      if (b < dbits) {
        const bool one = (digit >> b) & 1u;
        const uint64_t with = __ballot(one);
        peers &= one ? with : ~with;
      }
    const uint32_t lower = (uint32_t)__popcll(peers & below);
    uint32_t had = 0;
    if (valid) had = s.count[wave][digit];
    // the lowest lane of the set writes the new count; it depends on `had`, so the read above comes first
    if (valid && lower == 0) s.count[wave][digit] = had + (uint32_t)__popcll(peers);
    // LDS serves a wavefront in order; the fence holds the compiler to it (it emits nothing)
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    rank[r] = had + lower;
  }
  __syncthreads();
  uint32_t mine = 0, of[kSortWaves];
  const int digit_of = (int)threadIdx.x & (radix - 1);
#pragma unroll
  for (int w = 0; w < kSortWaves; ++w) of[w] = s.count[w][digit_of];
  if ((int)threadIdx.x < radix)
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) mine += of[w];
  const uint32_t first = group_exclusive(mine, s.wave_sums);
  if ((int)threadIdx.x < radix) {
    uint32_t run = first;
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) {
      s.count[w][threadIdx.x] = run;
      run += of[w];
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kKeysPerLane; ++r)
    if (wave * kWaveKeys + r * kWave + lane < here) {
      const uint32_t digit = ((uint32_t)key[r] >> shift) & (uint32_t)(radix - 1);
      const uint32_t at = s.count[wave][digit] + rank[r];
      s.key[at] = key[r];
      s.pos[at] = pos[r];
    }
  __syncthreads();
  return first;
}

// DIRECT: hist holds one row of counts per tile; otherwise the scanned counts of emb_scan_kernel, one row per digit.
template <bool DIRECT>
__global__ __launch_bounds__(kSortThreads) void emb_scatter_kernel(KeySource src, int64_t n, int shift, int dbits,
                                                                   const uint32_t *__restrict__ hist, int64_t tiles,
                                                                   const uint32_t *__restrict__ totals,
                                                                   int32_t *__restrict__ out_key,
                                                                   int32_t *__restrict__ out_pos, int32_t *__restrict__ hot_count) {
  __shared__ SortLds s;
  const int radix = 1 << dbits, lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const int64_t tile_base = (int64_t)blockIdx.x * kSortTile, left = n - tile_base;
  const int here = (int)(left < kSortTile ? left : kSortTile);
  if (blockIdx.x == 0 && (int)threadIdx.x < kHotLists) hot_count[threadIdx.x * kHotStride] = 0;
  int32_t key[kKeysPerLane], pos[kKeysPerLane];
#pragma unroll
  for (int r = 0; r < kKeysPerLane; ++r) {
    const int64_t i = tile_base + wave * kWaveKeys + r * kWave + lane, at = i < n ? i : n - 1;
    key[r] = key_at(src, at);
    pos[r] = src.pos ? src.pos[at] : (int32_t)at;
  }
  uint32_t before = 0, all = 0;  // of digit threadIdx.x % radix: in the tiles below, in all of them
  if (DIRECT) {
    const int digit = threadIdx.x & (radix - 1), parts = kSortThreads >> dbits;
#pragma unroll 8
    for (int t = threadIdx.x >> dbits; t < (int)tiles; t += parts) {
      const uint32_t c = hist[(int64_t)t * radix + digit];
      before += t < (int)blockIdx.x ? c : 0u;
      all += c;
    }
    s.before[threadIdx.x] = before;
    s.all[threadIdx.x] = all;
    __syncthreads();
    before = all = 0;
    if ((int)threadIdx.x < radix)
      for (int k = 0; k < parts; ++k) {
        before += s.before[(k << dbits) + threadIdx.x];
        all += s.all[(k << dbits) + threadIdx.x];
      }
  } else if ((int)threadIdx.x < radix) {
    before = hist[(int64_t)threadIdx.x * tiles + blockIdx.x];
    all = totals[threadIdx.x];
  }
  const uint32_t start = group_exclusive(all, s.wave_sums);
  const uint32_t first = sort_tile(s, key, pos, here, shift, dbits);
  // global place of a record = first place of its digit here + its place in the tile, modulo 2^32
  if ((int)threadIdx.x < radix) s.before[threadIdx.x] = start + before - first;
  __syncthreads();
  for (int i = threadIdx.x; i < here; i += kSortThreads) {
    const uint32_t to = s.before[((uint32_t)s.key[i] >> shift) & (uint32_t)(radix - 1)] + (uint32_t)i;
    out_key[to] = s.key[i];
    out_pos[to] = s.pos[i];
  }
}

// The segments of the table rows that have positions, and how many positions are inside the table: one thread per place
// between two sorted keys.  Rows without positions cost nothing here, however many of them lie between two keys.
__global__ __launch_bounds__(kEmbThreads) void emb_segment_kernel(const int32_t *__restrict__ key, int32_t n, int32_t rows,
                                                                  Segment *__restrict__ segments, int32_t *__restrict__ count) {
  const int32_t i = (int32_t)((int64_t)blockIdx.x * kEmbThreads + threadIdx.x);
  if (i > n) return;
  const int32_t before = i > 0 ? key[i - 1] : -1, here = i < n ? key[i] : rows;
  if (before != here) {
    if (before >= 0) segments[before].to = i;
    if (here < rows) segments[here].from = i;
  }
  if (before < rows && here == rows) *count = i;
}

// ---------------------------------------------------------------------------------------------
// Sums.  The sorted array is cut into chunks of `span` positions, one team of lanes each.  A table row with up to
// `span` positions ("light") is added up and written by the team whose chunk it begins in, also where it ends behind
// the chunk; the team streams through the positions with the same number of rows of g in flight whatever the rows of
// the table they belong to.  A row with more ("hot": with popular indices one can hold a tenth of all positions) covers
// the end of at least one chunk, so a chunk holds a part of at most two hot rows, the one it begins in and the one it
// ends in.  The team adds up each part into a partial row, and a second kernel adds a hot row's partial rows in order.
// Where all chunks of a workgroup lie inside one hot row (padding can make one row hold half of all positions) their
// sums are added in LDS first, and only the workgroup's first chunk has a partial row.
// ---------------------------------------------------------------------------------------------
struct SumArgs {
  const void *g;
  int64_t ldg;
  const Segment *segments;  // of every table row; nullptr after the one-launch sort, then `ends`
  const Segment *ends;    // of every chunk: the segments of its first and of its last position
  const int32_t *count;   // positions whose index is inside the table
  const int32_t *key, *pos;
  int64_t rows;
  int32_t d, span, chunks;
  float scale, beta;
  void *out;
  int64_t ldo;
  float *partial;               // [2 * chunks][d], float32
  int32_t *hot_count, *hot;     // kHotLists lists of parts (2 * chunk + which) that hot rows begin with, in any order
  int32_t hot_room;             // of one list
  int32_t teams;                // chunks of a workgroup
  unsigned chunk_groups;        // workgroups that stream; those behind them write the rows that no index names
};

// Rows of g in flight per lane: 232,965 x 128 float32 lookup and gradient 130 us with 8, 133 with 4, 132 with 16.
constexpr int kAhead = 8;

template <typename O, int V>
__device__ __forceinline__ void put_row(const SumArgs &a, int64_t v, int32_t j, int live, float (&sum)[V]) {
  O *out = (O *)a.out + v * a.ldo + j;
#pragma unroll
  for (int i = 0; i < V; ++i) sum[i] *= a.scale;
  if (a.beta != 0.f) {
    float old[V];
    load_some<O, V>(out, live, old);
#pragma unroll
    for (int i = 0; i < V; ++i) sum[i] += a.beta * old[i];
  }
  store_some<O, V>(out, live, sum);
}

// The same for a lane's 16 bytes of g's type: stored whole where nothing is read back, the elements that count otherwise
// (a repeated element would be read after the lane before has written it).
template <typename O, typename C>
__device__ __forceinline__ void put_span(const SumArgs &a, const C &c, int64_t v, float (&sum)[C::V]) {
  O *out = (O *)a.out + v * a.ldo + c.at;
#pragma unroll
  for (int i = 0; i < C::V; ++i) sum[i] *= a.scale;
  if (c.whole() && (a.beta == 0.f || c.dup == 0)) {
    if (a.beta != 0.f) {
      float old[C::V];
      load_pack<O, C::V>(out, old);
#pragma unroll
      for (int i = 0; i < C::V; ++i) sum[i] += a.beta * old[i];
    }
    store_pack<O, C::V>(out, sum);
    return;
  }
#pragma unroll
  for (int i = 0; i < C::V; ++i)
    if (c.counts(i)) out[i] = rounded<O>(a.beta != 0.f ? sum[i] + a.beta * (float)out[i] : sum[i]);
}

// Adds up the lane's columns of g's rows pos[from .. to) in order, one sum per stretch of equal keys, and hands each
// to done(key, sum).  The positions and keys of the next kAhead rows are loaded while those before are on their way.
template <typename T, typename C, typename F>
__device__ __forceinline__ void stream_rows(const SumArgs &a, const C &c, int32_t from, int32_t to, F done) {
  constexpr int V = C::V;
  if (from >= to) return;
  int32_t p[kAhead], key[kAhead], next[kAhead];
#pragma unroll
  for (int k = 0; k < kAhead; ++k) {
    const int32_t at = from + k < to ? from + k : to - 1;
    p[k] = a.pos[at];
    next[k] = a.key[at];
  }
  float sum[V];
#pragma unroll
  for (int i = 0; i < V; ++i) sum[i] = 0.f;
  int32_t now = next[0];
  for (int32_t at = from; at < to; at += kAhead) {
    Raw r[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      r[k] = Raw{0u, 0u, 0u, 0u};
      if (k == 0 || at + k < to) r[k] = c.load((const T *)a.g + (int64_t)p[k] * a.ldg);
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      key[k] = next[k];
      const int32_t ahead = at + kAhead + k < to ? at + kAhead + k : to - 1;
      p[k] = a.pos[ahead];
      next[k] = a.key[ahead];
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      float f[V];
      c.floats(r[k], f);
      if (key[k] != now) {  // never for the clamped entries behind `to`: they repeat the last key
        done(now, sum);
        now = key[k];
#pragma unroll
        for (int i = 0; i < V; ++i) sum[i] = 0.f;
      }
#pragma unroll
      for (int i = 0; i < V; ++i) sum[i] += f[i];
    }
  }
  done(now, sum);
}

__device__ __forceinline__ void list_hot(const SumArgs &a, int32_t part) {
  const int list = blockIdx.x % kHotLists;
  a.hot[(int64_t)list * a.hot_room + atomicAdd(a.hot_count + list * kHotStride, 1)] = part;
}

template <int DT, bool OUT_F32, int FIT>
__global__ __launch_bounds__(kEmbThreads) void emb_sum_kernel(SumArgs a, int lanes_log) {
  typedef typename Elem<DT>::type T;
  typedef typename Elem<OUT_F32 ? CG_F32 : DT>::type O;
  typedef Span<T, FIT> C;
  constexpr int V = C::V;
  __shared__ float sums[kEmbThreads][V];
  const int lane = threadIdx.x & ((1 << lanes_log) - 1), teams = kEmbThreads >> lanes_log, team = threadIdx.x >> lanes_log;
  const int32_t j = ((int32_t)blockIdx.y * (1 << lanes_log) + lane) * V;
  C c;
  c.place(j, a.d);
  if (blockIdx.x >= a.chunk_groups) {  // rows without positions
    float zero[V];
    if (!c.any() || a.beta == 1.f) return;
    const int64_t step = (int64_t)(gridDim.x - a.chunk_groups) * teams;
    for (int64_t v = (int64_t)(blockIdx.x - a.chunk_groups) * teams + team; v < a.rows; v += step)
      if (a.segments[v].to == 0) {
#pragma unroll
        for (int i = 0; i < V; ++i) zero[i] = 0.f;
        put_span<O>(a, c, v, zero);
      }
    return;
  }
  const int32_t chunk = (int32_t)blockIdx.x * teams + team, all = *a.count;
  if (chunk >= a.chunks || chunk * a.span >= all) return;
  const int32_t begin = chunk * a.span, end = all - begin < a.span ? all : begin + a.span;
  Segment first, last;
  if (a.segments) {
    first = a.segments[a.key[begin]];
    last = a.segments[a.key[end - 1]];
  } else {
    first = a.ends[2 * chunk];
    last = a.ends[2 * chunk + 1];
  }
  const bool hot_first = first.to - first.from > a.span, hot_last = last.to - last.from > a.span;
  const int32_t first_key = a.key[begin], last_key = a.key[end - 1];
  float *partial = a.partial + (int64_t)chunk * 2 * a.d + c.at;
  auto keep = [&](float *to, const float (&sum)[V]) {
    if (FIT != kShortRow) {
      store_pack<float, V>(to, sum);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (c.counts(i)) to[i] = sum[i];
    }
  };
  const int32_t group = (int32_t)blockIdx.x * teams * a.span;
  if (teams > 1 && first.from <= group && first.to - group >= teams * a.span) {  // of every thread alike; hot with two teams
    stream_rows<T>(a, c, begin, end, [&](int32_t, float (&sum)[V]) {
#pragma unroll
      for (int i = 0; i < V; ++i) sums[threadIdx.x][i] = sum[i];
    });
    __syncthreads();
    if (team != 0) return;
    float sum[V];
#pragma unroll
    for (int i = 0; i < V; ++i) sum[i] = 0.f;
    for (int t = 0; t < teams; ++t)
#pragma unroll
      for (int i = 0; i < V; ++i) sum[i] += sums[(t << lanes_log) + lane][i];
    if (c.any()) keep(partial, sum);
    if (first.from == begin && lane == 0 && blockIdx.y == 0) list_hot(a, 2 * chunk);
    return;
  }
  if (lane == 0 && blockIdx.y == 0) {
    if (hot_first && first.from == begin) list_hot(a, 2 * chunk);
    if (hot_last && last.from > begin) list_hot(a, 2 * chunk + 1);
  }
  // a light row that began in the chunk before is that chunk's, one that begins here is followed behind the end
  const int32_t from = !hot_first && first.from < begin ? first.to : begin, to = hot_last ? end : last.to;
  stream_rows<T>(a, c, from, to, [&](int32_t v, float (&sum)[V]) {
    if (!c.any()) return;
    if (hot_first && v == first_key)
      keep(partial, sum);
    else if (hot_last && v == last_key)
      keep(partial + a.d, sum);
    else
      put_span<O>(a, c, v, sum);
  });
}

// The partial rows of the hot rows, 256 columns a workgroup (of as many hot rows side by side as these hold): its 16
// wavefronts take every 16th partial row each, their sums are added in order.
constexpr int kFoldWaves = 16, kFoldColumns = kWave * 4;

template <int OT>
__global__ __launch_bounds__(kWave *kFoldWaves) void emb_fold_kernel(SumArgs a, int lanes_log) {
  typedef typename Elem<OT>::type O;
  __shared__ float lds[kFoldWaves][kFoldColumns];
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const int team = lane >> lanes_log, teams = kWave >> lanes_log;
  const int32_t j = blockIdx.y * kFoldColumns + (lane & ((1 << lanes_log) - 1)) * 4, all = *a.count;
  const int live = a.d - j < 4 ? a.d - j : 4;
  int32_t in_list[kHotLists], hot = 0;
#pragma unroll
  for (int l = 0; l < kHotLists; ++l) in_list[l] = a.hot_count[l * kHotStride];
#pragma unroll
  for (int l = 0; l < kHotLists; ++l) hot += in_list[l];
  for (int32_t h0 = blockIdx.x * teams; h0 < hot; h0 += gridDim.x * teams) {  // uniform in the workgroup
    int32_t h = h0 + team < hot ? h0 + team : h0, list = 0;  // the h-th of all lists
#pragma unroll
    for (int l = 0; l < kHotLists - 1; ++l)
      if (list == l && h >= in_list[l]) h -= in_list[l], ++list;
    const int32_t part = a.hot[(int64_t)list * a.hot_room + h];
    const int32_t chunk = part >> 1, which = part & 1, begin = chunk * a.span;
    const bool mine = h0 + team < hot && live > 0;
    const int32_t end = all - begin < a.span ? all : begin + a.span;
    const int32_t v = a.key[which ? end - 1 : begin];
    const Segment seg = a.segments ? a.segments[v] : a.ends[2 * chunk + which];
    // chunks with partial rows: those before the first whole workgroup of chunks, one of every whole workgroup, those behind
    const int32_t wide = a.span * a.teams, tail = (seg.to - 1) / a.span;
    int32_t lo = (seg.from + wide - 1) / wide, hi = seg.to / wide;
    if (hi < lo) lo = hi = (chunk + a.teams - 1) / a.teams;
    const int32_t head = lo * a.teams - chunk, whole = hi - lo, parts = head + whole + tail - hi * a.teams + 1;
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
    if (mine) {
#pragma unroll 8
      for (int32_t k = wave; k < parts; k += kFoldWaves) {
        const int32_t at = k < head ? chunk + k : k < head + whole ? (lo + k - head) * a.teams : hi * a.teams + k - head - whole;
        const int64_t slot = (int64_t)at * 2 + (at == chunk ? which : 0);
        float f[4];
        load_some<float, 4>(a.partial + slot * a.d + j, live, f);
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[i] += f[i];
      }
    }
    __syncthreads();  // the sums of the rows before have been read
#pragma unroll
    for (int i = 0; i < 4; ++i) lds[wave][lane * 4 + i] = sum[i];
    __syncthreads();
    if (wave != 0 || !mine) continue;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      sum[i] = 0.f;
      for (int w = 0; w < kFoldWaves; ++w) sum[i] += lds[w][lane * 4 + i];
    }
    put_row<O, 4>(a, v, j, live, sum);
  }
}

// One tile of indices: workgroup 0 sorts it in LDS and finds the chunks' first and last segments by bisection; the
// others clear the table meanwhile (beta == 0), whose named rows the sums then overwrite.
// first place of a key not below v, and of one above it
__device__ __forceinline__ Segment segment_of(const int32_t *key, int32_t n, int32_t v) {
  Segment lo = {0, 0}, hi = {n, n};
  while (lo.from < hi.from || lo.to < hi.to) {  // both bisections side by side: each step is an LDS round trip
    const int32_t m = (lo.from + hi.from) >> 1, k = (lo.to + hi.to) >> 1;
    const int32_t km = key[m < n ? m : n - 1], kk = key[k < n ? k : n - 1];
    if (lo.from < hi.from) {
      if (km < v)
        lo.from = m + 1;
      else
        hi.from = m;
    }
    if (lo.to < hi.to) {
      if (kk <= v)
        lo.to = k + 1;
      else
        hi.to = k;
    }
  }
  return lo;
}

template <typename O>
__global__ __launch_bounds__(kSortThreads) void emb_small_kernel(KeySource src, int32_t n, int passes, int dbits, int32_t span,
                                                                 int32_t *__restrict__ out_key, int32_t *__restrict__ out_pos,
                                                                 Segment *__restrict__ ends, int32_t *__restrict__ count,
                                                                 int32_t *__restrict__ hot_count, O *__restrict__ out,
                                                                 int64_t ldo, int32_t d) {
  __shared__ SortLds s;
  if (blockIdx.x > 0) {
    constexpr int V = 16 / (int)sizeof(O);
    const int32_t per_row = (d + V - 1) / V;
    const uint32_t step = (gridDim.x - 1) * kSortThreads, first = (blockIdx.x - 1) * kSortThreads + threadIdx.x;
    const uint32_t rows_on = step / per_row, chunks_on = step % per_row;
    float zero[V];
#pragma unroll
    for (int i = 0; i < V; ++i) zero[i] = 0.f;
    uint32_t at = first % per_row;
    for (int64_t row = first / per_row; row < src.rows; row += rows_on) {
      const int32_t j = (int32_t)at * V;
      store_some<O, V>(out + row * ldo + j, d - j < V ? d - j : V, zero);
      at += chunks_on;
      if (at >= (uint32_t)per_row) at -= per_row, ++row;
    }
    return;
  }
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  int32_t key[kKeysPerLane], pos[kKeysPerLane];
  int at[kKeysPerLane];
#pragma unroll
  for (int r = 0; r < kKeysPerLane; ++r) {
    const int i = wave * kWaveKeys + r * kWave + lane;
    at[r] = i < n ? i : n - 1;
    key[r] = key_at(src, at[r]);
    pos[r] = at[r];
  }
  for (int pass = 0; pass < passes; ++pass) {
    if (pass > 0) {
#pragma unroll
      for (int r = 0; r < kKeysPerLane; ++r) {
        key[r] = s.key[at[r]];
        pos[r] = s.pos[at[r]];
      }
      __syncthreads();
    }
    (void)sort_tile(s, key, pos, n, pass * dbits, dbits);
  }
  for (int i = threadIdx.x; i < n; i += kSortThreads) {
    out_key[i] = s.key[i];
    out_pos[i] = s.pos[i];
  }
  const int32_t all = segment_of(s.key, n, (int32_t)src.rows).from;
  if (threadIdx.x == 0) *count = all;
  if ((int)threadIdx.x < kHotLists) hot_count[threadIdx.x * kHotStride] = 0;
  for (int32_t e = threadIdx.x; (e >> 1) * span < all; e += kSortThreads) {
    const int32_t begin = (e >> 1) * span, end = all - begin < span ? all : begin + span;
    const int32_t v = s.key[(e & 1) ? end - 1 : begin];
    ends[e] = segment_of(s.key, n, v);
  }
}

// ---- host side ------------------------------------------------------------------------------------
struct EmbPlan {
  int passes, dbits;
  int64_t tiles, chunks;
  int32_t span;
  size_t key[2], pos[2], hist, totals, segments, ends, counters, hot, partial, bytes;  // offsets into the workspace
};
static EmbPlan emb_plan(int64_t n, int64_t rows, int32_t d, size_t elem) {
  EmbPlan p = {};
  const int bits = bits_for((int32_t)(rows + 1));
  p.passes = (bits + kMaxDigit - 1) / kMaxDigit;
  p.dbits = (bits + p.passes - 1) / p.passes;
  p.tiles = ceil_div64(n, kSortTile);
  // About sqrt(n / 256): the longest chain of additions in a team and the longest list of partial rows grow alike.
  // The gradient of 232,965 x 128 float32 with popular indices takes 69 us in chunks of 64 and of 32 (as here), 71 in chunks
  // of 16; 131,072 x 1024 bf16 144 us in chunks of 32 (as here) and 156 in chunks of 16.
  p.span = 8;
  while (p.span < 512 && (int64_t)p.span * p.span * 256 < n) p.span *= 2;
  // Rows of up to 128 bytes take 8 lanes or fewer: a quarter of that, or too few wavefronts run to hide their loads (1,000,000
  // x 8 bf16 96 -> 73 us, 100,000 x 64 bf16 39 -> 31; rows of 240 bytes 116 -> 125, of 256 all of one row 128 -> 165).
  if ((size_t)d * elem <= 128) p.span = p.span > 32 ? p.span / 4 : 8;
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
  p.segments = take((size_t)rows * sizeof(Segment));
  p.ends = take(p.tiles <= 1 ? (size_t)p.chunks * 2 * sizeof(Segment) : 0);
  p.counters = take((size_t)(1 + kHotLists) * kHotStride * 4);  // positions inside the table; hot rows of every list
  p.hot = take(((size_t)p.chunks * 2 + 2 * kHotLists * kEmbThreads) * 4);
  p.partial = take((size_t)p.chunks * 2 * (size_t)d * 4);
  p.bytes = at;
  return p;
}

static int check_lookup(const char *who, int64_t n, int64_t rows, int32_t d) {
  if (n < 0 || rows < 0 || (rows == 0 && n > 0) || d <= 0)
    CG_FAIL(CG_ERR_SIZE, "%s: n=%lld indices into rows=%lld of d=%d elements", who, (long long)n, (long long)rows, d);
  if (d > (1 << 23)) CG_FAIL(CG_ERR_OVERFLOW, "%s: rows of d=%d elements (at most 2^23)", who, d);
  if (n > 0x7ff00000LL || rows > 0x7ffffffdLL)
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
  const int32_t v = dtype == CG_F32 ? 4 : 8;
#define CG_FIT(DT, FIT)                                                                                                   \
  embedding_fwd_kernel<DT, FIT><<<(unsigned)groups, kEmbThreads, 0, s>>>((const Elem<DT>::type *)d_table, ldt, rows, view, \
                                                                          n, d, scale, lanes_log, (Elem<DT>::type *)d_out, ldo)
#define CG_CALL(DT)              \
  if (d % v == 0)                \
    CG_FIT(DT, kWholeChunks);    \
  else if (d < v)                \
    CG_FIT(DT, kShortRow);       \
  else                           \
    CG_FIT(DT, kPartChunk)
  CG_BY_DTYPE(dtype, CG_CALL)
#undef CG_FIT
#undef CG_CALL
  CG_LAUNCH_CHECK();
  return CG_OK;
}

int cg_embedding_bwd_workspace(int64_t n, int64_t rows, int32_t d, int64_t *bytes) {
  using namespace cg;
  if (!bytes) CG_FAIL(CG_ERR_NULL, "cg_embedding_bwd_workspace: null pointer");
  CG_TRY(check_lookup("cg_embedding_bwd_workspace", n, rows, d));
  *bytes = 0;
  if (rows == 0) return CG_OK;
  const size_t wide = emb_plan(n, rows, d, 4).bytes, narrow = emb_plan(n, rows, d, 2).bytes;
  *bytes = (int64_t)(wide > narrow ? wide : narrow);
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
  if (rows == 0) return CG_OK;
  if (!d_out || !d_work || (n > 0 && (!d_g || !d_idx))) CG_FAIL(CG_ERR_NULL, "%s: null pointer", who);
  if (ldo < d || (n > 0 && ldg < d)) CG_FAIL(CG_ERR_SIZE, "%s: leading dimension smaller than d", who);
  if (d_out == d_g) CG_FAIL(CG_ERR_ALIAS, "%s: the output may not be the input", who);
  const EmbPlan p = emb_plan(n, rows, d, elem_size(dtype));
  CG_TRY(check_work(who, d_work, work_bytes, (int64_t)p.bytes));
  hipStream_t s = (hipStream_t)stream;
  ProfScope prof("embedding_bwd", d, s);
  char *w = static_cast<char *>(d_work);
  int32_t *key[2] = {(int32_t *)(w + p.key[0]), (int32_t *)(w + p.key[1])};
  int32_t *pos[2] = {(int32_t *)(w + p.pos[0]), (int32_t *)(w + p.pos[1])};
  uint32_t *hist = (uint32_t *)(w + p.hist), *totals = (uint32_t *)(w + p.totals);
  Segment *segments = (Segment *)(w + p.segments);
  int32_t *counters = (int32_t *)(w + p.counters);
  SumArgs a = {};
  a.g = d_g, a.ldg = ldg, a.count = counters, a.rows = rows, a.d = d, a.span = p.span, a.chunks = (int32_t)p.chunks;
  a.scale = scale, a.beta = beta, a.out = d_out, a.ldo = ldo, a.partial = (float *)(w + p.partial);
  a.hot_count = counters + kHotStride, a.hot = (int32_t *)(w + p.hot);
  KeySource src = {{d_idx, idx64 != 0}, nullptr, nullptr, rows};
  const bool small = n > 0 && p.tiles <= 1 && (beta == 0.f || beta == 1.f);
  if (small) {
    Segment *ends = (Segment *)(w + p.ends);
    const int64_t units = beta == 0.f ? rows * ceil_div64(d, out_dtype == CG_F32 ? 4 : 8) : 0;
    int64_t groups = ceil_div64(units, kSortThreads * 4);
    groups = 1 + (groups < 1024 ? groups : 1024);
#define CG_CALL(OT)                                                                                                     \
  emb_small_kernel<<<(unsigned)groups, kSortThreads, 0, s>>>(src, (int32_t)n, p.passes, p.dbits, p.span, key[0], pos[0], ends, \
                                                             counters, counters + kHotStride, (Elem<OT>::type *)d_out, ldo, d)
    CG_BY_DTYPE(out_dtype, CG_CALL)
#undef CG_CALL
    CG_LAUNCH_CHECK();
    a.key = key[0], a.pos = pos[0], a.ends = ends;
  } else {
    int last = 0;
    const bool direct = p.tiles <= kDirectTiles;
    const int radix = 1 << p.dbits;
    int64_t clearing = ceil_div64(rows, kSortThreads * 4);
    if (clearing > 1024) clearing = 1024;
    if (n == 0) {
      emb_hist_kernel<<<(unsigned)clearing, kSortThreads, 0, s>>>(src, 0, 0, p.dbits, hist, 0, 0, 0, segments);
      CG_LAUNCH_CHECK();
    }
    for (int pass = 0; n > 0 && pass < p.passes; ++pass) {
      const int to = pass & 1, shift = pass * p.dbits;
      const int64_t groups = p.tiles + (pass == 0 ? clearing : 0);
      emb_hist_kernel<<<(unsigned)groups, kSortThreads, 0, s>>>(src, n, shift, p.dbits, hist, direct ? 1 : p.tiles,
                                                                direct ? radix : 1, p.tiles, segments);
      CG_LAUNCH_CHECK();
      if (direct) {
        emb_scatter_kernel<true><<<(unsigned)p.tiles, kSortThreads, 0, s>>>(src, n, shift, p.dbits, hist, p.tiles, totals,
                                                                            key[to], pos[to], counters + kHotStride);
      } else {
        emb_scan_kernel<<<(unsigned)ceil_div64(radix, kEmbWaves), kEmbThreads, 0, s>>>(hist, p.tiles, radix, totals);
        CG_LAUNCH_CHECK();
        emb_scatter_kernel<false><<<(unsigned)p.tiles, kSortThreads, 0, s>>>(src, n, shift, p.dbits, hist, p.tiles, totals,
                                                                             key[to], pos[to], counters + kHotStride);
      }
      CG_LAUNCH_CHECK();
      src.key = key[to], src.pos = pos[to];
      last = to;
    }
    if (n > 0) {
      emb_segment_kernel<<<(unsigned)ceil_div64(n + 1, kEmbThreads), kEmbThreads, 0, s>>>(key[last], (int32_t)n, (int32_t)rows,
                                                                                          segments, counters);
      CG_LAUNCH_CHECK();
    }
    a.key = key[last], a.pos = pos[last], a.segments = segments;
  }
  const int per_chunk = dtype == CG_F32 ? 4 : 8, lanes_log = lanes_log2(d, per_chunk), teams = kEmbThreads >> lanes_log;
  a.teams = teams, a.chunk_groups = (unsigned)ceil_div64(p.chunks, teams);
  a.hot_room = 2 * teams * (int32_t)ceil_div64(a.chunk_groups, kHotLists);  // every part of every chunk
  int64_t groups = small || beta == 1.f ? 0 : ceil_div64(rows, teams);
  if (groups > 256 * 16) groups = 256 * 16;
  groups += a.chunk_groups;
  if (groups == 0) return CG_OK;
  const dim3 grid((unsigned)groups, (unsigned)ceil_div64(d, (int64_t)per_chunk << lanes_log));
#define CG_FIT(DT, FIT)                                                       \
  if (out_dtype == CG_F32)                                                    \
    emb_sum_kernel<DT, true, FIT><<<grid, kEmbThreads, 0, s>>>(a, lanes_log); \
  else                                                                        \
    emb_sum_kernel<DT, false, FIT><<<grid, kEmbThreads, 0, s>>>(a, lanes_log)
#define CG_CALL(DT)               \
  if (d % per_chunk == 0) {       \
    CG_FIT(DT, kWholeChunks);     \
  } else if (d < per_chunk) {     \
    CG_FIT(DT, kShortRow);        \
  } else {                        \
    CG_FIT(DT, kPartChunk);       \
  }
  CG_BY_DTYPE(dtype, CG_CALL)
#undef CG_FIT
#undef CG_CALL
  CG_LAUNCH_CHECK();
  if (n <= p.span) return CG_OK;  // no row can be hot
  const int64_t columns = ceil_div64(d, kFoldColumns), at_once = columns < 8 ? 512 / columns : 64;  // two workgroups a CU
  const dim3 fold((unsigned)(p.chunks < at_once ? p.chunks : at_once), (unsigned)columns);
  int fold_lanes_log = lanes_log2(d, 4);
  if (fold_lanes_log > 6) fold_lanes_log = 6;
#define CG_CALL(OT) emb_fold_kernel<OT><<<fold, kWave * kFoldWaves, 0, s>>>(a, fold_lanes_log)
  CG_BY_DTYPE(out_dtype, CG_CALL)
#undef CG_CALL
  CG_LAUNCH_CHECK();
  return CG_OK;
}

}  // extern "C"
