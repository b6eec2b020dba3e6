// Embedding lookup with a scale, and the gradient of its table.
//
//   y_i = residual_i + scale table[id_i],  dtable[v] = scale sum over id_i = v of dy_i
//
// An id outside the table adds nothing and has no gradient.
//
// Memory bound.  The lookup reads whole rows in 16-byte pieces, four rows a
// lane in flight, with the next rows' ids ahead: 1,702,400 x 64 of bf16 with a
// residual 83 us (450 MB: 5.4 TB/s).
//
// The gradient has no atomics on sums, so results repeat bit for bit, by one
// of two ways:
//
// A small table of a 16-bit type fits the accumulators of one workgroup.  Its
// gradient is the product of the ids, as rows of a single one, with dy: the
// ones are made in registers by comparisons, dy comes through LDS with
// transposing reads, and each workgroup leaves one table of partial sums.  On
// the matrix cores that costs less than sorting the ids: 96 us for 1,702,400 x 64
// of 300 ids (232 MB at 2.4 TB/s; vector ALU 0.45, matrix cores 0.35, LDS 0.37
// busy, two workgroups of eight waves a CU).  A product with zero
// would spread an infinity or a NaN of dy to every id, so these are taken out
// of the tile and remembered by id and column.
//
// Otherwise the positions are sorted by their ids (stable, so in the order of
// the positions) and runs of equal ids summed: a group of lanes takes a chunk
// of the sorted positions, writes the runs that lie inside its chunk, and
// leaves a partial row for a run that began before it or goes on after it, at
// most two a chunk, which the workgroup of the run's first chunk joins.  Up to
// 8192 positions are sorted in one launch by counting the ids before each.  8192
// x 2048 of 32,000 ids: 30 us to sort and to clear the 131 MB of the table, 14
// for the runs, 9 for the joins.
#include "nest_internal.h"
#include "residual_internal.h"
#include "tile_gemm.h"

namespace nest {
namespace {

constexpr int kThreads = 256;
constexpr int kRowsInFlight = 4;
constexpr uint32_t kNoRun = 0xffffffffu;      // a partial row's key: none
constexpr uint32_t kNoRow = 0x80000000u;      // its run goes on, but there is no row

int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }
int pow2_at_least(int64_t v) {
  int p = 1;
  while (p < v) p *= 2;
  return p;
}
size_t align256(size_t b) { return (b + 255) & ~(size_t)255; }

// ---- lookup ----

template <typename T, typename I, bool kWhole>
__global__ __launch_bounds__(kThreads) void embedding_kernel(EmbeddingParams p, int lanes) {
  constexpr int N = Vec16<T>::kN, U = kRowsInFlight;
  const int lane = threadIdx.x & (lanes - 1), rows_wg = kThreads / lanes;
  const int64_t step = (int64_t)gridDim.x * rows_wg;
  const int D = p.cols;
  int64_t first = (int64_t)blockIdx.x * rows_wg + threadIdx.x / lanes;
  uint32_t next[U];   // kNoRun: none
  auto load_ids = [&](int64_t at) {
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int64_t id = at + u * step < p.rows ? (int64_t)static_cast<const I*>(p.ids)[at + u * step] : -1;
      next[u] = id >= 0 && id < p.table_rows ? (uint32_t)id : kNoRun;
    }
  };
  load_ids(first);
  for (; first < p.rows; first += step * U) {
    uint32_t at[U];
#pragma unroll
    for (int u = 0; u < U; u++) at[u] = next[u];
    load_ids(first + step * U);   // on their way while these rows are
    for (int c = (blockIdx.y * lanes + lane) * N; c < D; c += gridDim.y * lanes * N) {
      Words16<T> t[U], r[U];
#pragma unroll
      for (int u = 0; u < U; u++) {
        const int64_t row = first + u * step;
        if (p.residual) r[u] = load_words<kWhole>(static_cast<const T*>(p.residual) + row * D + c, row < p.rows ? D - c : 0);
        t[u] = load_words<kWhole>(static_cast<const T*>(p.table) + (int64_t)at[u] * D + c, at[u] != kNoRun ? D - c : 0);
      }
#pragma unroll
      for (int u = 0; u < U; u++) {
        const int64_t row = first + u * step;
        Vec16<T> out;
#pragma unroll
        for (int i = 0; i < N; i++) {
          const float v = p.residual ? fmaf(p.scale, to_f32(t[u][i]), to_f32(r[u][i])) : p.scale * to_f32(t[u][i]);
          out.v[i] = at[u] != kNoRun ? from_f32<T>(v) : p.residual ? r[u][i] : (T)0.0f;
        }
        store_piece<kWhole>(static_cast<T*>(p.y) + row * D + c, out, row < p.rows ? D - c : 0);
      }
    }
  }
}

// ---- gradient: positions sorted by id ----

__device__ __forceinline__ uint32_t key_of(int64_t id, int64_t table_rows) { return (uint32_t)(id >= 0 && id < table_rows ? id : table_rows); }

// Zeros, by thread `first` of `step`.
__device__ __forceinline__ void fill_zero(uint8_t* to, int64_t bytes, int64_t first, int64_t step) {
  const int64_t whole = bytes / 16;
  for (int64_t i = first; i < whole; i += step) store_whole(to + i * 16, make_uint4(0, 0, 0, 0));
  for (int64_t i = whole * 16 + first; i < bytes; i += step) to[i] = 0;
}

// The keys to sort, ids outside the table last, and a table of zeros.
template <typename I>
__global__ __launch_bounds__(kThreads) void embedding_keys_kernel(const I* ids, int64_t rows, int64_t table_rows, uint32_t* keys,
                                                                  uint8_t* zero, int64_t zero_bytes) {
  const int64_t step = (int64_t)gridDim.x * kThreads, first = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  for (int64_t i = first; i < rows; i += step) keys[i] = key_of(ids[i], table_rows);
  fill_zero(zero, zero_bytes, first, step);
}

// Sorted at once: a position's place is the number of keys before its own.  A
// workgroup takes kRanked positions and compares each with all keys, kThreads /
// kRanked threads a position.  N^2 comparisons, spread over the chip: 8192
// positions take less time than the launches of a radix sort, and the
// workgroups behind the last position's clear the table meanwhile.  us of a
// gradient so and with the radix sort: 8192 x 2048 of 32,000 ids 50 and 58, 8192
// x 64 of 5000 30 and 38, 1000 x 512 of 32,000 20 and 40.
constexpr int64_t kMostRanked = 8192;
constexpr int kRanked = 16;
template <typename I>
__global__ __launch_bounds__(kThreads) void embedding_rank_kernel(const I* ids, int rows, int64_t table_rows, uint32_t* sorted, uint32_t* index,
                                                                  uint8_t* zero, int64_t zero_bytes) {
  constexpr int kSlices = kThreads / kRanked;
  __shared__ uint4 keys[kMostRanked / 4];
  __shared__ int counts[kSlices][kRanked];
  const int ranking = (rows + kRanked - 1) / kRanked;
  if ((int)blockIdx.x >= ranking) {
    fill_zero(zero, zero_bytes, (int64_t)(blockIdx.x - ranking) * kThreads + threadIdx.x, (int64_t)(gridDim.x - ranking) * kThreads);
    return;
  }
  const int pieces = (rows + 3) / 4;
  for (int first = 0; first < pieces * 4; first += 8 * kThreads) {   // to LDS, eight loads in flight
    uint32_t v[8];
#pragma unroll
    for (int u = 0; u < 8; u++) {
      const int i = first + u * kThreads + threadIdx.x;
      v[u] = i < rows ? key_of(ids[i], table_rows) : kNoRun;
    }
#pragma unroll
    for (int u = 0; u < 8; u++) {
      const int i = first + u * kThreads + threadIdx.x;
      if (i < pieces * 4) reinterpret_cast<uint32_t*>(keys)[i] = v[u];
    }
  }
  __syncthreads();
  const int t = threadIdx.x % kRanked, slice = threadIdx.x / kRanked, first = blockIdx.x * kRanked, mine = first + t;
  const int per = (pieces + kSlices - 1) / kSlices | 1;   // pieces of 4 keys; odd, so the slices of a wave fall on different banks
  const int begin = slice * per, end = begin + per < pieces ? begin + per : pieces;
  const uint32_t key = mine < rows ? reinterpret_cast<const uint32_t*>(keys)[mine] : 0;
  int count = 0;
#pragma unroll 8
  for (int j = begin; j < end; j++) {
    const uint32_t least = j * 4 < first ? key + 1 : key;   // equal keys before these positions count too
    count += (keys[j].x < least) + (keys[j].y < least) + (keys[j].z < least) + (keys[j].w < least);
  }
  if (slice == 0)
    for (int j = first; j < mine; j++) count += reinterpret_cast<const uint32_t*>(keys)[j] == key;
  counts[slice][t] = count;
  __syncthreads();
  if (slice == 0 && mine < rows) {
    int place = 0;
#pragma unroll
    for (int s = 0; s < kSlices; s++) place += counts[s][t];
    sorted[place] = key;
    index[place] = (uint32_t)mine;
  }
}

template <typename T>
struct Runs {
  const T* dy;
  const uint32_t* keys;     // sorted; both readable to the end of a batch past n
  const uint32_t* index;    // the row of dy of a sorted position
  int64_t n, chunks;
  int chunk, cols;          // positions a chunk, a multiple of kBatch
  int64_t table_rows;
  float scale;
  T* dtable;
  float* part;              // [chunks][2][cols]
  uint32_t* part_keys;      // [chunks][2]
};
constexpr int kBatch = 16;   // rows in flight

// A group of `lanes` lanes takes chunk blockIdx.x * (groups of a workgroup) +
// its own, and columns from blockIdx.y * lanes * N on.
template <typename T, bool kWhole>
__global__ __launch_bounds__(kThreads) void embedding_runs_kernel(Runs<T> p, int lanes) {
  constexpr int N = Vec16<T>::kN;
  const int lane = threadIdx.x & (lanes - 1);
  const int64_t chunk = (int64_t)blockIdx.x * (kThreads / lanes) + threadIdx.x / lanes;
  if (chunk >= p.chunks) return;
  const int64_t begin = chunk * p.chunk, end = begin + p.chunk < p.n ? begin + p.chunk : p.n;
  const int c = (blockIdx.y * lanes + lane) * N, left = p.cols - c;
  const uint32_t previous = begin > 0 ? p.keys[begin - 1] : kNoRun, following = end < p.n ? p.keys[end] : kNoRun, last = p.keys[end - 1];
  uint32_t run = p.keys[begin];
  const bool before = previous == run, after = following == last;
  bool is_first = true;
  uint32_t slot0 = kNoRun, slot1 = kNoRun;
  float acc[N];
#pragma unroll
  for (int i = 0; i < N; i++) acc[i] = 0.0f;
  auto flush = [&](bool is_last) {
    if (run >= p.table_rows) return;   // of no id
    const bool to_first = is_first && before, to_last = is_last && after;
    if (to_first || to_last) {
      float* at = p.part + (2 * chunk + (to_first ? 0 : 1)) * p.cols + c;
#pragma unroll
      for (int i = 0; i < N; i++)
        if (i < left) at[i] = acc[i];
      if (to_first) slot0 = run;
      if (to_last) slot1 = to_first ? run | kNoRow : run;
    } else {
#pragma unroll
      for (int i = 0; i < N; i++) acc[i] *= p.scale;
      store_vec<T>(p.dtable + (int64_t)run * p.cols + c, acc, left);
    }
  };
  for (int64_t k = begin; k < end; k += kBatch) {
    uint32_t key[kBatch], row[kBatch];
    __builtin_memcpy(key, p.keys + k, sizeof(key));
    __builtin_memcpy(row, p.index + k, sizeof(row));
    Words16<T> v[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; u++) {
      const bool has = k + u < end && key[u] < p.table_rows;
      v[u] = load_words<kWhole>(p.dy + (int64_t)(has ? row[u] : 0) * p.cols + c, has ? left : 0);
    }
#pragma unroll
    for (int u = 0; u < kBatch; u++) {
      if (k + u < end && key[u] != run) {
        flush(false);
        is_first = false;
        run = key[u];
#pragma unroll
        for (int i = 0; i < N; i++) acc[i] = 0.0f;
      }
#pragma unroll
      for (int i = 0; i < N; i++) acc[i] += to_f32(v[u][i]);
    }
  }
  flush(true);
  if (lane == 0 && blockIdx.y == 0) {
    p.part_keys[2 * chunk] = slot0;
    p.part_keys[2 * chunk + 1] = slot1;
  }
}

// The runs that pass the end of a chunk: the second slot of the chunk that a
// run begins in, then the first of each that it passes or ends in.  A
// workgroup takes every gridDim.x-th chunk, and columns from blockIdx.y *
// lanes * 4 on; the groups of lanes take the partial rows in turn and are
// joined in LDS in their order.
template <typename T>
__global__ __launch_bounds__(kThreads) void embedding_join_kernel(Runs<T> p, int lanes) {
  __shared__ float4 sums[kThreads];
  __shared__ int ends;
  const int lane = threadIdx.x & (lanes - 1), group = threadIdx.x / lanes, groups = kThreads / lanes;
  const int c = (blockIdx.y * lanes + lane) * 4, left = p.cols - c;
  for (int64_t chunk = blockIdx.x; chunk < p.chunks; chunk += gridDim.x) {
    const uint32_t run = p.part_keys[2 * chunk + 1];
    if (run & kNoRow) continue;   // kNoRun, or a run that began before
    int64_t count = 0;            // chunks after this one that the run passes or ends in
    for (bool more = true; more;) {
      __syncthreads();
      if (threadIdx.x == 0) ends = kThreads;
      __syncthreads();
      const int64_t at = chunk + 1 + count + threadIdx.x;
      if (at >= p.chunks || p.part_keys[2 * at + 1] != (run | kNoRow)) atomicMin(&ends, (int)threadIdx.x);
      __syncthreads();
      more = ends == kThreads;
      count += more ? kThreads : ends + 1;
    }
    float4 s = make_float4(0, 0, 0, 0);
    for (int64_t k = group; k <= count; k += groups * 8) {
      float4 v[8];
#pragma unroll
      for (int u = 0; u < 8; u++) {
        const int64_t at = k + u * groups;
        const Vec16<float> t = load_raw(p.part + (2 * (chunk + at) + (at == 0 ? 1 : 0)) * p.cols + c, at <= count ? left : 0);
        v[u] = make_float4(t.v[0], t.v[1], t.v[2], t.v[3]);
      }
#pragma unroll
      for (int u = 0; u < 8; u++) s = make_float4(s.x + v[u].x, s.y + v[u].y, s.z + v[u].z, s.w + v[u].w);
    }
    sums[threadIdx.x] = s;
    __syncthreads();
    if (group == 0) {
      for (int g = 1; g < groups; g++) {
        const float4 v = sums[g * lanes + lane];
        s = make_float4(s.x + v.x, s.y + v.y, s.z + v.z, s.w + v.w);
      }
      T* at = p.dtable + (int64_t)run * p.cols + c;
      const float f[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
      for (int i = 0; i < 4; i++)
        if (i < left) at[i] = from_f32<T>(p.scale * f[i]);
    }
  }
}

int lanes_of(int cols, int values) {
  const int64_t vecs = cdiv(cols, values);
  return vecs >= 64 ? 64 : pow2_at_least(vecs);
}

// Positions a chunk: as many chunks as groups of lanes run at once, but no
// fewer than 16, below which the partial rows cost as much as the rows.
int chunk_of(int64_t n, int cols, int values) {
  const int lanes = lanes_of(cols, values);
  const int64_t at_once = 256 * 16 * (64 / lanes) / cdiv(cols, (int64_t)lanes * values);
  int64_t chunk = kBatch;
  while (chunk < 256 && chunk * at_once < n) chunk *= 2;
  return (int)chunk;
}

// ---- gradient: a small table in the accumulators ----

constexpr int kCountThreads = 512, kCountRows = 256;   // of a workgroup's turn
// Accumulators of 16 x 16 that a wave holds: up to 12 leave room for two
// workgroups a CU, whose loads overlap.
constexpr int kMostCounted = 16, kTwiceCounted = 12;

template <typename T>
struct Counted {
  const T* dy;
  const void* ids;
  bool wide_ids;
  int64_t rows;
  int cols, table_rows;
  float* part;         // [groups][table_rows][cols]
  uint32_t* flags;     // [table_rows][cols] bits: 1 an infinity, 2 a negative one, 4 a NaN
};

// A one is made as float16 for either type, and its bits are 2^-7 as bfloat16.
template <typename T>
constexpr float kOneInverse = 1.0f;
template <>
constexpr float kOneInverse<bf16_t> = 128.0f;
template <typename T>
constexpr uint16_t kInfinity = 0;
template <>
constexpr uint16_t kInfinity<f16_t> = 0x7c00;
template <>
constexpr uint16_t kInfinity<bf16_t> = 0x7f80;

typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

__global__ __launch_bounds__(kThreads) void embedding_clear_kernel(uint32_t* p, int64_t n) {
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < n; i += (int64_t)gridDim.x * kThreads) p[i] = 0;
}

// FD: 16s of columns, a power of two; FV: 16s of ids a wave, every eighth.
// Sums of ids 16 (8 i + wave) + lane % 16 and columns 16 j + 4 (lane / 16) + 0..3.
template <typename T, int FV, int FD>
__global__ __launch_bounds__(kCountThreads, (FD < 8 && FV * FD <= kTwiceCounted ? 4 : 2)) void embedding_count_kernel(Counted<T> p) {
  typedef typename Mma<T>::Frag Frag;
  constexpr int R = FD * 16, kVecs = R / 8, kLoads = kCountRows * kVecs / kCountThreads;   // pieces of 16 bytes
  __shared__ __attribute__((aligned(16))) uint8_t tile[2][kCountRows * R * 2];
  __shared__ __attribute__((aligned(16))) _Float16 keys[2][kCountRows];
  const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4, wave = wave_id();
  const int64_t step = (int64_t)gridDim.x * kCountRows;
  Words16<T> next[kLoads];
  _Float16 next_key = 0;   // at most 2048 ids: exact
  auto load = [&](int64_t turn) {
#pragma unroll
    for (int i = 0; i < kLoads; i++) {
      const int at = i * kCountThreads + threadIdx.x, row = at / kVecs, c = (at % kVecs) * 8;
      next[i] = load_words<false>(p.dy + (turn + row) * p.cols + c, turn + row < p.rows ? p.cols - c : 0);
    }
    if (threadIdx.x < kCountRows) {
      const int64_t row = turn + threadIdx.x;
      int64_t id = -1;
      if (row < p.rows) id = p.wide_ids ? static_cast<const int64_t*>(p.ids)[row] : static_cast<const int32_t*>(p.ids)[row];
      next_key = id >= 0 && id < p.table_rows ? (_Float16)(int)id : (_Float16)-1;
    }
  };
  auto stage = [&](int buf, int64_t turn) {
#pragma unroll
    for (int i = 0; i < kLoads; i++) {
      const int at = i * kCountThreads + threadIdx.x, row = at / kVecs, v = at % kVecs;
      u16x2 most = {0, 0};
#pragma unroll
      for (int k = 0; k < 4; k++) most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2, next[i].w[k] & 0x7fff7fffu));
      if (most[0] >= kInfinity<T> || most[1] >= kInfinity<T>) {   // taken out, and remembered for its id
        int64_t id = -1;
        if (turn + row < p.rows) id = p.wide_ids ? static_cast<const int64_t*>(p.ids)[turn + row] : static_cast<const int32_t*>(p.ids)[turn + row];
        const bool has = id >= 0 && id < p.table_rows;
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const uint16_t b = (uint16_t)(next[i].w[e / 2] >> (e % 2 * 16));
          if ((b & 0x7fff) < kInfinity<T>) continue;
          if (has) atomicOr(&p.flags[id * p.cols + v * 8 + e], (b & 0x7fff) > kInfinity<T> ? 4u : b >> 15 ? 2u : 1u);
          next[i].w[e / 2] &= e % 2 ? 0xffffu : 0xffff0000u;
        }
      }
      const int unit = (v >> 1) ^ unit_swizzle<T, R>(row);
      *reinterpret_cast<uint4*>(&tile[buf][row * R * 2 + (unit << 5) + (v & 1) * 16]) = __builtin_bit_cast(uint4, next[i]);
    }
    if (threadIdx.x < kCountRows) keys[buf][threadIdx.x] = next_key;
  };
  f32x4 acc[FV][FD] = {};
  const int base = fragment_base<T, false, R>(0);
  const int frags = (p.table_rows + 15) / 16;
  const int64_t first = (int64_t)blockIdx.x * kCountRows;
  load(first);
  stage(0, first);
  int buf = 0;
  for (int64_t turn = first; turn < p.rows; turn += step, buf ^= 1) {
    load(turn + step);
    __syncthreads();   // this turn's rows are in LDS, the other buffer is all read
#pragma unroll 2
    for (int kb = 0; kb < kCountRows / 32; kb++) {
      const uint4 k = *reinterpret_cast<const uint4*>(&keys[buf][kb * 32 + q * 8]);
      const uint32_t words[4] = {k.x, k.y, k.z, k.w};
      f16x2 mine[4];   // an id's distance from this lane's first
#pragma unroll
      for (int e = 0; e < 4; e++) mine[e] = __builtin_bit_cast(f16x2, words[e]) - (_Float16)(wave * 16 + r);
      Frag b[FD];
#pragma unroll
      for (int j = 0; j < FD; j++) b[j] = fragment<T, false, R>(tile[buf], base, j, kb);
#pragma unroll
      for (int i = 0; i < FV; i++) {
        if (i == FV - 1 && i * 8 + wave >= frags) break;   // no branch before the last: it would part the products
        uint32_t ones[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const f16x2 off = mine[e] - (_Float16)(i * 128);   // a whole number: 1 - off^2 is 1 or not above 0
          const f16x2 one = __builtin_elementwise_fma(off, -off, f16x2{1, 1});
          ones[e] = __builtin_bit_cast(uint32_t, __builtin_elementwise_min(__builtin_elementwise_max(one, f16x2{0, 0}), f16x2{1, 1}));
        }
        const Frag a = __builtin_bit_cast(Frag, make_uint4(ones[0], ones[1], ones[2], ones[3]));
#pragma unroll
        for (int j = 0; j < FD; j++) acc[i][j] = Mma<T>::run(b[j], a, acc[i][j]);
      }
    }
    if (turn + step < p.rows) stage(buf ^ 1, turn + step);
  }
  float* const part = p.part + (int64_t)blockIdx.x * p.table_rows * p.cols;
#pragma unroll
  for (int i = 0; i < FV; i++) {
    const int id = (i * 8 + wave) * 16 + r;
    if (id >= p.table_rows) continue;
#pragma unroll
    for (int j = 0; j < FD; j++) {
      const int c = j * 16 + q * 4;
#pragma unroll
      for (int e = 0; e < 4; e++)
        if (c + e < p.cols) part[(int64_t)id * p.cols + c + e] = acc[i][j][e] * kOneInverse<T>;
    }
  }
}

// dtable from the workgroups' sums: 32 columns a workgroup, 32 slices of the
// workgroups, joined in LDS in their order; then what was taken out.
template <typename T>
__global__ __launch_bounds__(1024) void embedding_sum_kernel(const float* part, int n, int64_t size, float scale, const uint32_t* flags, T* dtable) {
  __shared__ float lds[32][33];
  const int64_t col = (int64_t)blockIdx.x * 32 + (threadIdx.x & 31);
  const int slice = threadIdx.x >> 5;
  float s = 0.0f;
  if (col < size) {
    int k = slice;
    for (; k + 3 * 32 < n; k += 4 * 32) {   // four loads in flight
      float v[4];
#pragma unroll
      for (int i = 0; i < 4; i++) v[i] = part[(k + i * 32) * size + col];
#pragma unroll
      for (int i = 0; i < 4; i++) s += v[i];
    }
    for (; k < n; k += 32) s += part[k * size + col];
  }
  lds[slice][threadIdx.x & 31] = s;
  __syncthreads();
  if (slice == 0 && col < size) {
    float t = 0.0f;
#pragma unroll
    for (int k = 0; k < 32; k++) t += lds[k][threadIdx.x];
    const uint32_t f = flags[col];
    if (f) t = f >= 3 ? __builtin_nanf("") : f == 1 ? __builtin_inff() : -__builtin_inff();
    dtable[col] = from_f32<T>(scale * t);
  }
}

int column_frags(int cols) { return pow2_at_least(cdiv(cols, 16)); }

// Whether the table's sums are made in accumulators.  us, so and sorted, for
// bf16 rows: 1,702,400 x 64 of 16 ids 50 and 97, of 300 (12 accumulators) 95
// and 124, of 1000 (32) 214 and 126; 1,702,400 x 128 of 100 (8) 124 and 143, of
// 380 (24) 180 and 181; 65,536 x 64 of 300 29 and 42; 2000 x 64 of 300 19 and 23,
// of 1000 43 and 23.
bool counted(int64_t rows, int cols, int64_t table_rows, int dtype) {
  if (dtype == NEST_DTYPE_F32 || cols > 128) return false;
  return cdiv(table_rows, 16 * 8) * column_frags(cols) <= kMostCounted;
}

struct Plan {
  bool counted, ranked;
  int64_t groups;                                    // counted: workgroups
  size_t flags;
  size_t keys, sorted, index, sort, part, part_keys, bytes;
  int chunk;
  int64_t chunks;
};
Plan plan_of(int64_t rows, int cols, int64_t table_rows, int dtype) {
  Plan l{};
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t o = at;
    at += align256(bytes);
    return o;
  };
  l.counted = counted(rows, cols, table_rows, dtype);
  if (l.counted) {
    const int64_t turns = cdiv(rows, kCountRows);
    const int64_t at_once = cols <= 64 && cdiv(table_rows, 16 * 8) * column_frags(cols) <= kTwiceCounted ? 512 : 256;
    l.groups = turns < at_once ? turns : at_once;
    l.flags = take((size_t)table_rows * cols * 4);
    l.part = take((size_t)l.groups * table_rows * cols * 4);
    l.bytes = at;
    return l;
  }
  l.ranked = rows <= kMostRanked;
  l.chunk = chunk_of(rows, cols, dtype == NEST_DTYPE_F32 ? 4 : 8);
  l.chunks = cdiv(rows, l.chunk);
  if (!l.ranked) {
    l.keys = take((size_t)rows * 4);
    l.sort = take(index_sort_ws_bytes(rows));
  }
  l.sorted = take((size_t)(rows + kBatch) * 4);
  l.index = take((size_t)(rows + kBatch) * 4);
  l.part = take((size_t)l.chunks * 2 * cols * 4);
  l.part_keys = take((size_t)l.chunks * 2 * 4);
  l.bytes = at;
  return l;
}

// f with whether rows are whole vectors as a constant.
template <typename F>
void with_whole(bool whole, F f) {
  if (whole) f(Number<1>());
  else f(Number<0>());
}

template <typename T>
hipError_t lookup(const EmbeddingParams& p, hipStream_t s) {
  // As many workgroups as run at once, the columns split where rows are few (18
  // rows of 7771: 48 us unsplit).
  const int lanes = lanes_of(p.cols, Vec16<T>::kN);
  const int64_t need = cdiv(p.rows, kThreads / lanes), x = need < 1024 ? need : 1024, pieces = cdiv(p.cols, (int64_t)lanes * Vec16<T>::kN);
  const dim3 grid((unsigned)x, (unsigned)(pieces < 1024 / x ? pieces : 1024 / x));
  with_whole(p.cols % Vec16<T>::kN == 0, [&](auto whole) {
    if (p.wide_ids) embedding_kernel<T, int64_t, whole.value><<<grid, kThreads, 0, s>>>(p, lanes);
    else embedding_kernel<T, int32_t, whole.value><<<grid, kThreads, 0, s>>>(p, lanes);
  });
  return hipGetLastError();
}

template <typename T>
hipError_t count_gradient(const EmbeddingParams& p, const Plan& l, hipStream_t s) {
  uint8_t* ws = static_cast<uint8_t*>(p.ws);
  const int64_t size = p.table_rows * p.cols;
  const Counted<T> q{static_cast<const T*>(p.dy), p.ids, p.wide_ids, p.rows, p.cols, (int)p.table_rows, reinterpret_cast<float*>(ws + l.part),
                     reinterpret_cast<uint32_t*>(ws + l.flags)};
  embedding_clear_kernel<<<(unsigned)cdiv(size, kThreads), kThreads, 0, s>>>(q.flags, size);
  auto launch = [&](auto fd) {
    constexpr int FD = fd.value, kMost = kMostCounted / FD;
    const int need = (int)cdiv(p.table_rows, 16 * 8);
    auto with = [&](auto fv) { embedding_count_kernel<T, fv.value, FD><<<(unsigned)l.groups, kCountThreads, 0, s>>>(q); };
    if constexpr (FD == 8) {
      if (need == 1) with(Number<1>());
      else with(Number<2>());
    } else {
      if (need * 4 <= kMost) with(Number<kMost / 4>());
      else if (need * 2 <= kMost) with(Number<kMost / 2>());
      else if (need * 4 <= kMost * 3) with(Number<kMost * 3 / 4>());
      else with(Number<kMost>());
    }
  };
  const int fd = column_frags(p.cols);
  if (fd == 1) launch(Number<1>());
  else if (fd == 2) launch(Number<2>());
  else if (fd == 4) launch(Number<4>());
  else launch(Number<8>());
  if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  embedding_sum_kernel<T><<<(unsigned)cdiv(size, 32), 1024, 0, s>>>(q.part, (int)l.groups, size, p.scale, q.flags, static_cast<T*>(p.dtable));
  return hipGetLastError();
}

template <typename T, typename I>
hipError_t sort_ids(const EmbeddingParams& p, const Plan& l, uint32_t* sorted, uint32_t* index, hipStream_t s) {
  uint8_t *ws = static_cast<uint8_t*>(p.ws), *table = static_cast<uint8_t*>(p.dtable);
  const I* ids = static_cast<const I*>(p.ids);
  const int64_t bytes = p.table_rows * p.cols * (int64_t)sizeof(T), pieces = cdiv(bytes, 16 * kThreads);
  if (l.ranked) {
    const int64_t clearing = pieces < 512 ? pieces : 512;   // two a CU, beside as many that rank
    embedding_rank_kernel<I><<<(unsigned)(cdiv(p.rows, kRanked) + clearing), kThreads, 0, s>>>(ids, (int)p.rows, p.table_rows, sorted, index, table, bytes);
    return hipGetLastError();
  }
  uint32_t* keys = reinterpret_cast<uint32_t*>(ws + l.keys);
  const int64_t need = cdiv(p.rows, kThreads) > pieces ? cdiv(p.rows, kThreads) : pieces;
  embedding_keys_kernel<I><<<(unsigned)(need < 8192 ? need : 8192), kThreads, 0, s>>>(ids, p.rows, p.table_rows, keys, table, bytes);
  if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  int bits = 1;
  while (((int64_t)1 << bits) <= p.table_rows) bits++;
  return launch_sort_indices(keys, sorted, index, p.rows, bits, ws + l.sort, s);
}

template <typename T>
hipError_t gradient(const EmbeddingParams& p, hipStream_t s) {
  if (p.rows == 0) {
    const int64_t bytes = p.table_rows * p.cols * (int64_t)sizeof(T), pieces = cdiv(bytes, 16 * kThreads);
    embedding_keys_kernel<int32_t><<<(unsigned)(pieces < 8192 ? pieces : 8192), kThreads, 0, s>>>(nullptr, 0, p.table_rows, nullptr,
                                                                                                 static_cast<uint8_t*>(p.dtable), bytes);
    return hipGetLastError();
  }
  const Plan l = plan_of(p.rows, p.cols, p.table_rows, p.dtype);
  if constexpr (sizeof(T) == 2)
    if (l.counted) return count_gradient<T>(p, l, s);
  uint8_t* ws = static_cast<uint8_t*>(p.ws);
  uint32_t *sorted = reinterpret_cast<uint32_t*>(ws + l.sorted), *index = reinterpret_cast<uint32_t*>(ws + l.index);
  hipError_t e = p.wide_ids ? sort_ids<T, int64_t>(p, l, sorted, index, s) : sort_ids<T, int32_t>(p, l, sorted, index, s);
  if (e != hipSuccess) return e;
  const Runs<T> q{static_cast<const T*>(p.dy), sorted, index, p.rows, l.chunks, l.chunk, p.cols, p.table_rows, p.scale, static_cast<T*>(p.dtable),
                  reinterpret_cast<float*>(ws + l.part), reinterpret_cast<uint32_t*>(ws + l.part_keys)};
  constexpr int N = Vec16<T>::kN;
  const int lanes = lanes_of(p.cols, N);
  with_whole(p.cols % N == 0, [&](auto whole) {
    embedding_runs_kernel<T, whole.value><<<dim3((unsigned)cdiv(l.chunks, kThreads / lanes), (unsigned)cdiv(p.cols, (int64_t)lanes * N)), kThreads, 0, s>>>(
        q, lanes);
  });
  if (l.chunks > 1) {
    int wide = 1;   // lanes of a partial row: up to a workgroup
    while (wide < kThreads && wide * 4 < p.cols) wide *= 2;
    const unsigned grid = (unsigned)(l.chunks - 1 < 2048 ? l.chunks - 1 : 2048);
    embedding_join_kernel<T><<<dim3(grid, (unsigned)cdiv(p.cols, (int64_t)wide * 4)), kThreads, 0, s>>>(q, wide);
  }
  return hipGetLastError();
}

}  // namespace

size_t embedding_ws_bytes(int64_t rows, int cols, int64_t table_rows, int dtype) { return rows > 0 ? plan_of(rows, cols, table_rows, dtype).bytes : 0; }

hipError_t launch_embedding(const EmbeddingParams& p, hipStream_t s) {
  if (p.dtype == NEST_DTYPE_F32) return lookup<float>(p, s);
  return p.dtype == NEST_DTYPE_F16 ? lookup<f16_t>(p, s) : lookup<bf16_t>(p, s);
}
hipError_t launch_embedding_backward(const EmbeddingParams& p, hipStream_t s) {
  if (p.dtype == NEST_DTYPE_F32) return gradient<float>(p, s);
  return p.dtype == NEST_DTYPE_F16 ? gradient<f16_t>(p, s) : gradient<bf16_t>(p, s);
}

}  // namespace nest
