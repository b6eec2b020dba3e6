// Embedding lookup with a scale, and the gradient of its table.
//
//   y_i = residual_i + scale table[id_i],  dtable[v] = scale sum over id_i = v of dy_i
//
// An id outside the table adds nothing and has no gradient.
//
// Memory bound.  The lookup reads whole rows in 16-byte pieces, four rows a
// lane in flight.  The gradient sorts the positions by their ids (stable, so
// in the order of the positions) and sums runs of equal ids in float32,
// without atomics: a group of lanes takes a chunk of the sorted positions,
// writes the runs that lie inside its chunk and hands on a partial row for a
// run that began before it or goes on after it, at most two a chunk.  The
// partial rows are in sorted order too, and the same kernel sums them, level
// after level, until one chunk is left.  The sums' order depends on ids and
// sizes alone, so results repeat bit for bit.
#include "nest_internal.h"
#include "residual_internal.h"
#include "vec_io.h"

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

template <typename T, typename I>
__global__ __launch_bounds__(kThreads) void embedding_kernel(EmbeddingParams p, int lanes) {
  constexpr int N = Vec16<T>::kN, U = kRowsInFlight;
  const int lane = threadIdx.x & (lanes - 1), rows_wg = kThreads / lanes;
  const int64_t step = (int64_t)gridDim.x * rows_wg;
  const int D = p.cols;
  for (int64_t first = (int64_t)blockIdx.x * rows_wg + threadIdx.x / lanes; first < p.rows; first += step * U) {
    int64_t at[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int64_t row = first + u * step;
      const int64_t id = row < p.rows ? (int64_t)static_cast<const I*>(p.ids)[row] : -1;
      at[u] = id >= 0 && id < p.table_rows ? id * D : -1;
    }
    for (int c = lane * N; c < D; c += lanes * N) {
      Vec16<T> t[U], r[U];
#pragma unroll
      for (int u = 0; u < U; u++) {
        const int64_t row = first + u * step;
        t[u] = load_raw(static_cast<const T*>(p.table) + at[u] + c, at[u] >= 0 ? D - c : 0);
        if (p.residual) r[u] = load_raw(static_cast<const T*>(p.residual) + row * D + c, row < p.rows ? D - c : 0);
      }
#pragma unroll
      for (int u = 0; u < U; u++) {
        const int64_t row = first + u * step;
        Vec16<T> out;
#pragma unroll
        for (int i = 0; i < N; i++) {
          const float v = p.scale * to_f32(t[u].v[i]);
          out.v[i] = at[u] < 0 ? (p.residual ? r[u].v[i] : (T)0.0f)
                               : from_f32<T>(p.residual ? fmaf(p.scale, to_f32(t[u].v[i]), to_f32(r[u].v[i])) : v);
        }
        store_raw(static_cast<T*>(p.y) + row * D + c, out, row < p.rows ? D - c : 0);
      }
    }
  }
}

// ---- gradient ----

// The keys to sort, ids outside the table last, and a table of zeros.
template <typename I>
__global__ __launch_bounds__(kThreads) void embedding_keys_kernel(const I* ids, int64_t rows, int64_t table_rows, uint32_t* keys,
                                                                  uint8_t* zero, int64_t zero_bytes) {
  const int64_t step = (int64_t)gridDim.x * kThreads, first = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  for (int64_t i = first; i < rows; i += step) {
    const int64_t id = ids[i];
    keys[i] = (uint32_t)(id >= 0 && id < table_rows ? id : table_rows);
  }
  const int64_t whole = zero_bytes / 16;
  for (int64_t i = first; i < whole; i += step) {
    const uint4 z = make_uint4(0, 0, 0, 0);
    __builtin_memcpy(zero + i * 16, &z, 16);
  }
  for (int64_t i = whole * 16 + first; i < zero_bytes; i += step) zero[i] = 0;
}

template <typename S>
struct RunRows {
  const S* rows;            // of dy, or partial rows
  const uint32_t* keys;     // sorted
  const uint32_t* index;    // the row of dy of a sorted position; null: the position itself
  int64_t n;                // positions
  int chunk;
  int cols;
  int64_t table_rows;
  float scale;
  void* dtable;
  float* part;              // [2 chunks][cols]
  uint32_t* part_keys;
};

// A group of `lanes` lanes takes chunk blockIdx.x * (groups of a workgroup) +
// its own, and columns from blockIdx.y * lanes * N on.
template <typename S, typename T>
__global__ __launch_bounds__(kThreads) void embedding_runs_kernel(RunRows<S> p, int lanes) {
  constexpr int N = Vec16<S>::kN, U = 8;
  const int lane = threadIdx.x & (lanes - 1);
  const int64_t chunk = (int64_t)blockIdx.x * (kThreads / lanes) + threadIdx.x / lanes;
  const int64_t begin = chunk * p.chunk, end = begin + p.chunk < p.n ? begin + p.chunk : p.n;
  if (begin >= p.n) return;
  const int c = (blockIdx.y * lanes + lane) * N, left = p.cols - c;
  const bool speaks = lane == 0 && blockIdx.y == 0;
  auto run_of = [](uint32_t key) { return key == kNoRun ? key : key & ~kNoRow; };
  uint32_t run = run_of(p.keys[begin]);
  const bool before = begin > 0 && run_of(p.keys[begin - 1]) == run && run != kNoRun;
  const uint32_t last = run_of(p.keys[end - 1]);
  const bool after = end < p.n && run_of(p.keys[end]) == last && last != kNoRun;
  bool is_first = true;
  uint32_t slot[2] = {kNoRun, kNoRun};
  float acc[N];
#pragma unroll
  for (int i = 0; i < N; i++) acc[i] = 0.0f;
  auto flush = [&](bool is_last) {
    if (run >= p.table_rows) return;   // of no id, or no run
    const bool to_first = is_first && before, to_last = is_last && after;
    if (to_first || to_last) {
      float* at = p.part + (2 * chunk + (to_first ? 0 : 1)) * p.cols + c;
#pragma unroll
      for (int i = 0; i < N; i++)
        if (i < left) at[i] = acc[i];
      slot[to_first ? 0 : 1] = run;
      if (to_first && to_last) slot[1] = run | kNoRow;
    } else {
      T* at = static_cast<T*>(p.dtable) + (int64_t)run * p.cols + c;
#pragma unroll
      for (int i = 0; i < N; i++)
        if (i < left) at[i] = from_f32<T>(p.scale * acc[i]);
    }
  };
  for (int64_t k = begin; k < end; k += U) {
    uint32_t key[U];
    Vec16<S> v[U];
#pragma unroll
    for (int u = 0; u < U; u++) key[u] = k + u < end ? p.keys[k + u] : kNoRun;
#pragma unroll
    for (int u = 0; u < U; u++) {
      const bool has = key[u] < p.table_rows;   // neither kNoRun, nor kNoRow, nor of no id
      const int64_t row = !has ? 0 : p.index ? (int64_t)p.index[k + u] : k + u;
      v[u] = load_raw(p.rows + row * p.cols + c, has ? left : 0);
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
      if (k + u >= end) break;
      const uint32_t r = run_of(key[u]);
      if (r != run) {
        flush(false);
        is_first = false;
        run = r;
#pragma unroll
        for (int i = 0; i < N; i++) acc[i] = 0.0f;
      }
#pragma unroll
      for (int i = 0; i < N; i++) acc[i] += to_f32(v[u].v[i]);
    }
  }
  flush(true);
  if (speaks && p.part_keys) {
    p.part_keys[2 * chunk] = slot[0];
    p.part_keys[2 * chunk + 1] = slot[1];
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
  int64_t chunk = 16;
  while (chunk < 256 && chunk * at_once < n) chunk *= 2;
  return (int)chunk;
}
constexpr int kPartChunk = 64;   // partial rows a chunk

struct Plan {
  size_t keys, sorted, index, sort, part[2], part_keys[2], bytes;
  int chunk;
  int64_t chunks;
};
Plan plan_of(int64_t rows, int cols, int dtype) {
  Plan l{};
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t o = at;
    at += align256(bytes);
    return o;
  };
  l.chunk = chunk_of(rows, cols, dtype == NEST_DTYPE_F32 ? 4 : 8);
  l.chunks = cdiv(rows, l.chunk);
  l.keys = take((size_t)rows * 4);
  l.sorted = take((size_t)rows * 4);
  l.index = take((size_t)rows * 4);
  l.sort = take(index_sort_ws_bytes(rows > 0 ? rows : 1));
  int64_t entries = 2 * l.chunks;
  for (int i = 0; i < 2; i++) {   // the levels take turns
    l.part[i] = take((size_t)entries * cols * 4);
    l.part_keys[i] = take((size_t)entries * 4);
    entries = 2 * cdiv(entries, kPartChunk);
  }
  l.bytes = at;
  return l;
}

template <typename S, typename T>
hipError_t launch_runs(const RunRows<S>& p, hipStream_t s) {
  const int N = Vec16<S>::kN, lanes = lanes_of(p.cols, N);
  const dim3 grid((unsigned)cdiv(cdiv(p.n, p.chunk), kThreads / lanes), (unsigned)cdiv(p.cols, (int64_t)lanes * N));
  embedding_runs_kernel<S, T><<<grid, kThreads, 0, s>>>(p, lanes);
  return hipGetLastError();
}

template <typename T>
hipError_t lookup(const EmbeddingParams& p, hipStream_t s) {
  const int lanes = lanes_of(p.cols, Vec16<T>::kN);
  const int64_t need = cdiv(p.rows, (int64_t)(kThreads / lanes) * kRowsInFlight);
  const unsigned grid = (unsigned)(need < 8192 ? need : 8192);
  if (p.wide_ids) embedding_kernel<T, int64_t><<<grid, kThreads, 0, s>>>(p, lanes);
  else embedding_kernel<T, int32_t><<<grid, kThreads, 0, s>>>(p, lanes);
  return hipGetLastError();
}

template <typename T>
hipError_t gradient(const EmbeddingParams& p, hipStream_t s) {
  const Plan l = plan_of(p.rows, p.cols, p.dtype);
  uint8_t* ws = static_cast<uint8_t*>(p.ws);
  uint32_t *keys = reinterpret_cast<uint32_t*>(ws + l.keys), *sorted = reinterpret_cast<uint32_t*>(ws + l.sorted),
           *index = reinterpret_cast<uint32_t*>(ws + l.index);
  const int64_t bytes = p.table_rows * p.cols * (int64_t)sizeof(T);
  const int64_t need = cdiv(bytes / 16 > p.rows ? bytes / 16 : p.rows, kThreads);
  const unsigned grid = (unsigned)(need < 1 ? 1 : need < 8192 ? need : 8192);
  uint8_t* table = static_cast<uint8_t*>(p.dtable);
  if (p.wide_ids) embedding_keys_kernel<<<grid, kThreads, 0, s>>>(static_cast<const int64_t*>(p.ids), p.rows, p.table_rows, keys, table, bytes);
  else embedding_keys_kernel<<<grid, kThreads, 0, s>>>(static_cast<const int32_t*>(p.ids), p.rows, p.table_rows, keys, table, bytes);
  if (hipError_t e = hipGetLastError(); e != hipSuccess || p.rows == 0) return e;
  int bits = 1;
  while (((int64_t)1 << bits) <= p.table_rows) bits++;
  if (hipError_t e = launch_sort_indices(keys, sorted, index, p.rows, bits, ws + l.sort, s); e != hipSuccess) return e;
  auto part = [&](int i) { return reinterpret_cast<float*>(ws + l.part[i]); };
  auto part_keys = [&](int i) { return reinterpret_cast<uint32_t*>(ws + l.part_keys[i]); };
  const RunRows<T> first{static_cast<const T*>(p.dy), sorted, index, p.rows, l.chunk, p.cols, p.table_rows, p.scale, p.dtable, part(0),
                         part_keys(0)};
  if (hipError_t e = launch_runs<T, T>(first, s); e != hipSuccess) return e;
  int64_t chunks = l.chunks;
  for (int from = 0; chunks > 1; from ^= 1) {
    const RunRows<float> next{part(from), part_keys(from), nullptr, 2 * chunks, kPartChunk, p.cols, p.table_rows, p.scale, p.dtable,
                              part(from ^ 1), part_keys(from ^ 1)};
    if (hipError_t e = launch_runs<float, T>(next, s); e != hipSuccess) return e;
    chunks = cdiv(2 * chunks, kPartChunk);
  }
  return hipSuccess;
}

}  // namespace

size_t embedding_ws_bytes(int64_t rows, int cols, int64_t, int dtype) { return plan_of(rows, cols, dtype).bytes; }

hipError_t launch_embedding(const EmbeddingParams& p, hipStream_t s) {
  if (p.dtype == NEST_DTYPE_F32) return lookup<float>(p, s);
  return p.dtype == NEST_DTYPE_F16 ? lookup<f16_t>(p, s) : lookup<bf16_t>(p, s);
}
hipError_t launch_embedding_backward(const EmbeddingParams& p, hipStream_t s) {
  if (p.dtype == NEST_DTYPE_F32) return gradient<float>(p, s);
  return p.dtype == NEST_DTYPE_F16 ? gradient<f16_t>(p, s) : gradient<bf16_t>(p, s);
}

}  // namespace nest
