// Matrix products on MFMA with operands staged by direct loads into LDS: the
// tiles behind gated_ffn.
//
//   C[m][n] = sum_k A(m, k) B(n, k),  float32 sums
//
// 16-bit operands multiply on v_mfma_f32_16x16x32; float32 ones as three
// bfloat16 parts each on the same instruction (split, run_parts), which passes
// the rate of the float32 instructions.  An infinity has no such parts: the
// float32 results that it enters are NaN.
//
// An operand is stored with k contiguous ("kKM", rows of m or n) or with its
// own index contiguous (rows of k); every row length is a multiple of 16
// bytes.  A step takes 128 bytes of k (64 16-bit or 32 float32 values) of each
// row.  Two or four LDS buffers: the loads of the next one or three steps are in
// flight while the current one is multiplied, one barrier a step.
//
// LDS layouts.  k contiguous: rows of 128 bytes, the 16-byte chunk c of row r
// at slot c ^ (r & 7), so the 16 rows one fragment load touches fall on
// different banks.  k outermost: rows of R elements, 16-element units permuted
// by the row so that the rows one transposing load touches do too.  The
// permutation is done by the choice of what each lane loads: a direct load
// always writes 64 x 16 consecutive bytes.
//
// Out of range: a lane whose chunk lies outside its operand gives the buffer
// load an offset past the resource's size, which the hardware answers with
// zero.  k past the end is outside in both operands (or a zero of one's row
// padding), so nothing an operand does not hold is multiplied.
//
// Measured: 8192 x 2048 x 8192 bf16 1170 TFLOP/s, 8192 x 2048 x 16384 1260,
// where the library's 8192^3 product reaches 1380 on this card, its second
// operand transposed 1577; the matrix cores are busy 54 to 67% of the cycles, at a clock of 1.7 to 1.9 GHz, without
// LDS bank conflicts; the rest is the barrier and the wait for loads that two
// buffers leave.  float32 4096 x 2048, 4096: 202 TFLOP/s, 155 the library's
// product; that is 1210 of the parts' products, and in 64 x 64 tiles, whose
// fragments are cut four times for four products, the vector ALU is busy 0.64 to
// 0.85 of the cycles and 125 TFLOP/s come out.
#pragma once

#include "vec_io.h"

namespace nest {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));

constexpr int kStepBytes = 128;
constexpr uint32_t kOutside = 0x80000000u, kRecords = 0x7fffffffu;

template <typename T>
struct Mma;
template <>
struct Mma<bf16_t> {
  typedef bf16x8 Frag;
  static __device__ __forceinline__ f32x4 run(Frag a, Frag b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <>
struct Mma<f16_t> {
  typedef f16x8 Frag;
  static __device__ __forceinline__ f32x4 run(Frag a, Frag b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
template <>
struct Mma<float> {
  typedef f32x4 Frag;   // k = 4 (lane / 16) + j in element j: any order that both operands share
  static __device__ __forceinline__ f32x4 run(Frag a, Frag b, f32x4 c) {
#pragma unroll
    for (int j = 0; j < 4; j++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
    return c;
  }
};

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

// Eight float32 values of a lane as three bfloat16 parts each, their sum exact:
// the value to the nearest bfloat16, what is left to the nearest, the rest,
// which has 7 bits (Henry, Tang, Heinecke, "Leveraging the bfloat16 artificial
// intelligence datatype for higher-precision computations", 2019).  The first
// part is clamped to the largest bfloat16: values above it, up to the largest
// float32, would round to an infinity.  To the nearest, the parts are at most
// 2^-8 and 2^-17 of the value and of either sign; cut off instead, they would be
// up to 2^-7 and 2^-15 of it and of its own sign, so that what run_parts leaves
// out, up to 2^-21 of a product, would make every product smaller.  That took
// 248 us for a step of 1777 x 515, 1365 and 2870 for 4096 x 2048, 4096; the
// clamps are two of thirteen operations a pair of values, and it takes 282 and
// 3060.  The parts end at 2^-133, the smallest bfloat16: a value below 2^-110
// keeps its bits down to there.
struct Parts {
  bf16x8 p[3];
};

__device__ __forceinline__ Parts split(f32x4 lo, f32x4 hi) {
  constexpr float kMost = 0x1.fep127f;
  uint32_t w[3][4];
#pragma unroll
  for (int i = 0; i < 4; i++) {   // a word of parts for two values
    f32x2 v = i < 2 ? f32x2{lo[2 * i], lo[2 * i + 1]} : f32x2{hi[2 * i - 4], hi[2 * i - 3]};
#pragma unroll
    for (int k = 0; k < 3; k++) {
      const f32x2 c = k ? v : f32x2{__builtin_amdgcn_fmed3f(v[0], -kMost, kMost), __builtin_amdgcn_fmed3f(v[1], -kMost, kMost)};
      w[k][i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(c, bf16x2));
      if (k < 2) {
        v[0] -= __builtin_bit_cast(float, w[k][i] << 16);
        v[1] -= __builtin_bit_cast(float, w[k][i] & 0xffff0000u);
      }
    }
  }
  Parts r;
#pragma unroll
  for (int k = 0; k < 3; k++) r.p[k] = __builtin_bit_cast(bf16x8, w[k]);
  return r;
}

// The product of all parts but three, which together are at most 2^-24 of the
// whole, one rounding of float32; smallest first.
__device__ __forceinline__ f32x4 run_parts(const Parts& a, const Parts& b, f32x4 c) {
  c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.p[1], b.p[1], c, 0, 0, 0);
  c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.p[0], b.p[2], c, 0, 0, 0);
  c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.p[2], b.p[0], c, 0, 0, 0);
  c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.p[0], b.p[1], c, 0, 0, 0);
  c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.p[1], b.p[0], c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.p[0], b.p[0], c, 0, 0, 0);
}

typedef __attribute__((address_space(3))) void LdsVoid;
typedef __attribute__((address_space(3))) i16x4 LdsI16x4;

__device__ __forceinline__ int wave_id() { return __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)); }

// Unit permutation of a k-outermost row, for R / 16 units (a power of two).
template <typename T, int R>
__device__ __forceinline__ int unit_swizzle(int k) {
  const int s = sizeof(T) == 2 ? (k & 3) | ((k >> 3) & 1) << 2 : (k >> 2) & 3;
  return s & (R / 16 - 1);
}

// The direct loads of one operand's tile of R rows (kKM) or R columns.
template <typename T, bool kKM, int R, int NT>
struct Loader {
  static constexpr int kVec = 16 / (int)sizeof(T), kLoads = R * 8 / NT;
  static constexpr int kRow = R / kVec;              // chunks of a k-outermost row
  static constexpr int kStep = kStepBytes / (int)sizeof(T);
  static constexpr int kPer = kKM ? 0 : NT / kRow;   // rows of k between a lane's loads
  uint32_t off[kLoads];
  int k_first;            // this lane's first k inside a step
  const char* base;
  int64_t advance;

  // Rows first .. first + R - 1 of n (kKM), or columns of a matrix of `n` columns.
  __device__ __forceinline__ void init(const T* p, int64_t ld, int64_t first, int64_t n) {
    const int t = threadIdx.x;
    if constexpr (kKM) {
      const int r = t >> 3, c = (t & 7) ^ (r & 7);
      k_first = c * kVec;
      base = reinterpret_cast<const char*>(p + first * ld);
      advance = kStepBytes;
#pragma unroll
      for (int i = 0; i < kLoads; i++) {
        const int row = r + i * (NT / 8);
        off[i] = first + row < n ? (uint32_t)((row * ld + k_first) * (int64_t)sizeof(T)) : kOutside;
      }
    } else {
      const int k = t / kRow, c = t % kRow;
      constexpr int kUnit = (int)sizeof(T);          // chunks of a 16-element unit
      k_first = k;
      base = reinterpret_cast<const char*>(p + first);
      advance = ld * kStepBytes;                     // kStep rows
#pragma unroll
      for (int i = 0; i < kLoads; i++) {
        const int row = k + i * kPer;
        const int col = ((c / kUnit) ^ unit_swizzle<T, R>(row)) * 16 + (c % kUnit) * kVec;
        off[i] = first + col < n ? (uint32_t)((row * ld + col) * (int64_t)sizeof(T)) : kOutside;
      }
    }
  }

  // Two weight matrices as one tile of R rows: 16 rows of the first, the same
  // 16 of the second, and so on; rows first .. first + R / 2 - 1 of n of each.
  __device__ __forceinline__ void init_pair(const T* p0, const T* p1, int64_t ld, int64_t first, int64_t n) {
    static_assert(!kKM || NT % 256 == 0, "a wave's loads stay with one matrix");
    const int t = threadIdx.x;
    const int r = t >> 3, c = (t & 7) ^ (r & 7);
    k_first = c * kVec;
    base = reinterpret_cast<const char*>(((wave_id() >> 1) & 1 ? p1 : p0) + first * ld);
    advance = kStepBytes;
#pragma unroll
    for (int i = 0; i < kLoads; i++) {
      const int lrow = r + i * (NT / 8);
      const int row = (lrow >> 5) * 16 + (lrow & 15);
      off[i] = first + row < n ? (uint32_t)((row * ld + k_first) * (int64_t)sizeof(T)) : kOutside;
    }
  }

  // Loads the step at base into lds; k_left values of k remain.
  __device__ __forceinline__ void issue(uint8_t* lds, int64_t k_left) const {
    auto rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base), (short)0, (int)kRecords, 0x00020000);
    uint8_t* at = lds + wave_id() * 1024;
#pragma unroll
    for (int i = 0; i < kLoads; i++) {
      const uint32_t v = k_first + i * kPer < k_left ? off[i] : kOutside;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (LdsVoid*)(at + i * NT * 16), 16, (int)v, 0, 0, 0);
    }
  }
};

// Where a lane reads its part of the fragments of a wave whose first row (or
// column) is `first`, a multiple of 16 times the wave's power-of-two number of
// fragments: fragment i is at an XOR of this with a constant and a constant
// offset, so the addresses cost one register a fragment at most.
template <typename T, bool kKM, int R>
__device__ __forceinline__ int fragment_base(int first) {
  const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
  if constexpr (kKM) return (first + r) * kStepBytes + ((q ^ (r & 7)) << 4);
  if constexpr (sizeof(T) == 2) {
    // each group of 16 lanes reads 4 rows of 16 values and gets them transposed
    const int k = q * 8 + (r >> 2);
    return (k * (R * 2) + (unit_swizzle<T, R>(k) << 5) + (r & 3) * 8) ^ (first >> 4 << 5);
  }
  return (q * 4 * (R * 4) + (unit_swizzle<T, R>(q * 4) << 6) + r * 4) ^ (first >> 4 << 6);
}

// Fragment i (16 rows or columns) at half kb of a step.
template <typename T, bool kKM, int R>
__device__ __forceinline__ typename Mma<T>::Frag fragment(const uint8_t* lds, int base, int i, int kb) {
  if constexpr (kKM) {
    return *reinterpret_cast<const typename Mma<T>::Frag*>(lds + (base ^ (kb << 6)) + i * 16 * kStepBytes);
  } else if constexpr (sizeof(T) == 2) {
    const uint8_t* at = lds + (base ^ (i << 5)) + kb * 32 * (R * 2);
    i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsI16x4*)at);
    i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsI16x4*)(at + 4 * (R * 2)));
    return __builtin_bit_cast(typename Mma<T>::Frag, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  } else {
    f32x4 f;
#pragma unroll
    for (int j = 0; j < 4; j++) f[j] = *reinterpret_cast<const float*>(lds + (base ^ (i << 6)) + (kb * 16 + j) * (R * 4));
    return f;
  }
}

// BM x BN by WM x WN waves of (16 FM) x (16 FN), with `stages` LDS buffers.
template <int kBM, int kBN, int kWM, int kWN, int kStages>
struct Tile {
  static constexpr int BM = kBM, BN = kBN, WM = kWM, WN = kWN, NT = 64 * WM * WN, FM = BM / WM / 16, FN = BN / WN / 16;
  static constexpr int stages = kStages;
};
typedef Tile<256, 256, 2, 4, 2> TileL;
typedef Tile<128, 128, 2, 2, 2> TileM;
typedef Tile<64, 64, 2, 2, 2> TileS;
typedef Tile<64, 64, 2, 2, 4> TileS4;

// LDS buffer kBuf of a step.  They are separate arrays, so that the compiler
// knows a direct load into one not to touch a fragment of another.
template <typename C, int kBuf = 0>
__device__ __forceinline__ uint8_t* tile_lds() {
  __shared__ __attribute__((aligned(16))) uint8_t lds[(C::BM + C::BN) * kStepBytes];
  return lds;
}

template <int n>
struct Number {
  static constexpr int value = n;
};

// f(Number<0>()), f(Number<1>()), ... f(Number<n - 1>()).
template <int n, int i = 0, typename F>
__device__ __forceinline__ void each(F f) {
  if constexpr (i < n) {
    f(Number<i>());
    each<n, i + 1>(f);
  }
}

// step(Number<s % n>()) for each s < total.  One loop with one way out and, in
// the 16-bit products, no branch inside: after a jump from the middle, or a
// branch in a step, the compiler no longer knows which loads are in flight and
// waits for all of them at the loop's top.  With a branch at the second operand
// pair every other step of y, dx and dw did so: 2220 us for 8192 x 2048, 8192
// forward and backward, without it 2155.
template <int n, typename F>
__device__ __forceinline__ void each_step(int total, F step) {
  int left = total;
  for (; left >= n; left -= n) each<n>(step);
  each<n - 1>([&](auto i) {
    if (i.value < left) step(i);
  });
}

// A barrier after all but this wave's last n direct loads have landed; its LDS
// reads are done.  The wait is written out: __syncthreads() promises none for
// direct loads.
template <int n>
__device__ __forceinline__ void landed_barrier() {
  static_assert(n < 64, "");
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(n) : "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// acc[i][j]: rows m = 16 i + lane % 16, columns n = 16 j + 4 (lane / 16) + 0..3
// of the wave's part.  `steps` steps of k from each of `segments` operand
// pairs; a2 and b2: the second pair's bases.  Loads are issued past the last
// step, where all of their lanes are outside, so that each wait counts the
// same; a barrier has to follow before the LDS is used again.
template <typename T, bool kAK, bool kBK, typename C>
__device__ __forceinline__ void tile_product(Loader<T, kAK, C::BM, C::NT>& la, Loader<T, kBK, C::BN, C::NT>& lb, int64_t K,
                                             const char* a2, const char* b2, f32x4 (&acc)[C::FM][C::FN]) {
  constexpr int kStep = kStepBytes / (int)sizeof(T), kBufs = C::stages;
  constexpr int kStepLoads = Loader<T, kAK, C::BM, C::NT>::kLoads + Loader<T, kBK, C::BN, C::NT>::kLoads;
  const int steps = K > kStep ? (int)((K + kStep - 1) / kStep) : 1;
  const int total = a2 ? 2 * steps : steps;
  int64_t k_left = K;
  int next = 0;
  auto issue = [&](auto buf) {
    const bool second = a2 && next == steps;   // the second pair, by selects: see each_step
    la.base = second ? a2 : la.base;
    lb.base = second ? b2 : lb.base;
    k_left = second ? K : k_left;
    uint8_t* const lds = tile_lds<C, buf.value>();
    la.issue(lds, k_left);
    lb.issue(lds + C::BM * kStepBytes, k_left);
    la.base += la.advance;
    lb.base += lb.advance;
    k_left -= kStep;
    next++;
    __builtin_amdgcn_sched_barrier(0);   // first of all, not among the products
  };
  const int w = wave_id(), wm = (w / C::WN) * C::FM * 16, wn = (w % C::WN) * C::FN * 16;
  const int ba = fragment_base<T, kAK, C::BM>(wm), bb = fragment_base<T, kBK, C::BN>(wn);
  if constexpr (sizeof(T) == 4) {
    // Both halves of a step's k make one 32-wide product of the parts.
    each<kBufs - 1>(issue);
    each_step<kBufs>(total, [&](auto buf) {
      landed_barrier<(kBufs - 2) * kStepLoads>();   // this step has landed, the last one is all read
      issue(Number<(buf.value + kBufs - 1) % kBufs>());
      const uint8_t* a = tile_lds<C, buf.value>();
      const uint8_t* b = a + C::BM * kStepBytes;
      Parts pb[C::FN];
#pragma unroll
      for (int j = 0; j < C::FN; j++) pb[j] = split(fragment<T, kBK, C::BN>(b, bb, j, 0), fragment<T, kBK, C::BN>(b, bb, j, 1));
#pragma unroll
      for (int i = 0; i < C::FM; i++) {
        const Parts pa = split(fragment<T, kAK, C::BM>(a, ba, i, 0), fragment<T, kAK, C::BM>(a, ba, i, 1));
#pragma unroll
        for (int j = 0; j < C::FN; j++) acc[i][j] = run_parts(pb[j], pa, acc[i][j]);
      }
    });
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    return;
  }
  // A step is four phases: half kb of k times half of the wave's rows.  Each
  // phase reads the next one's fragments before its own products, so LDS works
  // beside the matrix cores; the barrier stands before the last phase, whose
  // fragments are in registers by then.
  constexpr int kHalf = C::FM / 2;
  typename Mma<T>::Frag fa[2][kHalf], fb[2][C::FN];
  auto load_a = [&](int to, const uint8_t* a, int kb, int half) {
#pragma unroll
    for (int i = 0; i < kHalf; i++) fa[to][i] = fragment<T, kAK, C::BM>(a, ba, half * kHalf + i, kb);
  };
  auto load_b = [&](int to, const uint8_t* a, int kb) {
#pragma unroll
    for (int j = 0; j < C::FN; j++) fb[to][j] = fragment<T, kBK, C::BN>(a + C::BM * kStepBytes, bb, j, kb);
  };
  auto products = [&](int half, int from_a, int from_b) {
#pragma unroll
    for (int i = 0; i < kHalf; i++)
#pragma unroll
      for (int j = 0; j < C::FN; j++)
        acc[half * kHalf + i][j] = Mma<T>::run(fb[from_b][j], fa[from_a][i], acc[half * kHalf + i][j]);
    __builtin_amdgcn_sched_barrier(0);
  };
  each<kBufs>(issue);
  landed_barrier<(kBufs - 1) * kStepLoads>();
  load_a(0, tile_lds<C>(), 0, 0);
  load_b(0, tile_lds<C>(), 0);
  each_step<kBufs>(total, [&](auto buf) {
    const uint8_t* const at = tile_lds<C, buf.value>();
    const uint8_t* const at_next = tile_lds<C, (buf.value + 1) % kBufs>();
    load_a(1, at, 0, 1);
    products(0, 0, 0);
    load_a(0, at, 1, 0);
    load_b(1, at, 1);
    products(1, 1, 0);
    load_a(1, at, 1, 1);
    products(0, 0, 1);
    landed_barrier<(kBufs - 2) * kStepLoads>();   // the next step has landed; this one's fragments are all read
    issue(buf);
    load_a(0, at_next, 0, 0);   // after the last step: of no use, and of no harm
    load_b(0, at_next, 0);
    products(1, 1, 1);
  });
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // no load into LDS outlives the workgroup
}

// The tile of a workgroup.  Workgroups go to the eight XCDs in turn, each with
// an L2 of its own: XCD x takes the x-th contiguous part of the tiles, and
// runs through them 4 rows at a time, so that the 32 tiles in flight there
// share 4 row panels and 8 column panels.
__device__ __forceinline__ void tile_of(int id, int tiles_m, int tiles_n, int& tm, int& tn) {
  const int n = tiles_m * tiles_n, q = n / 8, r = n % 8, x = id % 8, l = id / 8;
  const int t = x < r ? x * (q + 1) + l : r * (q + 1) + (x - r) * q + l;
  const int group = t / (4 * tiles_n), rest = t % (4 * tiles_n);
  const int rows = tiles_m - group * 4 < 4 ? tiles_m - group * 4 : 4;
  tm = group * 4 + rest % rows;
  tn = rest / rows;
}

}  // namespace nest
