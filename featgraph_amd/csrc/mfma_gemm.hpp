// Matrix product core of the linear cross entropy: C[m, n] = sum over k of A[m, k] * B[n, k] on the matrix cores, both
// operands of 16-bit floats with k contiguous, float32 accumulators that never leave the registers before the epilogue.
//
// bfloat16 operands are multiplied as they are.  A float32 operand comes as two float16 parts of x * 2^e: hi, the value
// rounded to 11 bits, and lo, the rest times 2^11 rounded to 11 bits, so that hi + lo * 2^-11 is x * 2^e to 2^-23 of
// itself (the exponent e of a row or a matrix brings its largest element to 2^14; elements down to 2^-28 of that keep
// full relative accuracy, smaller ones 2^-49 of the largest).  Three of the four products are added: hi * lo and lo * hi
// first, then, after the sum is multiplied by 2^-11, hi * hi; lo * lo is at most 2^-24 of the terms.  That is float32's
// accuracy at a third of the 16-bit rate, 5.3 times the peak rate of the float32 matrix instructions.
//
// A workgroup computes a BM x BN tile in steps of 32 k.  The operands' rows go straight to LDS (16 bytes per lane, no
// registers in between) into one of four stages, three steps ahead; the fragments of a step's first half are read
// while the step before it still multiplies, so that a wave never waits for LDS with nothing to issue.  A tile row is
// 64 bytes in LDS; its four 16-byte pieces are placed at (piece ^ (row / 4 % 4)), so that the lanes of a fragment read,
// which take the same piece of consecutive rows, spread over all banks.  The permutation is applied on the way in, by
// what each lane fetches.  Rows past the operands' ends are read as the last row and dropped by the epilogues; k is a
// multiple of 64 (padded copies hold zeros there).
#pragma once

#include "element.hpp"

namespace fg {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kPadK = 64;     // k is padded to a multiple of this
constexpr int kStepK = 32;    // k of one stage
constexpr int kStages = 4;
constexpr int kParts = 2;     // float16 parts of a float32
constexpr int kSegments = 3;  // products of parts that are added
constexpr int kLowBits = 11;  // lo is kept times 2^kLowBits

// How operands of type T (float or __bf16) are multiplied.
template <typename T>
struct Multiply;
template <>
struct Multiply<__bf16> {
  static constexpr int kParts = 1, kSegments = 1;
  static __device__ __forceinline__ f32x16 mfma(bf16x8 a, bf16x8 b, f32x16 c) {
#if defined(__HIP_DEVICE_COMPILE__)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
#else
    return c;
#endif
  }
};
template <>
struct Multiply<float> {
  static constexpr int kParts = fg::kParts, kSegments = fg::kSegments;
  static __device__ __forceinline__ f32x16 mfma(bf16x8 a, bf16x8 b, f32x16 c) {
#if defined(__HIP_DEVICE_COMPILE__)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
#else
    return c;
#endif
  }
};

struct GemmOperand {
  const uint16_t *p = nullptr;  // part 0
  int64_t part = 0;             // elements from one part to the next
  int64_t pitch = 0;            // elements from one row to the next, a multiple of 8
  int32_t rows = 0;
};

struct GemmShape {
  GemmOperand a, b;
  int32_t steps = 0;   // of kStepK per part
  int32_t splits = 1;  // workgroups that share one tile's k range
  int32_t tiles_m = 0, tiles_n = 0;
};

template <int BM_, int BN_, int WM_, int WN_>
struct GemmTile {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_;
  static constexpr int kWaves = WM * WN, kThreads = kWaves * kWaveSize;
  static constexpr int TM = BM / WM / 32, TN = BN / WN / 32;                  // 32 x 32 blocks of one wave
  static constexpr int kLoadsA = BM / 16 / kWaves, kLoadsB = BN / 16 / kWaves;  // 16 rows of 64 bytes per wave and load
  static constexpr int kStage = (BM + BN) * kStepK;                           // elements of one stage
  static constexpr int kLds = kStages * kStage;
  static_assert(kLoadsA * 16 * kWaves == BM && kLoadsB * 16 * kWaves == BN, "rows divide over the waves");
};

// Where this workgroup works: tile and share of k.  Workgroup id x runs on die x % 8; the ids of one die are mapped
// to consecutive tiles, n fastest, so that each die's L2 keeps the operand rows its tiles share.
struct GemmPlace {
  int32_t tm, tn, split;
};
__device__ __forceinline__ GemmPlace gemm_place(const GemmShape &g) {
  const uint32_t total = gridDim.x, q = total / kXcds, r = total % kXcds;
  const uint32_t die = blockIdx.x % kXcds, k = blockIdx.x / kXcds;
  const uint32_t id = die * q + min(die, r) + k;
  const uint32_t tiles = static_cast<uint32_t>(g.tiles_m) * static_cast<uint32_t>(g.tiles_n);
  GemmPlace p;
  p.split = static_cast<int32_t>(id / tiles);
  const uint32_t t = id - p.split * tiles;
  p.tm = static_cast<int32_t>(t / g.tiles_n);
  p.tn = static_cast<int32_t>(t - static_cast<uint32_t>(p.tm) * g.tiles_n);
  return p;
}

template <typename Tile>
struct GemmAcc {
  f32x16 c[Tile::TM][Tile::TN];
};

// Row of the accumulator's register r in a 32 x 32 block (the column is lane % 32).
__device__ __forceinline__ int acc_row(int r, int lane) { return 8 * (r / 4) + 4 * (lane / 32) + r % 4; }

// Every wave's loads but the newest `kAhead` and all its LDS reads are done, then all waves meet.
template <int kAhead>
__device__ __forceinline__ void arrive_and_meet() {
#if defined(__HIP_DEVICE_COMPILE__)
  static_assert(kAhead < 64, "vmcnt has six bits");
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"i"(kAhead) : "memory");
#endif
}

template <typename Tile, typename T>
__device__ __forceinline__ void gemm_tile(const GemmShape &g, const GemmPlace &at, uint16_t *lds, GemmAcc<Tile> &acc) {
#if defined(__HIP_DEVICE_COMPILE__)  // the host pass lacks the loads to LDS
  using LdsPtr = __attribute__((address_space(3))) void *;
  using M = Multiply<T>;
  constexpr int kLoads = Tile::kLoadsA + Tile::kLoadsB;
  const int lane = threadIdx.x & (kWaveSize - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWaveSize);
  const int wm = wave / Tile::WN, wn = wave % Tile::WN;
#pragma unroll
  for (int i = 0; i < Tile::TM; ++i)
#pragma unroll
    for (int j = 0; j < Tile::TN; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc.c[i][j][r] = 0.0f;

  // what this lane fetches: row lane / 4 of the sixteen of a load, the piece that belongs at place lane % 4
  const int64_t m0 = static_cast<int64_t>(at.tm) * Tile::BM, n0 = static_cast<int64_t>(at.tn) * Tile::BN;
  const int rows_a = static_cast<int>(min<int64_t>(Tile::BM, g.a.rows - m0));
  const int rows_b = static_cast<int>(min<int64_t>(Tile::BN, g.b.rows - n0));
  const uint32_t pitch_a = static_cast<uint32_t>(g.a.pitch) * 2, pitch_b = static_cast<uint32_t>(g.b.pitch) * 2;
  const uint32_t piece_in = ((lane % 4) ^ ((lane >> 4) & 3)) * 16;  // row / 4 % 4 = lane / 16
  uint32_t off_a[Tile::kLoadsA], off_b[Tile::kLoadsB];
#pragma unroll
  for (int j = 0; j < Tile::kLoadsA; ++j)
    off_a[j] = min((wave + j * Tile::kWaves) * 16 + lane / 4, rows_a - 1) * pitch_a + piece_in;
#pragma unroll
  for (int j = 0; j < Tile::kLoadsB; ++j)
    off_b[j] = min((wave + j * Tile::kWaves) * 16 + lane / 4, rows_b - 1) * pitch_b + piece_in;
  const uint32_t bytes_a = rows_a * pitch_a, bytes_b = rows_b * pitch_b;

  const int total = g.steps * M::kSegments;
  const int first = static_cast<int>(static_cast<int64_t>(total) * at.split / g.splits);
  const int last = static_cast<int>(static_cast<int64_t>(total) * (at.split + 1) / g.splits);
  // the next load's parts and step: segment 0 is hi * lo, 1 is lo * hi, 2 (or the only one) hi * hi
  int seg = first / g.steps, step = first - seg * g.steps;
  auto load = [&](int i) {
    const uint16_t *pa = g.a.p + (M::kSegments == 3 && seg == 1 ? g.a.part : 0) + m0 * g.a.pitch;
    const uint16_t *pb = g.b.p + (M::kSegments == 3 && seg == 0 ? g.b.part : 0) + n0 * g.b.pitch;
    const __amdgpu_buffer_rsrc_t ra = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t *>(pa), 0, bytes_a, 0x00020000);
    const __amdgpu_buffer_rsrc_t rb = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t *>(pb), 0, bytes_b, 0x00020000);
    const int k = step * (kStepK * 2);
    uint16_t *base = lds + (i & (kStages - 1)) * Tile::kStage;
#pragma unroll
    for (int j = 0; j < Tile::kLoadsA; ++j)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, (LdsPtr)(base + (wave + j * Tile::kWaves) * 16 * kStepK), 16, off_a[j], k, 0, 0);
#pragma unroll
    for (int j = 0; j < Tile::kLoadsB; ++j)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          rb, (LdsPtr)(base + (Tile::BM + (wave + j * Tile::kWaves) * 16) * kStepK), 16, off_b[j], k, 0, 0);
    if (++step == g.steps) {
      step = 0;
      ++seg;
    }
  };

  // fragments: lane l holds row l % 32, eight k from 16 * half + 8 * (l / 32) on
  const int row_a = wm * (Tile::BM / Tile::WM) + lane % 32, row_b = wn * (Tile::BN / Tile::WN) + lane % 32;
  const int twist = (lane >> 2) & 3;
  const int at_a = row_a * kStepK, at_b = (Tile::BM + row_b) * kStepK;
  const int half0 = ((lane / 32) ^ twist) * 8, half1 = ((2 + lane / 32) ^ twist) * 8;
  struct Fragments {
    bf16x8 a[Tile::TM], b[Tile::TN];
  };
  auto read = [&](Fragments &f, int i, int half) {
    const uint16_t *s = lds + (i & (kStages - 1)) * Tile::kStage + half;
#pragma unroll
    for (int t = 0; t < Tile::TM; ++t) f.a[t] = *reinterpret_cast<const bf16x8 *>(s + at_a + t * 32 * kStepK);
#pragma unroll
    for (int t = 0; t < Tile::TN; ++t) f.b[t] = *reinterpret_cast<const bf16x8 *>(s + at_b + t * 32 * kStepK);
  };
  auto multiply = [&](const Fragments &f) {
#pragma unroll
    for (int t = 0; t < Tile::TM; ++t)
#pragma unroll
      for (int u = 0; u < Tile::TN; ++u) acc.c[t][u] = M::mfma(f.a[t], f.b[u], acc.c[t][u]);
  };
  auto lower = [&]() {
#pragma unroll
    for (int t = 0; t < Tile::TM; ++t)
#pragma unroll
      for (int u = 0; u < Tile::TN; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc.c[t][u][r] *= 1.0f / (1 << kLowBits);
  };

  const int n = last - first;
  const int cross = M::kSegments == 3 ? 2 * g.steps - first : 0;  // steps of this share before hi * hi begins
  if (n > 0) {
    load(0);
    if (n > 1) load(1);
    if (n > 2) load(2);
    Fragments f0, f1;
    // step 0 has arrived (its loads are the oldest)
    if (n > 2) arrive_and_meet<2 * kLoads>();
    else arrive_and_meet<0>();
    read(f0, 0, half0);
    for (int i = 0; i < n; ++i) {
      // step i + 1 has arrived for every wave, and nobody reads step i - 1 any more, whose stage step i + 3 takes
      if (i + 2 < n) arrive_and_meet<kLoads>();
      else arrive_and_meet<0>();
      if (i + 3 < n) load(i + 3);
      if (M::kSegments == 3 && i > 0 && i == cross) lower();
      read(f1, i, half1);
      multiply(f0);
      if (i + 1 < n) read(f0, i + 1, half0);
      multiply(f1);
    }
    if (M::kSegments == 3 && cross >= n) lower();
  }
#endif
}

}  // namespace fg
