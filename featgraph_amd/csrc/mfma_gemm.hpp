// Matrix product core of the linear cross entropy: C[m, n] = sum over k of A[m, k] * B[n, k] on the matrix cores, both
// operands bfloat16 with k contiguous, float32 accumulators that never leave the registers before the epilogue.
//
// float32 operands come as three bfloat16 parts each (x = x0 + x1 + x2, 24 bits of the mantissa): six of the nine
// products are added, smallest first; the three that are left out are below 2^-24 of the result's terms.  Both cases
// are one loop over k, the segments only pick the parts.
//
// A workgroup computes a BM x BN tile.  Steps of 64 k are loaded straight to LDS (16 bytes per lane, no registers in
// between) into one of two stages while the other one feeds the matrix instructions.  A tile row is 128 bytes in LDS;
// its eight 16-byte pieces are placed at (piece ^ (row / 2 % 8)), so that the 64 lanes of a fragment read, which take
// the same piece of consecutive rows, spread over all banks.  The permutation is applied on the way in, by what each
// lane fetches.  Rows past the operands' ends are read as the last row and dropped by the epilogues; k is a multiple
// of 64 (padded copies hold zeros there).
#pragma once

#include "element.hpp"

namespace fg {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kStepK = 64;
constexpr int kParts = 3;     // bfloat16 parts of a float32
constexpr int kSegments = 6;  // products of parts that are added

struct GemmOperand {
  const uint16_t *p = nullptr;  // part 0
  int64_t part = 0;             // elements from one part to the next
  int64_t pitch = 0;            // elements from one row to the next, a multiple of 8
  int32_t rows = 0;
};

struct GemmShape {
  GemmOperand a, b;
  int32_t steps = 0;     // of kStepK per part
  int32_t segments = 1;  // 1, or kSegments for split float32
  int32_t splits = 1;    // workgroups that share one tile's k range
  int32_t tiles_m = 0, tiles_n = 0;
};

// Parts that segment s of kSegments multiplies; the last one is the plain product of the leading parts.
__device__ __forceinline__ int part_of_a(int s) { return (0x021010 >> (4 * (kSegments - 1 - s))) & 15; }
__device__ __forceinline__ int part_of_b(int s) { return (0x201100 >> (4 * (kSegments - 1 - s))) & 15; }

template <int BM_, int BN_, int WM_, int WN_>
struct GemmTile {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_;
  static constexpr int kWaves = WM * WN, kThreads = kWaves * kWaveSize;
  static constexpr int TM = BM / WM / 32, TN = BN / WN / 32;         // 32 x 32 blocks of one wave
  static constexpr int kLoadsA = BM / 8 / kWaves, kLoadsB = BN / 8 / kWaves;  // 8 rows of 128 bytes per wave and load
  static constexpr int kStage = (BM + BN) * kStepK;                  // elements of one stage
  static constexpr int kLds = 2 * kStage;                            // both stages
  static_assert(kLoadsA * 8 * kWaves == BM && kLoadsB * 8 * kWaves == BN, "rows divide over the waves");
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

template <typename Tile>
__device__ __forceinline__ void gemm_tile(const GemmShape &g, const GemmPlace &at, uint16_t *lds, GemmAcc<Tile> &acc) {
#if defined(__HIP_DEVICE_COMPILE__)  // the host pass lacks the loads to LDS
  using LdsPtr = __attribute__((address_space(3))) void *;
  const int lane = threadIdx.x & (kWaveSize - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWaveSize);
  const int wm = wave / Tile::WN, wn = wave % Tile::WN;
#pragma unroll
  for (int i = 0; i < Tile::TM; ++i)
#pragma unroll
    for (int j = 0; j < Tile::TN; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc.c[i][j][r] = 0.0f;

  // what this lane fetches: row lane / 8 of the eight of a load, piece (lane % 8) after the permutation
  const int64_t m0 = static_cast<int64_t>(at.tm) * Tile::BM, n0 = static_cast<int64_t>(at.tn) * Tile::BN;
  const int rows_a = static_cast<int>(min<int64_t>(Tile::BM, g.a.rows - m0));
  const int rows_b = static_cast<int>(min<int64_t>(Tile::BN, g.b.rows - n0));
  const uint32_t pitch_a = static_cast<uint32_t>(g.a.pitch) * 2, pitch_b = static_cast<uint32_t>(g.b.pitch) * 2;
  uint32_t off_a[Tile::kLoadsA], off_b[Tile::kLoadsB];
#pragma unroll
  for (int j = 0; j < Tile::kLoadsA; ++j) {
    const int row = (wave + j * Tile::kWaves) * 8 + lane / 8;
    off_a[j] = min(row, rows_a - 1) * pitch_a + ((lane % 8) ^ ((row >> 1) & 7)) * 16;
  }
#pragma unroll
  for (int j = 0; j < Tile::kLoadsB; ++j) {
    const int row = (wave + j * Tile::kWaves) * 8 + lane / 8;
    off_b[j] = min(row, rows_b - 1) * pitch_b + ((lane % 8) ^ ((row >> 1) & 7)) * 16;
  }
  const uint32_t bytes_a = rows_a * pitch_a, bytes_b = rows_b * pitch_b;

  const int total = g.steps * g.segments;
  const int first = static_cast<int>(static_cast<int64_t>(total) * at.split / g.splits);
  const int last = static_cast<int>(static_cast<int64_t>(total) * (at.split + 1) / g.splits);
  int seg = first / g.steps, step = first - seg * g.steps;  // of the next load
  auto load = [&](int stage) {
    const int s = seg + kSegments - g.segments;
    const uint16_t *pa = g.a.p + part_of_a(s) * g.a.part + m0 * g.a.pitch;
    const uint16_t *pb = g.b.p + part_of_b(s) * g.b.part + n0 * g.b.pitch;
    const __amdgpu_buffer_rsrc_t ra = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t *>(pa), 0, bytes_a, 0x00020000);
    const __amdgpu_buffer_rsrc_t rb = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t *>(pb), 0, bytes_b, 0x00020000);
    const int k = step * (kStepK * 2);
    uint16_t *base = lds + stage * Tile::kStage;
#pragma unroll
    for (int j = 0; j < Tile::kLoadsA; ++j)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, (LdsPtr)(base + (wave + j * Tile::kWaves) * 8 * kStepK), 16, off_a[j], k, 0, 0);
#pragma unroll
    for (int j = 0; j < Tile::kLoadsB; ++j)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          rb, (LdsPtr)(base + (Tile::BM + (wave + j * Tile::kWaves) * 8) * kStepK), 16, off_b[j], k, 0, 0);
    if (++step == g.steps) {
      step = 0;
      ++seg;
    }
  };

  // fragment reads: lane l takes row l % 32, pieces 2 kk + l / 32 of the row for k step kk of 16
  const int row_a = wm * (Tile::BM / Tile::WM) + lane % 32, row_b = wn * (Tile::BN / Tile::WN) + lane % 32;
  const int twist = (lane >> 1) & 7;
  if (first < last) load(0);
  for (int i = first; i < last; ++i) {
    const int stage = (i - first) & 1;
    __syncthreads();  // this stage has arrived, and nobody reads the other one any more
    if (i + 1 < last) load(stage ^ 1);
    const uint16_t *sa = lds + stage * Tile::kStage + row_a * kStepK;
    const uint16_t *sb = lds + stage * Tile::kStage + (Tile::BM + row_b) * kStepK;
#pragma unroll
    for (int kk = 0; kk < kStepK / 16; ++kk) {
      const int piece = ((2 * kk + lane / 32) ^ twist) * 8;
      bf16x8 fa[Tile::TM], fb[Tile::TN];
#pragma unroll
      for (int t = 0; t < Tile::TM; ++t) fa[t] = *reinterpret_cast<const bf16x8 *>(sa + t * 32 * kStepK + piece);
#pragma unroll
      for (int t = 0; t < Tile::TN; ++t) fb[t] = *reinterpret_cast<const bf16x8 *>(sb + t * 32 * kStepK + piece);
#pragma unroll
      for (int t = 0; t < Tile::TM; ++t)
#pragma unroll
        for (int u = 0; u < Tile::TN; ++u)
          acc.c[t][u] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa[t], fb[u], acc.c[t][u], 0, 0, 0);
    }
  }
#endif
}

}  // namespace fg
