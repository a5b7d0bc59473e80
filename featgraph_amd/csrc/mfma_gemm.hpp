// Matrix product core of the linear cross entropy: C[m, n] = sum over k of A[m, k] * B[n, k] on the matrix cores, both
// operands of 16-bit floats with k contiguous, float32 accumulators that never leave the registers before the epilogue.
//
// bfloat16 operands are multiplied as they are.  A float32 operand comes as two float16 parts of x * 2^e: hi, the value
// rounded to 11 bits, and lo, the rest times 2^11 rounded to 11 bits, so that hi + lo * 2^-11 is x * 2^e to 2^-23 of
// itself (the exponent e of a row or a matrix brings its largest element to 2^14 or more; elements down to 2^-27 of that keep
// their relative accuracy, smaller ones 2^-50 of the largest, and weigh like 2^-28 of it where the matrix instructions align
// the products that they add: a denormal factor counts as 2^-14 there).  Three of the four products are added: hi * lo and lo * hi
// first, then, after the sum is multiplied by 2^-11, hi * hi; lo * lo is at most 2^-22 of a term, of either sign.  That is
// near float32's accuracy at a third of the 16-bit rate, 5.3 times the peak rate of the float32 matrix instructions.
//
// A workgroup computes a BM x BN tile in steps of 64 k.  The operands' rows go straight to LDS (16 bytes per lane, whole
// 128-byte lines, no registers in between) into the next of two stages of B and, where LDS allows, three of A: then only
// the loads of the step's second half have to arrive within it.  The fragments of each quarter of a step are read
// while the quarter before it multiplies, over the border of the steps too: the waves meet before the last quarter, when
// its fragments are in registers, the next stage has arrived and this one can be filled again.  A tile row is 128 bytes
// in LDS; its eight 16-byte pieces are placed at (piece ^ (row / 2 % 8)), so that the lanes of a fragment read, which
// take the same piece of consecutive rows, spread over all banks.  The permutation is applied on the way in, by what
// each lane fetches.  Rows past the operands' ends are read as the last row and dropped by the epilogues; k is a
// multiple of 64 (padded copies hold zeros there).
//
// A may also be turned: panels of 64 of its rows, one line per k.  Its stage is then [64 k][BM] in LDS, and a lane reads
// TM neighbouring rows of eight k lines; halves of two lines put together are a pair of k of one row.  The TM rows belong
// to the TM blocks of the wave, so that nothing moves between lanes: row r of block i is row TM * r + i of the wave's.
#pragma once

#include <type_traits>

#include "element.hpp"

namespace fg {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kStepK = 64;    // k of one stage; k is padded to a multiple of this
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

// float32 operands as they are, on the float32 matrix instructions: a fragment of 16 bytes is four k.  A sixth of the
// rate, but no copies: for products that are bound by reading one of the operands.
struct MultiplyNative {
  static constexpr int kParts = 1, kSegments = 1;
  static __device__ __forceinline__ f32x16 mfma(bf16x8 a, bf16x8 b, f32x16 c) {
#if defined(__HIP_DEVICE_COMPILE__)
    typedef float f32x4 __attribute__((ext_vector_type(4)));
    const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
    for (int k = 0; k < 4; ++k) c = __builtin_amdgcn_mfma_f32_32x32x2f32(x[k], y[k], c, 0, 0, 0);
#endif
    return c;
  }
};

// Elements are 16 bits; a native float32 counts as two.
struct GemmOperand {
  const uint16_t *p = nullptr;  // part 0
  int64_t part = 0;             // elements from one part to the next
  int64_t row = kStepK;         // elements from one row to the next: a multiple of 8, native float32 of 2
  int64_t step = 0;             // elements from one step of k to the next
  int32_t rows = 0;
};

// Parts of `rows` rows of k elements each, as panels.
inline int64_t panel_elements(int64_t rows, int64_t k) { return (k + kStepK - 1) / kStepK * kStepK * rows; }
inline GemmOperand panels(const uint16_t *p, int64_t rows, int64_t k) {
  GemmOperand o;
  o.p = p;
  o.part = panel_elements(rows, k);
  o.step = rows * kStepK;
  o.rows = static_cast<int32_t>(rows);
  return o;
}
// Rows of the same panels as columns, and columns as rows: `rows` operand rows over `k` k lines, padded to whole panels.
inline GemmOperand turned_panels(const uint16_t *p, int64_t rows, int64_t k) {
  const int64_t lines = (k + kStepK - 1) / kStepK * kStepK;
  GemmOperand o;
  o.p = p;
  o.part = panel_elements(lines, rows);
  o.row = lines;  // a panel of 64 rows has `lines` lines of 64
  o.step = kStepK * kStepK;
  o.rows = static_cast<int32_t>(rows);
  return o;
}
__device__ __forceinline__ int64_t panel_at(int64_t rows, int64_t row, int64_t k) {
  return k / kStepK * (rows * kStepK) + row * kStepK + k % kStepK;
}

struct GemmShape {
  GemmOperand a, b;
  int32_t steps = 0;   // of kStepK per part
  int32_t splits = 1;  // workgroups that share one tile's k range
  int32_t tail = kStepK;  // native: elements of the last step that exist (the others are whole in copies and in place)
  int32_t tiles_m = 0, tiles_n = 0;
};

template <int BM_, int BN_, int WM_, int WN_, int kStagesA_>
struct GemmTile {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, kStagesA = kStagesA_;
  static constexpr int kWaves = WM * WN, kThreads = kWaves * kWaveSize;
  static constexpr int TM = BM / WM / 32, TN = BN / WN / 32;                  // 32 x 32 blocks of one wave
  static constexpr int kLoadsA = BM / 8 / kWaves, kLoadsB = BN / 8 / kWaves;  // 8 rows of 128 bytes per wave and load
  static constexpr int kStageA = BM * kStepK, kStageB = BN * kStepK;          // elements of one stage
  static constexpr int kLds = kStagesA * kStageA + 2 * kStageB;
  static_assert(kStagesA == 2 || kStagesA == 3);
  static_assert(kLds * 2 <= 163840, "the LDS of a CU");
  static_assert(kLoadsA * 8 * kWaves == BM && kLoadsB * 8 * kWaves == BN, "rows divide over the waves");
};

// Where this workgroup works: tile and share of k.  Workgroup id x runs on die x % 8; the ids of one die are mapped
// to consecutive tiles, and those run down kGroupM tiles of m before n moves on: the 32 workgroups that a die runs at a
// time then share 8 tiles' rows of A and 4 of B, which its L2 fetches once.
constexpr uint32_t kGroupM = 8;
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
  const uint32_t band = t / (kGroupM * g.tiles_n), in_band = t - band * kGroupM * g.tiles_n;
  const uint32_t height = min(kGroupM, static_cast<uint32_t>(g.tiles_m) - band * kGroupM);
  p.tn = static_cast<int32_t>(in_band / height);
  p.tm = static_cast<int32_t>(band * kGroupM + in_band - p.tn * height);
  return p;
}

// Row of a wave's rows that register r of block i holds.
template <typename Tile, bool kTurnA>
__device__ __forceinline__ int tile_row(int i, int acc_row) {
  return kTurnA ? Tile::TM * acc_row + i : 32 * i + acc_row;
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

// The tiles at.tm .. at.tm + tiles - 1 of m one after the other, as one sequence of loads: done(i) is called with the sums
// of the i-th in acc while the next one's first rows are under way to LDS, and zeroes acc with clear() if more follow.
template <typename Tile>
__device__ __forceinline__ void clear(GemmAcc<Tile> &acc) {
#pragma unroll
  for (int i = 0; i < Tile::TM; ++i)
#pragma unroll
    for (int j = 0; j < Tile::TN; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc.c[i][j][r] = 0.0f;
}

template <typename Tile, typename M, bool kTurnA, typename Done>
__device__ __forceinline__ void gemm_tiles(const GemmShape &g, const GemmPlace &at, int tiles, uint16_t *lds,
                                           GemmAcc<Tile> &acc, Done &&done) {
#if defined(__HIP_DEVICE_COMPILE__)  // the host pass lacks the loads to LDS
  using LdsPtr = __attribute__((address_space(3))) void *;
  constexpr bool kNative = std::is_same<M, MultiplyNative>::value;
  constexpr int kLoads = Tile::kLoadsA + Tile::kLoadsB;
  const int lane = threadIdx.x & (kWaveSize - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWaveSize);
  const int wm = wave / Tile::WN, wn = wave % Tile::WN;
  clear(acc);

  // what this lane fetches: row lane / 8 of the eight of a load, the piece that belongs at place lane % 8
  const int64_t m0 = static_cast<int64_t>(at.tm) * Tile::BM, n0 = static_cast<int64_t>(at.tn) * Tile::BN;
  const uint32_t pitch_a = static_cast<uint32_t>(g.a.row) * 2, pitch_b = static_cast<uint32_t>(g.b.row) * 2;
  uint32_t off_a[Tile::kLoadsA], off_b[Tile::kLoadsB];
#pragma unroll
  for (int j = 0; j < Tile::kLoadsA; ++j) {
    if constexpr (kTurnA) {
      constexpr int kLine = Tile::BM / 8;  // 16-byte pieces of a k line in LDS
      const int at_piece = (wave + j * Tile::kWaves) * kWaveSize + lane, k = at_piece / kLine, piece = at_piece % kLine;
      off_a[j] = static_cast<uint32_t>(piece / 8) * (static_cast<uint32_t>(g.a.row) * (kStepK * 2)) + k * (kStepK * 2) + piece % 8 * 16;
    } else {
      const int row = (wave + j * Tile::kWaves) * 8 + lane / 8;
      off_a[j] = row * pitch_a + ((lane % 8) ^ ((row >> 1) & 7)) * 16;
    }
  }
#pragma unroll
  for (int j = 0; j < Tile::kLoadsB; ++j) {
    const int row = (wave + j * Tile::kWaves) * 8 + lane / 8;
    off_b[j] = row * pitch_b + ((lane % 8) ^ ((row >> 1) & 7)) * 16;
  }
  const int total = g.steps * M::kSegments;
  const int first = static_cast<int>(static_cast<int64_t>(total) * at.split / g.splits);
  const int last = static_cast<int>(static_cast<int64_t>(total) * (at.split + 1) / g.splits);
  const int per_tile = last - first, n = per_tile * tiles;
  // Where the next loads of an operand come from and go to: its part (segment 0 is hi * lo, 1 is lo * hi, 2 or the only one
  // hi * hi), step and tile, with the address and the bytes in range (the rows that are there, of each the line of this
  // step) kept up to date.  Past the last step nothing is in range, so that the loop has no branches around its loads and
  // always the same number of them under way.
  struct Cursor {
    const uint16_t *p;
    uint32_t bytes;
    int seg, slot, left, tile_left, until;  // until: steps before p has to be taken anew
  };
  const int first_seg = first / g.steps, first_step = first - first_seg * g.steps;
  int64_t m_a = m0;  // first row of the tile that cursor a is in
  auto begin = [&](Cursor &c, const GemmOperand &o, int64_t row, int rows, int step, int hi_segment, auto turned) {
    c.p = o.p + (M::kSegments == 3 && c.seg == hi_segment ? o.part : 0) + row * o.row + step * o.step;
    const uint32_t there = static_cast<uint32_t>(min<int64_t>(rows, o.rows - row));
    if constexpr (decltype(turned)::value)
      c.bytes = ((there + kStepK - 1) / kStepK - 1) * (static_cast<uint32_t>(o.row) * (kStepK * 2)) + kStepK * kStepK * 2;
    else
      c.bytes = (there - 1) * static_cast<uint32_t>(o.row * 2) + (kNative && step == g.steps - 1 ? g.tail : kStepK) * 2;
    c.until = min(kNative && step < g.steps - 1 ? g.steps - 1 - step : g.steps - step, c.tile_left);
  };
  auto advance = [&](Cursor &c, const GemmOperand &o, int64_t &row, int rows, int stride, int hi_segment, int stages, auto turned) {
    if (++c.slot == stages) c.slot = 0;
    c.p += o.step;
    --c.tile_left;
    if (--c.left <= 0) {
      c.bytes = 0;
    } else if (--c.until == 0) {
      int step = kNative ? g.steps - 1 : 0;  // native: the last step, whose rows may end early
      if (!kNative) ++c.seg;
      if (c.tile_left == 0) {
        c.tile_left = per_tile;
        c.seg = first_seg;
        step = first_step;
        row += stride;
      }
      begin(c, o, row, rows, step, hi_segment, turned);
    }
  };
  Cursor ca{nullptr, 0, first_seg, 0, n, per_tile, 0}, cb = ca;
  using TurnA = std::integral_constant<bool, kTurnA>;
  int64_t m_b = n0;
  begin(ca, g.a, m_a, Tile::BM, first_step, 1, TurnA{});
  begin(cb, g.b, m_b, Tile::BN, first_step, 0, std::false_type{});
  auto advance_a = [&]() { advance(ca, g.a, m_a, Tile::BM, Tile::BM, 1, Tile::kStagesA, TurnA{}); };
  auto advance_b = [&]() { advance(cb, g.b, m_b, Tile::BN, 0, 0, 2, std::false_type{}); };
  uint16_t *const lds_b = lds + Tile::kStagesA * Tile::kStageA;
  auto load_a = [&](int j) {
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t *>(ca.p), 0, ca.bytes, 0x00020000);
    uint16_t *to = lds + ca.slot * Tile::kStageA + (wave + j * Tile::kWaves) * 8 * kStepK;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (LdsPtr)to, 16, off_a[j], 0, 0, 0);
  };
  auto load_b = [&](int j) {
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t *>(cb.p), 0, cb.bytes, 0x00020000);
    uint16_t *to = lds_b + cb.slot * Tile::kStageB + (wave + j * Tile::kWaves) * 8 * kStepK;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (LdsPtr)to, 16, off_b[j], 0, 0, 0);
  };
  // One period of loads, from one meeting of the waves to the next: B's next step, then A's next (the one after, where A
  // has three stages).  They are issued a few at a time between the matrix instructions of the period's first kQuarters
  // quarters: all at once they would fill the queue and hold the waves up.
  constexpr bool kDeep = Tile::kStagesA == 3;
  constexpr int kQuarters = kDeep ? 4 : 2, kPerQuarter = (kLoads + kQuarters - 1) / kQuarters;
  auto load_one = [&](int l) {
    if (l < Tile::kLoadsB) load_b(l);
    else if (l < kLoads) load_a(l - Tile::kLoadsB);
    if (l == Tile::kLoadsB - 1) advance_b();
    if (l == kLoads - 1) advance_a();
  };

  // fragments: lane l holds row l % 32, eight k from 16 * quarter + 8 * (l / 32) on
  const int row_a = wm * (Tile::BM / Tile::WM) + lane % 32, row_b = wn * (Tile::BN / Tile::WN) + lane % 32;
  const int at_a = row_a * kStepK, at_b = row_b * kStepK;
  const int twist = (lane >> 1) & 7;
  // turned: k lines 16 * quarter + 8 * (l / 32) on, rows TM * (l % 32) on
  static_assert(Tile::TM == 2 || Tile::TM == 4, "a turned row group is one or two words");
  typedef uint32_t Rows __attribute__((ext_vector_type(Tile::TM / 2)));
  const int at_turned = 8 * (lane / 32) * Tile::BM + wm * (Tile::BM / Tile::WM) + lane % 32 * Tile::TM;
  struct Fragments {
    bf16x8 a[kTurnA ? 1 : Tile::TM], b[Tile::TN];
    Rows lines[kTurnA ? 8 : 1];
  };
  int slot_a = 0, slot_b = 0;  // of the step that is read
  int left_in_tile = per_tile;  // steps from it to the tile's end
  auto read = [&](Fragments &f, int quarter) {
    const int piece = ((2 * quarter + lane / 32) ^ twist) * 8;
    const uint16_t *sb = lds_b + slot_b * Tile::kStageB + at_b + piece;
    if constexpr (kTurnA) {
      const uint16_t *sa = lds + slot_a * Tile::kStageA + quarter * 16 * Tile::BM + at_turned;
#pragma unroll
      for (int k = 0; k < 8; ++k) f.lines[k] = *reinterpret_cast<const Rows *>(sa + k * Tile::BM);
    } else {
      const uint16_t *sa = lds + slot_a * Tile::kStageA + at_a + piece;
#pragma unroll
      for (int t = 0; t < Tile::TM; ++t) f.a[t] = *reinterpret_cast<const bf16x8 *>(sa + t * 32 * kStepK);
    }
#pragma unroll
    for (int t = 0; t < Tile::TN; ++t) f.b[t] = *reinterpret_cast<const bf16x8 *>(sb + t * 32 * kStepK);
    if constexpr (kNative) {
      if (left_in_tile == 1 && g.tail < kStepK) {  // what lies behind the rows' ends belongs to the next rows
        typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
        const int first_k = (2 * quarter + lane / 32) * 4, end_k = g.tail / 2;
        auto cut = [&](bf16x8 &x) {
          u32x4 w = __builtin_bit_cast(u32x4, x);
#pragma unroll
          for (int k = 0; k < 4; ++k) w[k] = first_k + k < end_k ? w[k] : 0;
          x = __builtin_bit_cast(bf16x8, w);
        };
#pragma unroll
        for (int t = 0; t < Tile::TM; ++t) cut(f.a[t]);
#pragma unroll
        for (int t = 0; t < Tile::TN; ++t) cut(f.b[t]);
      }
    }
  };
  // kQuarter of the period, whose share of the loads goes out between the products
  auto multiply = [&](const Fragments &f, auto quarter) {
    constexpr int kQuarter = decltype(quarter)::value, kProducts = Tile::TM * Tile::TN;
    constexpr int kShare = kQuarter < kQuarters ? kPerQuarter : 0;
    __builtin_amdgcn_sched_barrier(0);  // the reads before it are under way
    bf16x8 row;
#pragma unroll
    for (int p = 0; p < kProducts; ++p) {
      const int t = p / Tile::TN, u = p % Tile::TN;
      if constexpr (kTurnA) {
        if (u == 0) {
          typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
          u32x4 w;
#pragma unroll
          for (int k = 0; k < 4; ++k)
            w[k] = __builtin_amdgcn_perm(f.lines[2 * k + 1][t / 2], f.lines[2 * k][t / 2], t % 2 ? 0x07060302u : 0x05040100u);
          row = __builtin_bit_cast(bf16x8, w);
        }
      } else {
        row = f.a[t];
      }
      acc.c[t][u] = M::mfma(row, f.b[u], acc.c[t][u]);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int l = kShare * p / kProducts; l < kShare * (p + 1) / kProducts; ++l) load_one(kQuarter * kPerQuarter + l);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  auto lower = [&]() {
#pragma unroll
    for (int t = 0; t < Tile::TM; ++t)
#pragma unroll
      for (int u = 0; u < Tile::TN; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc.c[t][u][r] *= 1.0f / (1 << kLowBits);
  };

  using Q0 = std::integral_constant<int, 0>;
  using Q1 = std::integral_constant<int, 1>;
  using Q2 = std::integral_constant<int, 2>;
  using Q3 = std::integral_constant<int, 3>;
  const int cross = M::kSegments == 3 ? 2 * g.steps - first : 0;  // steps of this share before hi * hi begins
  Fragments f0, f1;
#pragma unroll
  for (int j = 0; j < Tile::kLoadsA; ++j) load_a(j);
  advance_a();
#pragma unroll
  for (int j = 0; j < Tile::kLoadsB; ++j) load_b(j);
  advance_b();
  if constexpr (kDeep) {
#pragma unroll
    for (int j = 0; j < Tile::kLoadsA; ++j) load_a(j);
    advance_a();
  }
#pragma unroll
  for (int l = 0; l < kPerQuarter; ++l) load_one(l);
  arrive_and_meet<kPerQuarter + (kDeep ? Tile::kLoadsA : 0)>();
  read(f0, 0);
  int tile = 0;
  for (int i = 0, in_tile = 0; i < n; ++i) {
    if (M::kSegments == 3 && in_tile > 0 && in_tile == cross) lower();
    read(f1, 1);
    multiply(f0, Q1{});
    read(f0, 2);
    multiply(f1, Q2{});
    read(f1, 3);
    multiply(f0, Q3{});
    // the next step is there for every wave (only A's step after it may still be on its way), nobody reads this one
    arrive_and_meet<kDeep ? Tile::kLoadsA : 0>();
    if (++slot_a == Tile::kStagesA) slot_a = 0;
    slot_b ^= 1;
    if (--left_in_tile == 0) left_in_tile = per_tile;
    read(f0, 0);  // past the last step: what is read is not used
    multiply(f1, Q0{});
    if (++in_tile == per_tile) {
      if (M::kSegments == 3 && cross >= per_tile) lower();
      done(tile);
      in_tile = 0;
      ++tile;
    }
  }
  arrive_and_meet<0>();  // the LDS may be used for other things
#endif
}

// One tile, left in acc.
template <typename Tile, typename T, bool kTurnA = false>
__device__ __forceinline__ void gemm_tile(const GemmShape &g, const GemmPlace &at, uint16_t *lds, GemmAcc<Tile> &acc) {
  gemm_tiles<Tile, Multiply<T>, kTurnA>(g, at, 1, lds, acc, [](int) {});
}

}  // namespace fg
