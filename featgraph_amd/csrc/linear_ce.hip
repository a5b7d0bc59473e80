// Softmax cross entropy of a linear scorer, without keeping the logits, and its gradients:
//
//   l[n, v]  = <h[n], w[v]>                    lse[n] = log sum over v of exp l[n, v]
//   loss[n]  = lse[n] - l[n, y[n]]             (0 where the label y[n] is outside [0, V): the row is ignored)
//   P[n, v]  = exp(l[n, v] - lse[n]) - [v = y[n]]          (0 for an ignored row)
//   dh[n]    = dloss[n] * sum over v of P[n, v] w[v]       dw[v] = sum over n of P[n, v] dloss[n] h[n]
//
// Forward: one matrix product whose epilogue keeps, per row n and range of the vocabulary, the largest logit and the sum
// of exponentials relative to it, and picks the label's logit out where it meets it; a second kernel joins the ranges.
// Backward: the logits are computed again piece by piece of the vocabulary; the epilogue turns them into P, and two
// more products over P give the piece's rows of dw and its share of dh.  P is stored once, as [v, n]: dw's product reads
// its rows, dh's its columns (mfma_gemm.hpp).  h and w are transposed into copies for these products (2 N D + 2 V D
// elements of traffic against 6 N V D flops), bfloat16 rows that have to be padded in the same pass (19 rows x 137,737 classes
// x 89: 103 -> 76 us); the copy of h also holds zeros in place of the rows to ignore.
//
// Where it stands (bfloat16), whole calls: 4096 rows x 65,536 classes x 1024: loss 446 us (1233 TFLOP/s), gradient 1495 (its
// three products: 1103); a library's product of 8192^3 reaches 1333.  1024 x 232,965 x 128: 89 to 100 and 447, bound by the
// epilogues: an exponential per logit, P written once and read twice.
//
// Types: bfloat16 operands are used as they are; P is stored times dloss, rounded to bfloat16 (half a step, 2^-8, of each
// term: the matrix instructions take no wider type, two parts would double both products, and the results are rounded to
// bfloat16 themselves); everything between is float32.  float32
// operands, P among them, are split into two float16 parts (mfma_gemm.hpp); the loss multiplies them as they are where
// reading one of them bounds it (few rows, or few classes).  P is at most 1 and stored times 2^14; dloss is applied to the
// rows of dh in the epilogue and to the copy of h for dw.  What the parts keep: x of a row (logits) or of a whole matrix
// (transposed copies) with the largest element m to 2^-23 |x| + 2^-50 m, P to 2^-23 P + 2^-50; sums are rounded as if
// every factor were at least 2^-28 of the largest.  Smaller probabilities and features than 2^-27 of the largest so lose
// relative accuracy; a third part would keep them at twice the products.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "mfma_gemm.hpp"

namespace fg {
namespace {

// Keeps the compiler from moving the work of one block of accumulators into another's, which costs registers.
#if defined(__HIP_DEVICE_COMPILE__)
#define FG_IN_ORDER() __builtin_amdgcn_sched_barrier(0)
// ... and fixes the point at which x is computed.
#define FG_HERE(x) asm volatile("" : "+v"(x))
#else
#define FG_IN_ORDER()
#define FG_HERE(x)
#endif

constexpr float kLog2e = 1.44269504088896340736f;
constexpr int kTop = 14;  // binary exponent that a scaled float32 operand's largest element is brought to

using Big = GemmTile<256, 256, 2, 4, 3>;   // 128 x 64 per wave, one workgroup per CU
using Mid = GemmTile<128, 128, 2, 2, 3>;   // 64 x 64 per wave, two workgroups per CU
using Flat = GemmTile<64, 256, 1, 4, 2>;   // few rows of A
using Tall = GemmTile<256, 64, 4, 1, 2>;   // few rows of B

// ------------------------------------------------------------------------------------------------ operand copies
__device__ __forceinline__ uint32_t bits_of(float x) { return __builtin_bit_cast(uint16_t, narrow<__bf16>(x)); }
__device__ __forceinline__ uint32_t half_bits(float x) { return __builtin_bit_cast(uint16_t, narrow<_Float16>(x)); }

// Part `part` of x, whose exponent has been brought into float16's range.  What is not finite has no second part, so
// that it does not turn into NaN by inf - inf.
template <typename T>
__device__ __forceinline__ uint32_t part_of(float x, int part) {
  if constexpr (sizeof(T) == 2) {
    return bits_of(x);
  } else {
    const _Float16 hi = narrow<_Float16>(x);
    if (part == 0) return __builtin_bit_cast(uint16_t, hi);
    const float rest = x - widen(hi);
    return half_bits(__builtin_fabsf(x) < INFINITY ? rest * (1 << kLowBits) : 0.0f);
  }
}

// The exponent that brings a largest element (as float bits) to 2^kTop; 0 when there is none.
__device__ __forceinline__ int exponent_for(uint32_t peak) {
  if (peak == 0) return 0;
  return min(126, max(-126, kTop - (static_cast<int>(peak >> 23) - 127)));
}

// The largest element of a matrix is collected in kPeakSlots words of lines of their own, by workgroup: one word would
// serialise the workgroups.
constexpr int kPeakSlots = 64, kPeakStride = 32;
__device__ __forceinline__ uint32_t read_peak(const uint32_t *peak) {
  uint32_t m = peak[(threadIdx.x & (kPeakSlots - 1)) * kPeakStride];
#pragma unroll
  for (int d = 1; d < kWaveSize; d <<= 1) m = max(m, static_cast<uint32_t>(__shfl_xor(static_cast<int>(m), d, kWaveSize)));
  return m;
}

__device__ __forceinline__ uint32_t finite_bits(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x) & 0x7fffffffu;
  return u < 0x7f800000u ? u : 0u;
}

// One matrix to copy for the products; a launch takes two (h and a piece of w), either of which may have no blocks.
struct CopyJob {
  const void *x;            // [rows, D]
  uint16_t *out;
  int64_t rows;
  int32_t D;
  uint32_t blocks;          // of the launch
  int32_t *exps;            // float32, row copy: exponents of the rows
  uint32_t *peak;           // float32: the largest |x| * |factor[row]| of the rows that are kept; written by the row copy
                            // (null: not wanted), read by the transposed copy
  const int32_t *keep;      // rows whose keep[] is negative do not count in peak, and are zeros in the transposed copy
  const float *factor;      // float32: per row, for peak and the transposed copy (null: 1)
  uint16_t *rows_out;       // bfloat16, transposed copy: where the row copy goes, made in the same pass (null: not wanted)
};
struct CopyJobs {
  CopyJob job[2];
};
// This block's job and its number in it.
__device__ __forceinline__ const CopyJob &job_of(const CopyJobs &jobs, uint32_t *block) {
  const bool second = blockIdx.x >= jobs.job[0].blocks;
  *block = second ? blockIdx.x - jobs.job[0].blocks : blockIdx.x;
  return jobs.job[second];
}

// kVec elements from any address of theirs on; past the row's end zeros.
template <typename T, int kVec>
__device__ __forceinline__ Pack<T, kVec> load_within(const T *row, int64_t c, int32_t D) {
  Pack<T, kVec> v;
  if (c + kVec <= D) {
    __builtin_memcpy(&v, row + c, sizeof(v));
  } else {
#pragma unroll
    for (int j = 0; j < kVec; ++j) v.v[j] = c + j < D ? row[c + j] : T{};
  }
  return v;
}

// bfloat16: [rows, D] -> panels, eight elements per lane
__device__ __forceinline__ void pad_rows(const CopyJob &job, uint32_t block) {
  constexpr int kPieces = kStepK / 8;  // of a row in a panel
  const auto *x = static_cast<const uint16_t *>(job.x);
  const int64_t per_panel = job.rows * kPieces;
  const int64_t total = per_panel * ((job.D + kStepK - 1) / kStepK), stride = static_cast<int64_t>(job.blocks) * kBlockThreads;
  for (int64_t t = static_cast<int64_t>(block) * kBlockThreads + threadIdx.x; t < total; t += stride) {
    const int64_t panel = t / per_panel, in_panel = t - panel * per_panel;
    *reinterpret_cast<Pack<uint16_t, 8> *>(job.out + t * 8) =
        load_within<uint16_t, 8>(x + in_panel / kPieces * job.D, panel * kStepK + in_panel % kPieces * 8, job.D);
  }
}

// float32: [rows, D] -> two parts as panels, each row by its own exponent.  One wave per row; rows of up to 64 * kHeld
// elements stay in registers between the search for the largest and the split, and the next row is under way meanwhile
// (161,783 rows of 332: 187 -> 83 us).
template <int kHeld>
__device__ __forceinline__ void split_rows(const CopyJob &job, uint32_t block) {
  __shared__ uint32_t peaks[kWavesPerBlock];
  const auto *x = static_cast<const float *>(job.x);
  const int lane = threadIdx.x & (kWaveSize - 1), wave = threadIdx.x / kWaveSize;
  const int32_t D = job.D, padded = (D + kStepK - 1) / kStepK * kStepK;
  const int64_t part = job.rows * padded, stride = static_cast<int64_t>(job.blocks) * kWavesPerBlock;
  uint32_t most = 0;
  constexpr int kRegs = kHeld > 0 ? kHeld : 1;
  float held[kRegs], ahead[kRegs];
  auto fetch = [&](int64_t r, float *to) {
#pragma unroll
    for (int u = 0; u < kHeld; ++u) to[u] = r < job.rows && u * kWaveSize + lane < D ? x[r * D + u * kWaveSize + lane] : 0.0f;
  };
  auto put = [&](int64_t r, int32_t c, float y) {
    const int64_t to = panel_at(job.rows, r, c);
    job.out[to] = static_cast<uint16_t>(part_of<float>(y, 0));
    job.out[part + to] = static_cast<uint16_t>(part_of<float>(y, 1));
  };
  int64_t r = static_cast<int64_t>(block) * kWavesPerBlock + wave;
  fetch(r, held);
  for (; r < job.rows; r += stride) {
    fetch(r + stride, ahead);
    uint32_t top = 0;
    if constexpr (kHeld > 0) {
#pragma unroll
      for (int u = 0; u < kHeld; ++u) top = max(top, finite_bits(held[u]));
    } else {
      for (int32_t c = lane; c < D; c += kWaveSize) top = max(top, finite_bits(x[r * D + c]));
    }
#pragma unroll
    for (int d = 1; d < kWaveSize; d <<= 1) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), d, kWaveSize)));
    const int e = exponent_for(top);
    if (lane == 0) job.exps[r] = e;
    if constexpr (kHeld > 0) {
#pragma unroll
      for (int u = 0; u < kHeld; ++u)
        if (u * kWaveSize < padded) put(r, u * kWaveSize + lane, __builtin_ldexpf(held[u], e));
    } else {
      for (int32_t c = lane; c < padded; c += kWaveSize) put(r, c, c < D ? __builtin_ldexpf(x[r * D + c], e) : 0.0f);
    }
    if (job.peak && (!job.keep || job.keep[r] >= 0))
      most = max(most, finite_bits(__builtin_bit_cast(float, top) * (job.factor ? job.factor[r] : 1.0f)));
#pragma unroll
    for (int u = 0; u < kHeld; ++u) held[u] = ahead[u];
  }
  if (!job.peak) return;
  if (lane == 0) peaks[wave] = most;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kWavesPerBlock; ++w) most = max(most, peaks[w]);
    atomicMax(job.peak + block % kPeakSlots * kPeakStride, most);  // a largest value does not depend on the order
  }
}

template <typename T, int kHeld>
__global__ __launch_bounds__(kBlockThreads) void copy_rows_kernel(CopyJobs jobs) {
  uint32_t block;
  const CopyJob &job = job_of(jobs, &block);
  if constexpr (sizeof(T) == 4) split_rows<kHeld>(job, block);
  else pad_rows(job, block);
}

// [rows, D] -> parts of its transpose as panels of 64 rows' elements, zeros in place of rows whose keep[] is negative
// (whatever those hold must not reach the sum over rows).  float32: times factor[row] and brought into range by *peak.
// 64 x 64 elements per workgroup, 16 bytes per lane on both sides.
template <typename T>
__global__ __launch_bounds__(kBlockThreads) void copy_transposed_kernel(CopyJobs jobs) {
  constexpr int kVec = 16 / sizeof(T), kLanes = 64 / kVec;  // per row
  __shared__ float tile[64][65];
  uint32_t block;
  const CopyJob &job = job_of(jobs, &block);
  const int64_t panels = (job.rows + kStepK - 1) / kStepK, panel = block % panels;
  const int64_t r0 = panel * kStepK;
  const int32_t D = job.D;
  const int c0 = static_cast<int>(block / panels) * 64;
  const int e = sizeof(T) == 4 ? exponent_for(read_peak(job.peak)) : 0;
  const int c = c0 + threadIdx.x % kLanes * kVec;
  for (int k = threadIdx.x / kLanes; k < 64; k += kBlockThreads / kLanes) {
    const int64_t r = r0 + k;
    Pack<T, kVec> v;
    const bool there = r < job.rows && (!job.keep || job.keep[r] >= 0);
    if (there) v = load_within<T, kVec>(static_cast<const T *>(job.x) + r * D, c, D);
    const float f = sizeof(T) == 4 && there && job.factor ? job.factor[r] : 1.0f;
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
      float y = there ? widen(v.v[j]) : 0.0f;
      if constexpr (sizeof(T) == 4) y = there ? __builtin_ldexpf(y * f, e) : 0.0f;
      tile[k][threadIdx.x % kLanes * kVec + j] = y;
    }
  }
  __syncthreads();
  for (int t = threadIdx.x; t < 512; t += kBlockThreads) {  // eight rows of one column each
    const int g = t % 8, col = t / 8;
    if (c0 + col >= D) continue;
#pragma unroll
    for (int p = 0; p < Multiply<T>::kParts; ++p) {
      Pack<uint16_t, 8> y;
#pragma unroll
      for (int k = 0; k < 8; ++k) y.v[k] = static_cast<uint16_t>(part_of<T>(tile[8 * g + k][col], p));
      *reinterpret_cast<Pack<uint16_t, 8> *>(job.out + ((panel + p * panels) * D + c0 + col) * kStepK + 8 * g) = y;
    }
  }
  if constexpr (sizeof(T) == 2) {
    if (job.rows_out == nullptr) return;
    for (int t = threadIdx.x; t < 512; t += kBlockThreads) {  // eight columns of one row each
      const int g = t % 8, k = t / 8;
      if (r0 + k >= job.rows) continue;
      Pack<uint16_t, 8> y;
#pragma unroll
      for (int j = 0; j < 8; ++j) y.v[j] = static_cast<uint16_t>(bits_of(tile[k][8 * g + j]));
      *reinterpret_cast<Pack<uint16_t, 8> *>(job.rows_out + panel_at(job.rows, r0 + k, c0 + 8 * g)) = y;
    }
  }
}

// Labels as int32, -1 for rows to ignore; clears the words that collect the largest elements.
template <typename Id>
__global__ __launch_bounds__(kBlockThreads) void labels_kernel(const Id *labels, int32_t n, int64_t V, int32_t *out,
                                                               uint32_t *peaks, int32_t n_peaks) {
  const int i = blockIdx.x * kBlockThreads + threadIdx.x;
  if (i < n) {
    const Id y = labels[i];
    out[i] = y >= 0 && static_cast<int64_t>(y) < V ? static_cast<int32_t>(y) : -1;
  }
  for (int k = i; k < n_peaks; k += gridDim.x * kBlockThreads) peaks[k] = 0;
}

// ------------------------------------------------------------------------------------------------ forward
// Statistics of a set of logits: {r, s} with s = sum of exp(l) / 2^r, r a whole number at or just above the largest
// logit / ln 2.  A whole r is exact, so exp2(l * log2(e) - r) is one multiply-add, rounded once, near the terms that count.
struct StatsArgs {
  GemmShape g;             // a: rows of w, b: h
  const int32_t *exp_a, *exp_b;  // float32: exponents of the rows
  float2 *part;            // [ranges of vocabulary, N]
  int32_t ranges;          // that the tiles of vocabulary of this piece are divided into
  int32_t range0;          // first of them
  const void *labels;      // [N]
  int64_t v0;              // first vocabulary row of this piece
  float *label_logit;      // [N], written where the label's row is met
};

__device__ __forceinline__ float2 join_stats(float2 a, float2 b) {
  const float r = fmaxf(a.x, b.x);
  if (r == -INFINITY) return float2{r, a.y + b.y};
  return float2{r, a.y * __builtin_amdgcn_exp2f(a.x - r) + b.y * __builtin_amdgcn_exp2f(b.x - r)};
}

// Takes the rows' exponents back out of the accumulators: what is left are the logits.
template <typename Tile, typename T>
__device__ __forceinline__ void to_logits(GemmAcc<Tile> &acc, const int32_t *exp_a, const int32_t *exp_b, int64_t v0,
                                          int64_t n0, int32_t N, int lane) {
  if constexpr (sizeof(T) == 4) {
    int en[Tile::TN];
#pragma unroll
    for (int j = 0; j < Tile::TN; ++j) {
      const int64_t n = n0 + 32 * j + lane % 32;
      en[j] = n < N ? exp_b[n] : 0;
    }
#pragma unroll
    for (int i = 0; i < Tile::TM; ++i) {
      FG_IN_ORDER();
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int4 ev = *reinterpret_cast<const int4 *>(exp_a + v0 + 32 * i + acc_row(4 * q, lane));
#pragma unroll
        for (int j = 0; j < Tile::TN; ++j) {
          const int en_ev[4] = {en[j] + ev.x, en[j] + ev.y, en[j] + ev.z, en[j] + ev.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            float x = __builtin_ldexpf(acc.c[i][j][4 * q + k], -en_ev[k]);
            FG_HERE(x);  // done here, so that the exponents' registers are free again
            acc.c[i][j][4 * q + k] = x;
          }
        }
      }
    }
  }
}

// First tile of a workgroup that takes one tile of rows n and a range of the vocabulary, and how many follow each other.
__device__ __forceinline__ GemmPlace range_place(const GemmShape &g, int ranges, int *range, int *tiles) {
  GemmShape places = g;
  places.tiles_m = ranges;
  GemmPlace at = gemm_place(places);
  *range = at.tm;
  at.tm = static_cast<int32_t>(static_cast<int64_t>(g.tiles_m) * *range / ranges);
  *tiles = static_cast<int>(static_cast<int64_t>(g.tiles_m) * (*range + 1) / ranges) - at.tm;
  return at;
}

// A workgroup takes one tile of rows n and a range of the vocabulary, tile after tile without a pause in its loads; each
// lane keeps the statistics of the logits it meets (its column n, half the rows of its wave) until the end.
template <typename Tile, typename T, typename M, typename Id>
__global__ __launch_bounds__(Tile::kThreads) void stats_kernel(StatsArgs a) {
  __shared__ __attribute__((aligned(1024))) uint16_t lds[Tile::kLds];
  GemmAcc<Tile> acc;
  int range, tiles;
  const GemmPlace at = range_place(a.g, a.ranges, &range, &tiles);
  const int lane = threadIdx.x & (kWaveSize - 1), wave = threadIdx.x / kWaveSize;
  const int wm = wave / Tile::WN, wn = wave % Tile::WN;
  const int64_t n0 = static_cast<int64_t>(at.tn) * Tile::BN + wn * (Tile::BN / Tile::WN);
  const int64_t first_v = static_cast<int64_t>(at.tm) * Tile::BM + wm * (Tile::BM / Tile::WM);
  float top[Tile::TN], sum[Tile::TN], rest[Tile::TN];  // the sum is sum + rest
  int64_t label[Tile::TN];  // row of the piece that is the label's, relative to this wave's first
#pragma unroll
  for (int j = 0; j < Tile::TN; ++j) {
    const int64_t n = n0 + 32 * j + lane % 32;
    top[j] = -INFINITY;
    sum[j] = rest[j] = 0.0f;
    label[j] = n < a.g.b.rows ? static_cast<int64_t>(static_cast<const Id *>(a.labels)[n]) - a.v0 - first_v : -1;
  }
  gemm_tiles<Tile, M, false>(a.g, at, tiles, lds, acc, [&](int tile) {
    const int64_t v0 = first_v + static_cast<int64_t>(tile) * Tile::BM;
    if constexpr (M::kSegments > 1) to_logits<Tile, T>(acc, a.exp_a, a.exp_b, v0, n0, a.g.b.rows, lane);
#pragma unroll
    for (int j = 0; j < Tile::TN; ++j) {
      if (v0 + Tile::BM / Tile::WM > a.g.a.rows) {
        const int end = static_cast<int>(max<int64_t>(a.g.a.rows - v0, 0)) - acc_row(0, lane);
#pragma unroll
        for (int i = 0; i < Tile::TM; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (32 * i + acc_row(r, 0) >= end) acc.c[i][j][r] = -INFINITY;
      }
      const int64_t past = label[j] - static_cast<int64_t>(tile) * Tile::BM;
      const int hit = past >= 0 && past < Tile::BM / Tile::WM && v0 + past < a.g.a.rows ? static_cast<int>(past) : -1;
      if (__any(hit >= 0)) {
        float logit = 0.0f;
        const int mine = hit - acc_row(0, lane);
#pragma unroll
        for (int i = 0; i < Tile::TM; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r) logit = 32 * i + acc_row(r, 0) == mine ? acc.c[i][j][r] : logit;
        if (hit >= 0 && hit / 4 % 2 == lane / 32) a.label_logit[n0 + 32 * j + lane % 32] = logit;
      }
      float m = -INFINITY;
#pragma unroll
      for (int i = 0; i < Tile::TM; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) m = fmaxf(m, acc.c[i][j][r]);
      m = fmaxf(top[j], __builtin_ceilf(m * kLog2e));
      const float from = m == -INFINITY ? 0.0f : m;
      // The tile's terms: 16 one by one, then the sums of 16.
      float s = 0.0f;
#pragma unroll
      for (int i = 0; i < Tile::TM; ++i) {
        float t = 0.0f;
#pragma unroll
        for (int r = 0; r < 16; ++r) t += __builtin_amdgcn_exp2f(__builtin_fmaf(acc.c[i][j][r], kLog2e, -from));
        s += t;
      }
      // Added to the sum of the tiles before, what the addition rounds off to the rest: a range may have thousands of
      // tiles, each of them small against the sum.
      const float times = __builtin_amdgcn_exp2f(top[j] - from), old = sum[j] * times;
      sum[j] = old + s;
      const float added = sum[j] - old;
      rest[j] = rest[j] * times + ((old - (sum[j] - added)) + (s - added));
      top[j] = m;
    }
    clear(acc);
  });
  float2 *stats = reinterpret_cast<float2 *>(lds);  // [WM][BN]
#pragma unroll
  for (int j = 0; j < Tile::TN; ++j) {
    sum[j] += rest[j];
    const float2 s = join_stats(float2{top[j], sum[j]},
                                float2{__shfl_xor(top[j], 32, kWaveSize), __shfl_xor(sum[j], 32, kWaveSize)});
    if (lane < 32) stats[wm * Tile::BN + wn * (Tile::BN / Tile::WN) + 32 * j + lane] = s;
  }
  __syncthreads();
  for (int c = threadIdx.x; c < Tile::BN; c += Tile::kThreads) {
    const int64_t n = static_cast<int64_t>(at.tn) * Tile::BN + c;
    if (n >= a.g.b.rows) continue;
    float2 s = stats[c];
#pragma unroll
    for (int w = 1; w < Tile::WM; ++w) s = join_stats(s, stats[w * Tile::BN + c]);
    a.part[(static_cast<int64_t>(a.range0) + range) * a.g.b.rows + n] = s;
  }
}

// kShares threads per row share its ranges, whose sums are added in double.  `loss` holds the label's logits on entry.
constexpr int kFewRanges = 8;
template <typename Id, int kShares>
__global__ __launch_bounds__(kBlockThreads) void loss_kernel(const float2 *part, int32_t ranges, const Id *labels,
                                                             int32_t N, int64_t V, float *loss, float *lse) {
  constexpr int kRows = kBlockThreads / kShares;
  struct Sum {
    double s;
    float r;  // whole, of s * 2^r
  };
  auto join = [](const Sum &a, const Sum &b) {
    const float r = fmaxf(a.r, b.r);
    if (r == -INFINITY) return Sum{a.s + b.s, r};
    auto down = [r](const Sum &x) { return ldexp(x.s, static_cast<int>(fmaxf(x.r - r, -2000.0f))); };  // 0 beyond 2^-1074
    return Sum{down(a) + down(b), r};
  };
  __shared__ Sum joined[kShares][kRows];
  const int row = threadIdx.x % kRows, share = threadIdx.x / kRows;
  const int64_t n = static_cast<int64_t>(blockIdx.x) * kRows + row;
  Sum s{0.0, -INFINITY};
  if (n < N)
    for (int32_t t = share; t < ranges; t += kShares) {
      const float2 x = part[static_cast<int64_t>(t) * N + n];
      s = join(s, Sum{x.y, x.x});
    }
  if constexpr (kShares > 1) {
    joined[share][row] = s;
#pragma unroll
    for (int half = kShares / 2; half > 0; half >>= 1) {
      __syncthreads();
      if (share < half) joined[share][row] = s = join(s, joined[share + half][row]);
    }
  }
  if (share == 0 && n < N) {
    const float r = static_cast<float>((static_cast<double>(s.r) + log2(s.s)) * 0.69314718055994530942);
    const Id y = labels[n];
    lse[n] = r;
    loss[n] = y >= 0 && static_cast<int64_t>(y) < V ? r - loss[n] : 0.0f;
  }
}

// ------------------------------------------------------------------------------------------------ backward
// Four lanes that hold the same four rows of four neighbouring columns, two 16-bit elements per word (rows 0, 1 in a,
// rows 2, 3 in b), turn them: afterwards lane q of the four holds row q, its four columns in a (0, 1) and b (2, 3).
__device__ __forceinline__ uint2 turn4(uint2 x, int lane) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int kSwap1 = 0xB1, kSwap2 = 0x4E;  // quad permutations: lane ^ 1, lane ^ 2
  const uint32_t ta = __builtin_amdgcn_mov_dpp(x.x, kSwap1, 0xf, 0xf, true);
  const uint32_t tb = __builtin_amdgcn_mov_dpp(x.y, kSwap1, 0xf, 0xf, true);
  const uint32_t pick = lane & 1 ? 0x03020706u : 0x05040100u;  // even: own and other's low half; odd: the high halves
  const uint32_t a = __builtin_amdgcn_perm(ta, x.x, pick), b = __builtin_amdgcn_perm(tb, x.y, pick);
  const uint32_t got = __builtin_amdgcn_mov_dpp(lane & 2 ? a : b, kSwap2, 0xf, 0xf, true);
  return lane & 2 ? uint2{got, b} : uint2{a, got};
#else
  return x;
#endif
}

// After turn4 of the two blocks of a wave's 64 columns: neighbouring fours of lanes exchange halves, so that a lane holds
// eight neighbouring columns of its row and eight lanes a whole line, at columns line_column() on.  Stores of half lines
// cost the 232,965 x 256 gradient of 41 classes 60 us where whole lines take 55.
__device__ __forceinline__ uint4 line_of(uint2 first, uint2 second, int lane) {
#if defined(__HIP_DEVICE_COMPILE__)
  auto swap4 = [](uint32_t x) {  // lane ^ 4: fours 0 and 2 of a row take from above, 1 and 3 from below
    constexpr int kUp4 = 0x104, kDown4 = 0x114;  // from lane + 4, from lane - 4
    const int up = __builtin_amdgcn_update_dpp(0, static_cast<int>(x), kUp4, 0xf, 0x5, false);
    return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(up, static_cast<int>(x), kDown4, 0xf, 0xa, false));
  };
  const bool odd = lane & 4;
  const uint32_t x = swap4(odd ? first.x : second.x), y = swap4(odd ? first.y : second.y);
  return odd ? uint4{x, y, second.x, second.y} : uint4{first.x, first.y, x, y};
#else
  return uint4{first.x, first.y, second.x, second.y};
#endif
}
__device__ __forceinline__ int line_column(int lane) { return lane / 4 % 2 * 32 + lane % 32 / 8 * 8; }

struct GradArgs {
  GemmShape g;               // a: the piece's rows of w, b: h
  const int32_t *exp_a, *exp_b;
  const int32_t *label;      // [N], negative: ignored
  const float *lse, *dloss;  // [N]
  int32_t v0;                // first vocabulary row of the piece
  int32_t ranges;            // that the tiles of vocabulary are divided into
  uint16_t *vn;              // P as panels of [v, n], the rows of the piece padded to whole panels with zeros
  int64_t vn_part;           // elements from one part to the next
};

// T: type of the operands, which says how P is stored: straight from the registers, four n per lane.
template <typename Tile, typename T>
__global__ __launch_bounds__(Tile::kThreads) void grad_logits_kernel(GradArgs a) {
  __shared__ __attribute__((aligned(1024))) uint16_t lds[Tile::kLds];
  GemmAcc<Tile> acc;
  int range, tiles;
  const GemmPlace at = range_place(a.g, a.ranges, &range, &tiles);
  const int lane = threadIdx.x & (kWaveSize - 1), wave = threadIdx.x / kWaveSize;
  const int wm = wave / Tile::WN, wn = wave % Tile::WN;
  const int first_v = at.tm * Tile::BM + wm * (Tile::BM / Tile::WM);
  const int64_t n0 = static_cast<int64_t>(at.tn) * Tile::BN + wn * (Tile::BN / Tile::WN);
  // P = exp2(l * log2(e) - r) * 2^(r - lse * log2(e)) with a whole r: the first factor is one multiply-add, rounded once,
  // the second one is taken per row, in double, together with what P is stored times.
  int32_t label[Tile::TN];
  float whole_lse[Tile::TN], times[Tile::TN], scale[Tile::TN];
#pragma unroll
  for (int j = 0; j < Tile::TN; ++j) {
    const int64_t n = n0 + 32 * j + lane % 32;
    label[j] = n < a.g.b.rows ? a.label[n] : -1;
    times[j] = label[j] < 0 ? 0.0f : sizeof(T) == 4 ? static_cast<float>(1 << kTop) : a.dloss[n];
    const double lse2 = label[j] < 0 ? 0.0 : static_cast<double>(a.lse[n]) * 1.44269504088896340736;
    whole_lse[j] = static_cast<float>(rint(lse2));
    scale[j] = times[j] * __builtin_amdgcn_exp2f(static_cast<float>(static_cast<double>(whole_lse[j]) - lse2));
  }
  const int64_t M = a.g.a.rows, N = a.g.b.rows;
  const int64_t end_v = (M + kStepK - 1) / kStepK * kStepK, end_n = (N + kStepK - 1) / kStepK * kStepK;  // of the panels
  // the 16-bit form of the accumulator x; a float32's rest takes its place for the next part
  auto take = [](float &x) -> uint32_t {
    const uint32_t bits = part_of<T>(x, 0);
    if constexpr (sizeof(T) == 4) {
      x = (x - widen(__builtin_bit_cast(_Float16, static_cast<uint16_t>(bits)))) * (1 << kLowBits);
      FG_HERE(x);  // in x's place, not beside it
    }
    return bits;
  };
  gemm_tiles<Tile, Multiply<T>, false>(a.g, at, tiles, lds, acc, [&](int tile) {
    const int v0 = first_v + tile * Tile::BM;
    to_logits<Tile, T>(acc, a.exp_a, a.exp_b, v0, n0, a.g.b.rows, lane);
#pragma unroll
    for (int j = 0; j < Tile::TN; ++j) {
#pragma unroll
      for (int i = 0; i < Tile::TM; ++i)
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(acc.c[i][j][k], kLog2e, -whole_lse[j])) * scale[j];
          acc.c[i][j][k] = label[j] >= 0 ? p : 0.0f;
        }
      const int32_t hit = label[j] >= 0 ? label[j] - a.v0 - v0 : -1;  // row of this wave's block that is the label's
      if (__any(hit >= 0 && hit < Tile::BM / Tile::WM)) {
        const int mine = hit - acc_row(0, lane);
#pragma unroll
        for (int i = 0; i < Tile::TM; ++i)
#pragma unroll
          for (int k = 0; k < 16; ++k)
            if (32 * i + acc_row(k, 0) == mine) acc.c[i][j][k] -= times[j];
      }
      if (v0 + Tile::BM / Tile::WM > M) {  // nothing past the end
        const int end = max(static_cast<int>(M) - v0, 0) - acc_row(0, lane);
#pragma unroll
        for (int i = 0; i < Tile::TM; ++i)
#pragma unroll
          for (int k = 0; k < 16; ++k)
            if (32 * i + acc_row(k, 0) >= end) acc.c[i][j][k] = 0.0f;
      }
    }
    const bool whole = v0 + Tile::BM / Tile::WM <= M && n0 + Tile::BN / Tile::WN <= N;
    auto store = [&](auto inside, int part) {  // inside: the wave's whole block lies within the matrix
      constexpr bool kInside = decltype(inside)::value;
      static_assert(Tile::TN == 2, "a wave's columns are a line");
      const int64_t col = n0 + line_column(lane);
#pragma unroll
      for (int i = 0; i < Tile::TM; ++i) {
        FG_IN_ORDER();
        const int64_t row = v0 + 32 * i + acc_row(0, lane) + lane % 4;
        uint16_t *to = a.vn + part * a.vn_part + panel_at(end_v, row, col);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          uint2 x[2];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float e[4] = {acc.c[i][j][4 * q], acc.c[i][j][4 * q + 1], acc.c[i][j][4 * q + 2], acc.c[i][j][4 * q + 3]};
            x[j].x = take(e[0]);
            x[j].x |= take(e[1]) << 16;
            x[j].y = take(e[2]);
            x[j].y |= take(e[3]) << 16;
#pragma unroll
            for (int k = 0; k < 4; ++k) acc.c[i][j][4 * q + k] = e[k];
            x[j] = turn4(x[j], lane);
          }
          const uint4 y = line_of(x[0], x[1], lane);
          if (kInside || (row + 8 * q < end_v && col < end_n)) *reinterpret_cast<uint4 *>(to + 8 * q * kStepK) = y;
        }
      }
    };
#pragma unroll
    for (int part = 0; part < Multiply<T>::kParts; ++part) {
      if (sizeof(T) == 2 && whole) store(std::true_type{}, part);  // a second copy of the code costs float32 its registers
      else store(std::false_type{}, part);
    }
    clear(acc);
  });
}

struct StoreArgs {
  GemmShape g;
  void *out;               // [rows of a, rows of b] of T
  const int32_t *keep;     // rows of a to write as zeros where negative (null: none)
  const float *factor;     // float32: of the rows of a (null: 1)
  const uint32_t *peak;    // float32: what operand b was scaled by; a is P times 2^kTop
  float *part;             // or float32 sums of each split, [splits, part_stride], added to what is there
  int64_t part_stride;
  int32_t accumulate;
  int32_t wide;            // 16-bit out: elements per store that its alignment and the row length allow: 8, 4 or 0 (single ones)
};

// kPartial: the sums go to a.part for join_kernel, else rounded to a.out.  kTurnA: operand a is turned.
template <typename Tile, typename T, bool kPartial, bool kTurnA>
__global__ __launch_bounds__(Tile::kThreads) void product_kernel(StoreArgs a) {
  __shared__ __attribute__((aligned(1024))) uint16_t lds[Tile::kLds];
  GemmAcc<Tile> acc;
  const GemmPlace at = gemm_place(a.g);
  gemm_tile<Tile, T, kTurnA>(a.g, at, lds, acc);
  const int lane = threadIdx.x & (kWaveSize - 1), wave = threadIdx.x / kWaveSize;
  const int wm = wave / Tile::WN, wn = wave % Tile::WN;
  const int64_t m0 = static_cast<int64_t>(at.tm) * Tile::BM + wm * (Tile::BM / Tile::WM);
  const int64_t n0 = static_cast<int64_t>(at.tn) * Tile::BN + wn * (Tile::BN / Tile::WN);
  const int64_t M = a.g.a.rows, N = a.g.b.rows;
  // What the rows need is loaded before the first store: loads and stores are counted in one order, so that a load behind
  // a store would wait for it.
  if constexpr (sizeof(T) == 2 && !kPartial) {
    if (a.wide) {
      uint32_t drop = 0;  // bit 4 i + q: the row is to be zeros
      if (a.keep) {
        int32_t keep[Tile::TM][4];
#pragma unroll
        for (int i = 0; i < Tile::TM; ++i)
#pragma unroll
          for (int q = 0; q < 4; ++q)
            keep[i][q] = a.keep[min(m0 + tile_row<Tile, kTurnA>(i, acc_row(4 * q, lane) + lane % 4), M - 1)];
#pragma unroll
        for (int i = 0; i < Tile::TM; ++i)
#pragma unroll
          for (int q = 0; q < 4; ++q) drop |= static_cast<uint32_t>(keep[i][q] < 0) << (4 * i + q);
      }
#pragma unroll
      for (int i = 0; i < Tile::TM; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int64_t m = m0 + tile_row<Tile, kTurnA>(i, acc_row(4 * q, lane) + lane % 4);
          const bool zero = drop >> (4 * i + q) & 1;
          static_assert(Tile::TN == 2, "a wave's columns are a line");
          uint2 x[2];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            x[j].x = bits_of(acc.c[i][j][4 * q]) | bits_of(acc.c[i][j][4 * q + 1]) << 16;
            x[j].y = bits_of(acc.c[i][j][4 * q + 2]) | bits_of(acc.c[i][j][4 * q + 3]) << 16;
            x[j] = turn4(x[j], lane);
          }
          uint4 y = line_of(x[0], x[1], lane);
          if (zero) y = uint4{0, 0, 0, 0};
          const int64_t n = n0 + line_column(lane);
          uint16_t *to = static_cast<uint16_t *>(a.out) + m * N + n;
          if (a.wide == 8) {
            if (m < M && n < N) *reinterpret_cast<uint4 *>(to) = y;
          } else {
            if (m < M && n < N) *reinterpret_cast<uint2 *>(to) = uint2{y.x, y.y};
            if (m < M && n + 4 < N) *reinterpret_cast<uint2 *>(to + 4) = uint2{y.z, y.w};
          }
        }
      return;
    }
  }
  const int e = sizeof(T) == 4 ? -(kTop + exponent_for(read_peak(a.peak))) : 0;
  float *part = kPartial ? a.part + at.split * a.part_stride : nullptr;
  auto write = [&](auto add) {
    constexpr bool kAdd = decltype(add)::value;  // to what is there
#pragma unroll
    for (int i = 0; i < Tile::TM; ++i) {
      auto row = [&](int r) { return m0 + tile_row<Tile, kTurnA>(i, acc_row(r, lane)); };
      float f[16], before[kAdd ? 16 : 1][Tile::TN];
      bool drop[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int64_t m = min(row(r), M - 1);
        f[r] = sizeof(T) == 4 && a.factor ? a.factor[m] : 1.0f;
        drop[r] = !kPartial && a.keep && a.keep[m] < 0;
        if constexpr (kAdd) {
#pragma unroll
          for (int j = 0; j < Tile::TN; ++j) before[r][j] = part[m * N + min(n0 + 32 * j + lane % 32, N - 1)];
        }
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int64_t m = row(r);
        if (m >= M) continue;
#pragma unroll
        for (int j = 0; j < Tile::TN; ++j) {
          const int64_t n = n0 + 32 * j + lane % 32;
          if (n >= N) continue;
          const int64_t to = m * N + n;
          float x = acc.c[i][j][r];
          if constexpr (sizeof(T) == 4) x = __builtin_ldexpf(x, e) * f[r];
          if constexpr (kAdd) x += before[r][j];
          if constexpr (kPartial) part[to] = x;
          else static_cast<T *>(a.out)[to] = narrow<T>(drop[r] ? 0.0f : x);
        }
      }
    }
  };
  if constexpr (kPartial) {
    if (a.accumulate) {
      write(std::true_type{});
      return;
    }
  }
  write(std::false_type{});
}

// out = sum over the splits; rows with keep < 0 become zeros.  Four elements per thread; kShares threads of a workgroup
// share the splits where these are many and the elements few.  A launch takes two products.
struct JoinJob {
  const float *part;
  int64_t part_stride;
  int32_t splits, D;
  int64_t rows;
  void *out;
  const int32_t *keep;
  uint32_t blocks;
};
struct JoinJobs {
  JoinJob job[2];
};
constexpr int kJoinMany = 16, kJoinShares = 8;  // splits from which eight threads share an element's

template <typename T, int kShares>
__device__ __forceinline__ void join_splits(const JoinJob &j, uint32_t block) {
  constexpr int kQuads = kBlockThreads / kShares;
  __shared__ float4 joined[kShares][kQuads];
  const int share = threadIdx.x / kQuads;
  const int64_t total = j.rows * j.D, t = (static_cast<int64_t>(block) * kQuads + threadIdx.x % kQuads) * 4;
  float4 s{0.0f, 0.0f, 0.0f, 0.0f};
  if (t < total)
#pragma unroll 4
    for (int32_t z = j.splits * share / kShares; z < j.splits * (share + 1) / kShares; ++z) {
      const float4 x = *reinterpret_cast<const float4 *>(j.part + z * j.part_stride + t);
      s.x += x.x;
      s.y += x.y;
      s.z += x.z;
      s.w += x.w;
    }
  if constexpr (kShares > 1) {
    joined[share][threadIdx.x % kQuads] = s;
    __syncthreads();
    if (share) return;
#pragma unroll
    for (int k = 1; k < kShares; ++k) {
      const float4 x = joined[k][threadIdx.x];
      s.x += x.x;
      s.y += x.y;
      s.z += x.z;
      s.w += x.w;
    }
  }
  const float x[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (t + k < total) static_cast<T *>(j.out)[t + k] = narrow<T>(j.keep && j.keep[(t + k) / j.D] < 0 ? 0.0f : x[k]);
}

template <typename T>
__global__ __launch_bounds__(kBlockThreads) void join_kernel(JoinJobs jobs) {
  const bool second = blockIdx.x >= jobs.job[0].blocks;
  const JoinJob &j = jobs.job[second];
  const uint32_t block = second ? blockIdx.x - jobs.job[0].blocks : blockIdx.x;
  if (j.splits >= kJoinMany) join_splits<T, kJoinShares>(j, block);
  else join_splits<T, 1>(j, block);
}

__global__ __launch_bounds__(kBlockThreads) void zero_kernel(uint16_t *out, int64_t n) {
  const int64_t stride = static_cast<int64_t>(gridDim.x) * kBlockThreads;
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * kBlockThreads + threadIdx.x; t < n; t += stride) out[t] = 0;
}

// ------------------------------------------------------------------------------------------------ host side
enum TileKind { kBig, kMid, kFlat, kTall };
struct TileSize {
  int bm, bn, per_cu;
  double step;                      // microseconds per step of k with every CU full
  double stats, grad, store;        // ... per tile for the epilogues of the three kernels (16-bit results)
};
// Measured on products of 1024 .. 8192 terms and epilogues of 4096 x 65536 logits.
constexpr TileSize kTileSize[] = {{256, 256, 1, 1.95, 3.1, 12.0, 6.0},
                                  {128, 128, 2, 1.15, 1.4, 5.7, 3.5},
                                  {64, 256, 2, 1.25, 1.4, 6.0, 3.5},
                                  {256, 64, 2, 1.25, 1.4, 6.0, 3.5}};
// Native float32: the step is 32 k, bound by the float32 matrix instructions.
constexpr TileSize kNativeSize[] = {{256, 256, 1, 7.8, 3.1, 0.0, 0.0},
                                    {128, 128, 2, 3.9, 1.4, 0.0, 0.0},
                                    {64, 256, 2, 3.9, 1.4, 0.0, 0.0},
                                    {256, 64, 2, 3.9, 1.4, 0.0, 0.0}};
constexpr double kBytesPerUs = 4.5e6;  // that a pass over memory reaches
constexpr int kCus = 256;

int64_t up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }
int64_t steps_of(int64_t k) { return (k + kStepK - 1) / kStepK; }

int64_t tiles_of(int64_t n, int64_t per) { return (n + per - 1) / per; }

// Microseconds that `groups` workgroups of this kind take, each `work` with the device full.
double rounds_time(const TileSize &s, int64_t groups, double work) {
  const int64_t slots = kCus * s.per_cu;
  if (groups <= kCus && s.per_cu > 1) return 0.7 * work;  // alone on its CU
  return static_cast<double>((groups + slots - 1) / slots) * work;
}

// Ranges of the vocabulary tiles for the statistics: the division with the shortest time, each workgroup costing about
// three microseconds to begin.
constexpr int kMostRanges = 256;
double choose_ranges(const TileSize &s, int64_t M, int64_t N, int64_t steps, double epilogue, int *ranges) {
  const int64_t tiles_m = tiles_of(M, s.bm), tiles_n = tiles_of(N, s.bn);
  double least = -1.0;
  for (int64_t each = tiles_of(tiles_m, kMostRanges); each <= tiles_m;) {  // tiles per workgroup
    const int64_t r = tiles_of(tiles_m, each);
    const double t = rounds_time(s, tiles_n * r, static_cast<double>(each) * (steps * s.step + epilogue) + 3.0);
    if (least < 0.0 || t < least) {
      *ranges = static_cast<int>(r);
      least = t;
    }
    if (r == 1) break;
    each = tiles_of(tiles_m, r - 1);  // the next one that needs fewer ranges
  }
  return least;
}

// Splits of a product's k: more workgroups where there are few tiles, against partial sums written and read again (about
// 4 TB/s, and a launch).
double choose_splits(const TileSize &s, int64_t M, int64_t N, int64_t steps, int *splits) {
  const int64_t tiles = tiles_of(M, s.bm) * tiles_of(N, s.bn);
  double least = 0.0;
  for (int z = 1; z <= 256 && (z == 1 || (steps / z >= 4 && z * M * N <= (int64_t{1} << 28))); z += z < 8 ? 1 : z / 4) {
    double t = rounds_time(s, tiles * z, static_cast<double>(tiles_of(steps, z)) * s.step + s.store);
    if (z > 1) t += 4.0 + static_cast<double>(z) * M * N * 8.0 / 4e6;
    if (z == 1 || t < least) {
      *splits = z;
      least = t;
    }
  }
  return least;
}

// The kind of tile with the shortest time by `cost`, which goes to *time.
template <typename F>
TileKind choose_tile(F &&cost, const TileSize *sizes = kTileSize, double *time = nullptr) {
  int best = kBig;
  double least = 0.0;
  const int forced = config().ce_tile;
  for (int k = 0; k < 4; ++k) {
    if (forced && k != std::min(forced, 4) - 1) continue;
    const double t = cost(sizes[k]);
    if (forced || k == 0 || t < least) {
      best = k;
      least = t;
    }
  }
  if (time) *time = least;
  return static_cast<TileKind>(best);
}

// Copies and P of one piece of the vocabulary.  As few pieces as memory allows: smaller ones, that the last-level cache
// would hold, cost more in short launches than the cache gives back (4096 x 65536 x 1024: 2371 us for the gradient in
// pieces of 256 MiB, 2005 of 512, 1891 of 1024, 1780 in one).
constexpr int64_t kPieceBytes = int64_t{4} << 30;
constexpr int64_t kMostPieceRows = 1 << 22;  // which 32-bit offsets into four panels reach

struct Layout {
  int parts, segments;
  int64_t pieces;
  int ranges;            // of a piece's vocabulary tiles
  bool native;           // float32 multiplied as it is (loss only)
  bool packed;           // operands copied with k padded (float32, or rows that are no multiple of kStepK or 16 bytes)
  int64_t piece;         // vocabulary rows per piece, a multiple of 256
  TileKind logits, dh, dw;
  int dh_splits, dw_splits;
  int64_t h_pack, w_pack, h_exp, w_exp, peaks, stats, label, ht, wt, vn, dh_part, dw_part, bytes;
};

Layout layout(int64_t N, int64_t V, int64_t D, int dtype, bool aligned, bool backward) {
  Layout l{};
  l.parts = dtype == FG_F32 ? kParts : 1;
  l.segments = dtype == FG_F32 ? kSegments : 1;
  if (dtype == FG_F32 && !backward) {
    // as they are, against three products of copies, which are written once and read twice (with a launch of their own)
    double split, native;
    int r;
    choose_tile([&](const TileSize &s) { return choose_ranges(s, V, N, steps_of(D) * kSegments, s.stats, &r); }, kTileSize, &split);
    choose_tile([&](const TileSize &s) { return choose_ranges(s, V, N, steps_of(2 * D), s.stats, &r); }, kNativeSize, &native);
    const double bytes = 4.0 * static_cast<double>(N + V) * static_cast<double>(D);
    l.native = std::max(native, bytes / kBytesPerUs) < split + 5.0 + 3.0 * bytes / kBytesPerUs;
    if (config().ce_native >= 0) l.native = config().ce_native != 0;
  }
  if (l.native) l.segments = 1;
  l.packed = !l.native && (dtype == FG_F32 || D % kStepK != 0 || !aligned);
  int64_t per_row = l.packed ? 2 * l.parts * up(D, kStepK) : 0;
  if (backward) per_row += 2 * l.parts * (up(N, kStepK) + D);
  const int64_t most = per_row ? std::clamp<int64_t>(kPieceBytes / per_row / 256 * 256, 256, kMostPieceRows) : up(V, 256);
  l.piece = up((V + (V + most - 1) / most - 1) / ((V + most - 1) / most), 256);  // as many pieces as needed, of equal size
  if (const int64_t rows = config().ce_piece_rows) l.piece = std::min(up(rows, 256), kMostPieceRows);
  const int64_t in_piece = std::min(l.piece, V);
  l.pieces = (V + l.piece - 1) / l.piece;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += up(bytes, 1024);
    return here;
  };
  l.h_pack = take(l.packed ? 2 * l.parts * panel_elements(N, D) : 0);
  l.w_pack = take(l.packed ? 2 * l.parts * panel_elements(in_piece, D) : 0);
  if (l.packed && dtype == FG_F32) {
    l.h_exp = take(4 * up(N, 256));
    l.w_exp = take(4 * up(in_piece, 256));
    l.peaks = take(4 * kPeakSlots * kPeakStride * (1 + l.pieces));
  }
  const int64_t steps = l.native ? steps_of(2 * D) : steps_of(D) * l.segments;
  if (!backward) {
    const TileSize *sizes = l.native ? kNativeSize : kTileSize;
    l.logits = choose_tile([&](const TileSize &s) { return choose_ranges(s, in_piece, N, steps, s.stats, &l.ranges); }, sizes);
    choose_ranges(sizes[l.logits], in_piece, N, steps, sizes[l.logits].stats, &l.ranges);
    l.stats = take(l.pieces * l.ranges * N * 8);
  } else {
    l.logits = choose_tile([&](const TileSize &s) { return choose_ranges(s, in_piece, N, steps, l.parts * s.grad, &l.ranges); });
    choose_ranges(kTileSize[l.logits], in_piece, N, steps, l.parts * kTileSize[l.logits].grad, &l.ranges);
    int z;
    const int64_t dh_steps = steps_of(in_piece) * l.segments, dw_steps = steps_of(N) * l.segments;
    l.dh = choose_tile([&](const TileSize &s) { return choose_splits(s, N, D, dh_steps, &z); });
    l.dw = choose_tile([&](const TileSize &s) { return choose_splits(s, in_piece, D, dw_steps, &z); });
    choose_splits(kTileSize[l.dh], N, D, dh_steps, &l.dh_splits);
    choose_splits(kTileSize[l.dw], in_piece, D, dw_steps, &l.dw_splits);
    l.label = take(4 * N);
    l.ht = take(2 * l.parts * panel_elements(D, N));
    l.wt = take(2 * l.parts * panel_elements(D, in_piece));
    l.vn = take(2 * l.parts * panel_elements(up(in_piece, kStepK), N));
    l.dh_part = take(l.dh_splits > 1 || V > l.piece ? 4 * l.dh_splits * up(N * D, 4) : 0);
    l.dw_part = take(l.dw_splits > 1 ? 4 * l.dw_splits * up(in_piece * D, 4) : 0);
  }
  l.bytes = std::max<int64_t>(at, 1024);
  return l;
}

template <typename F>
int with_tile(TileKind kind, GemmShape *g, F &&launch) {
  const TileSize &s = kTileSize[kind];
  g->tiles_m = (g->a.rows + s.bm - 1) / s.bm;
  g->tiles_n = (g->b.rows + s.bn - 1) / s.bn;
  const int64_t blocks = static_cast<int64_t>(g->tiles_m) * g->tiles_n * g->splits;
  if (blocks > 0x7fffffffLL) return fail(FG_EUNSUPPORTED, "%lld tiles are too many", (long long)blocks);
  const dim3 grid(static_cast<unsigned>(blocks));
  switch (kind) {
    case kBig: launch(Big{}, grid); break;
    case kMid: launch(Mid{}, grid); break;
    case kFlat: launch(Flat{}, grid); break;
    case kTall: launch(Tall{}, grid); break;
  }
  FG_HIP_TRY(hipGetLastError());
  return FG_OK;
}

unsigned flat_grid(int64_t threads) {
  return static_cast<unsigned>(std::max<int64_t>(1, std::min<int64_t>((threads + kBlockThreads - 1) / kBlockThreads, 1 << 14)));
}

// The matrix x as an operand of the logits: used in place, or where job->out will have copied it.
template <typename T>
GemmOperand operand(const CopyJob &job, const Layout &l) {
  if (l.packed) return panels(job.out, job.rows, job.D);
  GemmOperand o;
  o.rows = static_cast<int32_t>(job.rows);
  o.p = static_cast<const uint16_t *>(job.x);
  o.row = job.D * static_cast<int64_t>(sizeof(T) / 2);
  o.step = kStepK;
  return o;
}

template <typename T>
void copy_rows(CopyJobs jobs, hipStream_t stream) {
  for (CopyJob &j : jobs.job)
    j.blocks = j.rows == 0 ? 0
               : sizeof(T) == 4 ? static_cast<uint32_t>(std::min<int64_t>((j.rows + kWavesPerBlock - 1) / kWavesPerBlock, 4096))
                                : flat_grid(panel_elements(j.rows, j.D) / 8);
  const dim3 grid(jobs.job[0].blocks + jobs.job[1].blocks);
  const int64_t D = std::max(jobs.job[0].D, jobs.job[1].D);
  auto launch = [&](auto held) {
    copy_rows_kernel<T, decltype(held)::value><<<grid, dim3(kBlockThreads), 0, stream>>>(jobs);
  };
  if constexpr (sizeof(T) == 2) launch(std::integral_constant<int, 0>{});
  else if (D > 16 * kWaveSize) launch(std::integral_constant<int, 0>{});
  else if (D > 8 * kWaveSize) launch(std::integral_constant<int, 16>{});
  else if (D > 2 * kWaveSize) launch(std::integral_constant<int, 8>{});
  else launch(std::integral_constant<int, 2>{});
}

template <typename T>
void copy_transposed(CopyJobs jobs, hipStream_t stream) {
  for (CopyJob &j : jobs.job) j.blocks = static_cast<uint32_t>(steps_of(j.rows) * ((j.D + 63) / 64));
  const dim3 grid(jobs.job[0].blocks + jobs.job[1].blocks);
  copy_transposed_kernel<T><<<grid, dim3(kBlockThreads), 0, stream>>>(jobs);
}

template <typename T>
void join(JoinJobs jobs, hipStream_t stream) {
  for (JoinJob &j : jobs.job) {
    const int quads = j.splits >= kJoinMany ? kBlockThreads / kJoinShares : kBlockThreads;  // of a workgroup
    j.blocks = static_cast<uint32_t>(((j.rows * j.D + 3) / 4 + quads - 1) / quads);
  }
  const dim3 grid(jobs.job[0].blocks + jobs.job[1].blocks);
  if (grid.x > 0) join_kernel<T><<<grid, dim3(kBlockThreads), 0, stream>>>(jobs);
}

template <typename T, typename Id>
int forward(int64_t N, int64_t V, int64_t D, const T *h, const T *w, const Id *labels, float *loss, float *lse,
            char *ws, const Layout &l, hipStream_t stream) {
  StatsArgs a{};
  a.g.splits = 1;
  a.labels = labels;
  a.label_logit = loss;
  a.part = reinterpret_cast<float2 *>(ws + l.stats);
  a.g.steps = static_cast<int32_t>(steps_of(l.native ? 2 * D : D));
  a.g.tail = static_cast<int32_t>(l.native ? 2 * D - (a.g.steps - 1) * kStepK : kStepK);
  auto *h_exp = reinterpret_cast<int32_t *>(ws + l.h_exp), *w_exp = reinterpret_cast<int32_t *>(ws + l.w_exp);
  a.exp_a = w_exp;
  a.exp_b = h_exp;
  CopyJobs jobs{};
  jobs.job[0] = CopyJob{h, reinterpret_cast<uint16_t *>(ws + l.h_pack), N, static_cast<int32_t>(D), 0, h_exp};
  a.g.b = operand<T>(jobs.job[0], l);
  for (int64_t v0 = 0; v0 < V; v0 += l.piece) {
    jobs.job[1] = CopyJob{w + v0 * D, reinterpret_cast<uint16_t *>(ws + l.w_pack), std::min(l.piece, V - v0), static_cast<int32_t>(D), 0, w_exp};
    a.g.a = operand<T>(jobs.job[1], l);
    if (l.packed) copy_rows<T>(jobs, stream);
    jobs.job[0].rows = 0;  // h is there now
    a.v0 = v0;
    const int rc = with_tile(l.logits, &a.g, [&](auto tile, dim3) {
      using Tile = decltype(tile);
      a.ranges = std::min(l.ranges, a.g.tiles_m);
      const dim3 grid(static_cast<unsigned>(a.ranges * a.g.tiles_n));
      if constexpr (sizeof(T) == 4) {
        if (l.native) {
          stats_kernel<Tile, T, MultiplyNative, Id><<<grid, dim3(Tile::kThreads), 0, stream>>>(a);
          return;
        }
      }
      stats_kernel<Tile, T, Multiply<T>, Id><<<grid, dim3(Tile::kThreads), 0, stream>>>(a);
    });
    if (rc) return rc;
    a.range0 += a.ranges;
  }
  auto finish = [&](auto shares) {
    constexpr int kRows = kBlockThreads / decltype(shares)::value;
    loss_kernel<Id, decltype(shares)::value><<<dim3(static_cast<unsigned>(tiles_of(N, kRows))), dim3(kBlockThreads), 0, stream>>>(
        a.part, a.range0, labels, static_cast<int32_t>(N), V, loss, lse);
  };
  if (a.range0 <= kFewRanges) finish(std::integral_constant<int, 1>{});
  else finish(std::integral_constant<int, 16>{});
  FG_HIP_TRY(hipGetLastError());
  return FG_OK;
}

// out[M, D] = the product, through partial sums where k is shared or earlier pieces have added to them
template <typename T, bool kTurnA>
int product(TileKind kind, StoreArgs a, T *out, bool partial, hipStream_t stream) {
  a.out = out;
  a.wide = a.g.b.rows % 8 == 0 && aligned_to(out, 16) ? 8 : a.g.b.rows % 4 == 0 && aligned_to(out, 8) ? 4 : 0;
  return with_tile(kind, &a.g, [&](auto tile, dim3 grid) {
    using Tile = decltype(tile);
    if (partial)
      product_kernel<Tile, T, true, kTurnA><<<grid, dim3(Tile::kThreads), 0, stream>>>(a);
    else
      product_kernel<Tile, T, false, kTurnA><<<grid, dim3(Tile::kThreads), 0, stream>>>(a);
  });
}

template <typename T>
int backward(int64_t N, int64_t V, int64_t D, const T *h, const T *w, const float *lse, const float *dloss, T *dh,
             T *dw, char *ws, const Layout &l, hipStream_t stream) {
  const int32_t *label = reinterpret_cast<const int32_t *>(ws + l.label);
  auto *ht = reinterpret_cast<uint16_t *>(ws + l.ht), *wt = reinterpret_cast<uint16_t *>(ws + l.wt);
  auto *vn = reinterpret_cast<uint16_t *>(ws + l.vn);
  GradArgs a{};
  a.label = label;
  a.lse = lse;
  a.dloss = dloss;
  a.vn = vn;
  a.g.steps = static_cast<int32_t>(steps_of(D));
  auto *h_exp = reinterpret_cast<int32_t *>(ws + l.h_exp), *w_exp = reinterpret_cast<int32_t *>(ws + l.w_exp);
  uint32_t *peaks = sizeof(T) == 4 ? reinterpret_cast<uint32_t *>(ws + l.peaks) : nullptr;  // of h, then of each piece of w
  const float *factor = sizeof(T) == 4 ? dloss : nullptr;
  a.exp_a = w_exp;
  a.exp_b = h_exp;
  CopyJobs rows_of, transposed;
  rows_of.job[0] = CopyJob{h, reinterpret_cast<uint16_t *>(ws + l.h_pack), N, static_cast<int32_t>(D), 0, h_exp, peaks, label, factor};
  transposed.job[0] = rows_of.job[0];
  transposed.job[0].out = ht;
  const bool together = sizeof(T) == 2 && l.packed;  // both copies in one pass
  if (together) transposed.job[0].rows_out = rows_of.job[0].out;
  a.g.b = operand<T>(rows_of.job[0], l);
  const bool dh_partial = l.dh_splits > 1 || V > l.piece;
  JoinJobs joins{};
  for (int64_t v0 = 0; v0 < V; v0 += l.piece) {
    const int64_t rows = std::min(l.piece, V - v0);
    a.v0 = static_cast<int32_t>(v0);
    a.vn_part = panel_elements(up(rows, kStepK), N);
    uint32_t *peak = peaks ? peaks + (1 + v0 / l.piece) * kPeakSlots * kPeakStride : nullptr;
    rows_of.job[1] = CopyJob{w + v0 * D, reinterpret_cast<uint16_t *>(ws + l.w_pack), rows, static_cast<int32_t>(D), 0, w_exp, peak};
    transposed.job[1] = rows_of.job[1];
    transposed.job[1].out = wt;
    if (together) transposed.job[1].rows_out = rows_of.job[1].out;
    a.g.a = operand<T>(rows_of.job[1], l);
    if (l.packed && !together) copy_rows<T>(rows_of, stream);
    copy_transposed<T>(transposed, stream);
    rows_of.job[0].rows = transposed.job[0].rows = 0;  // h is there now
    int rc = with_tile(l.logits, &a.g, [&](auto tile, dim3) {
      using Tile = decltype(tile);
      a.ranges = std::min(l.ranges, a.g.tiles_m);
      grad_logits_kernel<Tile, T><<<dim3(static_cast<unsigned>(a.ranges * a.g.tiles_n)), dim3(Tile::kThreads), 0, stream>>>(a);
    });
    if (rc) return rc;

    StoreArgs s{};  // dw[v, d] = sum over n of G[v, n] * h[n, d]
    s.g.steps = static_cast<int32_t>(steps_of(N));
    s.g.splits = l.dw_splits;
    s.g.a = panels(vn, up(rows, kStepK), N);
    s.g.a.rows = static_cast<int32_t>(rows);
    s.g.b = panels(ht, D, N);
    s.peak = peaks;
    s.part = reinterpret_cast<float *>(ws + l.dw_part);
    s.part_stride = up(rows * D, 4);
    rc = product<T, false>(l.dw, s, dw + v0 * D, l.dw_splits > 1, stream);
    if (rc) return rc;
    if (l.dw_splits > 1)
      joins.job[0] = JoinJob{s.part, s.part_stride, l.dw_splits, static_cast<int32_t>(D), rows, dw + v0 * D, nullptr, 0};

    s.g.steps = static_cast<int32_t>(steps_of(rows));  // dh[n, d] = sum over v of G[n, v] * w[v, d]
    s.g.splits = l.dh_splits;
    s.g.a = turned_panels(vn, N, rows);
    s.g.b = panels(wt, D, rows);
    s.keep = label;
    s.factor = factor;
    s.peak = peak;
    s.part = reinterpret_cast<float *>(ws + l.dh_part);
    s.part_stride = up(N * D, 4);
    s.accumulate = v0 > 0;
    rc = product<T, true>(l.dh, s, dh, dh_partial, stream);
    if (rc) return rc;
    if (dh_partial && v0 + l.piece >= V)
      joins.job[1] = JoinJob{s.part, s.part_stride, l.dh_splits, static_cast<int32_t>(D), N, dh, label, 0};
    join<T>(joins, stream);
  }
  FG_HIP_TRY(hipGetLastError());
  return FG_OK;
}

int check_ce(int64_t N, int64_t V, int64_t D, int32_t dtype, int32_t itype) {
  if (N < 0 || N > (1 << 22)) return fail(FG_EINVAL, "N = %lld is out of range", (long long)N);
  if (V < 1 || V >= 0x7fff0000LL) return fail(FG_EINVAL, "V = %lld is out of range", (long long)V);
  if (D < 1 || D > (1 << 16)) return fail(FG_EINVAL, "D = %lld is out of range", (long long)D);
  if (dtype != FG_F32 && dtype != FG_BF16) return fail(FG_EUNSUPPORTED, "dtype code %d: float32 and bfloat16 only", dtype);
  if (!index_type_ok(itype)) return fail(FG_EINVAL, "index type code %d is unknown", itype);
  return FG_OK;
}

int check_space(const void *workspace, int64_t bytes, int64_t need) {
  if (!workspace || !aligned_to(workspace, 256) || bytes < need)
    return fail(FG_EINVAL, "the workspace needs %lld bytes at a multiple of 256", (long long)need);
  return FG_OK;
}

// Bytes for operands of any alignment.
int64_t space(int64_t N, int64_t V, int64_t D, int32_t dtype, bool backward) {
  return std::max(layout(N, V, D, dtype, true, backward).bytes, layout(N, V, D, dtype, false, backward).bytes);
}

}  // namespace
}  // namespace fg

extern "C" {

int fg_linear_ce_workspace(int64_t N, int64_t V, int64_t D, int32_t dtype, int64_t *bytes) {
  if (int rc = fg::check_ce(N, V, D, dtype, FG_I32)) return rc;
  if (!bytes) return fg::fail(FG_EINVAL, "bytes is null");
  *bytes = fg::space(std::max<int64_t>(N, 1), V, D, dtype, false);
  return FG_OK;
}

int fg_linear_ce(int64_t N, int64_t V, int64_t D, const void *hidden, const void *weight, const void *labels,
                 float *loss, float *lse, int32_t dtype, int32_t itype, void *workspace, int64_t workspace_bytes,
                 void *stream) {
  if (int rc = fg::check_ce(N, V, D, dtype, itype)) return rc;
  if (N == 0) return FG_OK;
  if (!hidden || !weight || !labels || !loss || !lse) return fg::fail(FG_EINVAL, "a data pointer is null");
  const fg::Layout l = fg::layout(N, V, D, dtype, fg::aligned_to(hidden, 16) && fg::aligned_to(weight, 16), false);
  if (int rc = fg::check_space(workspace, workspace_bytes, l.bytes)) return rc;
  char *ws = static_cast<char *>(workspace);
  hipStream_t s = static_cast<hipStream_t>(stream);
#define FG_TYPED(T, Id)                                                                                        \
  fg::forward<T, Id>(N, V, D, static_cast<const T *>(hidden), static_cast<const T *>(weight),                  \
                     static_cast<const Id *>(labels), loss, lse, ws, l, s)
  if (dtype == FG_F32) return itype == FG_I32 ? FG_TYPED(float, int32_t) : FG_TYPED(float, int64_t);
  return itype == FG_I32 ? FG_TYPED(__bf16, int32_t) : FG_TYPED(__bf16, int64_t);
#undef FG_TYPED
}

int fg_linear_ce_grad_workspace(int64_t N, int64_t V, int64_t D, int32_t dtype, int64_t *bytes) {
  if (int rc = fg::check_ce(N, V, D, dtype, FG_I32)) return rc;
  if (!bytes) return fg::fail(FG_EINVAL, "bytes is null");
  *bytes = fg::space(std::max<int64_t>(N, 1), V, D, dtype, true);
  return FG_OK;
}

int fg_linear_ce_grad(int64_t N, int64_t V, int64_t D, const void *hidden, const void *weight, const void *labels,
                      const float *lse, const float *dloss, void *dhidden, void *dweight, int32_t dtype, int32_t itype,
                      void *workspace, int64_t workspace_bytes, void *stream) {
  if (int rc = fg::check_ce(N, V, D, dtype, itype)) return rc;
  if (!dweight) return fg::fail(FG_EINVAL, "a data pointer is null");
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (N == 0) {  // no rows: the weight's gradient is zero
    const int64_t bytes = V * D * fg::element_bytes(dtype);
    fg::zero_kernel<<<dim3(fg::flat_grid(bytes / 2)), dim3(fg::kBlockThreads), 0, s>>>(static_cast<uint16_t *>(dweight), bytes / 2);
    FG_HIP_TRY(hipGetLastError());
    return FG_OK;
  }
  if (!hidden || !weight || !labels || !lse || !dloss || !dhidden) return fg::fail(FG_EINVAL, "a data pointer is null");
  const fg::Layout l = fg::layout(N, V, D, dtype, fg::aligned_to(hidden, 16) && fg::aligned_to(weight, 16), true);
  if (int rc = fg::check_space(workspace, workspace_bytes, l.bytes)) return rc;
  char *ws = static_cast<char *>(workspace);
  int32_t *label = reinterpret_cast<int32_t *>(ws + l.label);
  uint32_t *peaks = reinterpret_cast<uint32_t *>(ws + l.peaks);
  const int32_t n_peaks = dtype == FG_F32 ? static_cast<int32_t>(fg::kPeakSlots * fg::kPeakStride * (1 + l.pieces)) : 0;
  const dim3 grid(static_cast<unsigned>((N + fg::kBlockThreads - 1) / fg::kBlockThreads));
  if (itype == FG_I32)
    fg::labels_kernel<int32_t><<<grid, dim3(fg::kBlockThreads), 0, s>>>(static_cast<const int32_t *>(labels), static_cast<int32_t>(N), V, label, peaks, n_peaks);
  else
    fg::labels_kernel<int64_t><<<grid, dim3(fg::kBlockThreads), 0, s>>>(static_cast<const int64_t *>(labels), static_cast<int32_t>(N), V, label, peaks, n_peaks);
#define FG_TYPED(T)                                                                                              \
  fg::backward<T>(N, V, D, static_cast<const T *>(hidden), static_cast<const T *>(weight), lse, dloss,           \
                  static_cast<T *>(dhidden), static_cast<T *>(dweight), ws, l, s)
  return dtype == FG_F32 ? FG_TYPED(float) : FG_TYPED(__bf16);
#undef FG_TYPED
}

}  // extern "C"
