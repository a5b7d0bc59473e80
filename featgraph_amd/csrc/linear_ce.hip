// Softmax cross entropy of a linear scorer, without keeping the logits:
//
//   l[n, v]  = <h[n], w[v]>                    lse[n] = log sum over v of exp l[n, v]
//   loss[n]  = lse[n] - l[n, y[n]]             (0 where the label y[n] is outside [0, V): the row is ignored)
//   G[n, v]  = dloss[n] * (exp(l[n, v] - lse[n]) - [v = y[n]])          (0 for an ignored row)
//   dh = G w        dw = G^T h
//
// Forward: one matrix product whose epilogue keeps, per row n and tile of vocabulary, the largest logit and the sum
// of exponentials relative to it; a second kernel joins the tiles and takes the label's logit as a dot product of its
// own.  Backward: the logits are computed again piece by piece of the vocabulary; the epilogue turns them into G,
// written once as [n, v] and once as [v, n], and two more products over them give the piece's rows of dw and its
// share of dh.  All three products are the same kernel over operands with k contiguous, so h and w are transposed
// into padded copies for the backward products (2 N D + 2 V D elements of traffic against 6 N V D flops).
//
// Types: bfloat16 operands are used as they are; G is rounded to bfloat16 for the products (half a step, 2^-9 of each
// term, random in sign; the results are rounded to bfloat16 themselves), everything between is float32.  float32
// operands, G among them, are split into three bfloat16 parts (mfma_gemm.hpp), which keeps float32's accuracy: six
// bfloat16 products run at 2.6 times the peak rate of the float32 matrix instructions.
#include <algorithm>
#include <cmath>

#include "mfma_gemm.hpp"

namespace fg {
namespace {

constexpr float kLog2e = 1.44269504088896340736f;

using Big = GemmTile<256, 256, 2, 4>;   // 128 x 64 per wave, one workgroup per CU
using Mid = GemmTile<128, 128, 2, 2>;   // 64 x 64 per wave, two workgroups per CU
using Flat = GemmTile<64, 256, 1, 4>;   // few rows of A
using Tall = GemmTile<256, 64, 4, 1>;   // few rows of B

// ------------------------------------------------------------------------------------------------ operand copies
struct Split {
  uint16_t part[kParts];
};
__device__ __forceinline__ uint16_t bits_of(float x) { return __builtin_bit_cast(uint16_t, narrow<__bf16>(x)); }
__device__ __forceinline__ float from_bits(uint16_t b) { return __builtin_bit_cast(float, static_cast<uint32_t>(b) << 16); }

// x = part 0 + part 1 + part 2 to 2^-24 of x and better.  A finite x that would round to infinity is cut instead; what is
// not finite has no further parts, so that it does not turn into NaN by inf - inf.
__device__ __forceinline__ Split split3(float x) {
  Split s;
  uint32_t u = __builtin_bit_cast(uint32_t, x);
  s.part[0] = bits_of(x);
  if ((s.part[0] & 0x7f80) == 0x7f80) {
    if ((u & 0x7f800000u) == 0x7f800000u) {
      s.part[1] = s.part[2] = 0;
      return s;
    }
    s.part[0] = static_cast<uint16_t>(u >> 16);
  }
  const float r = x - from_bits(s.part[0]);
  s.part[1] = bits_of(r);
  s.part[2] = bits_of(r - from_bits(s.part[1]));
  return s;
}

template <typename T>
__device__ __forceinline__ void store_parts(uint16_t *out, int64_t at, int64_t part, float x) {
  if constexpr (sizeof(T) == 4) {
    const Split s = split3(x);
#pragma unroll
    for (int p = 0; p < kParts; ++p) out[p * part + at] = s.part[p];
  } else {
    out[at] = bits_of(x);
  }
}

// [rows, D] -> parts of [rows, Dp], zeros behind D
template <typename T>
__global__ __launch_bounds__(kBlockThreads) void pack_kernel(const T *x, uint16_t *out, int64_t rows, int32_t D,
                                                             int32_t Dp) {
  const int64_t total = rows * Dp, stride = static_cast<int64_t>(gridDim.x) * kBlockThreads;
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * kBlockThreads + threadIdx.x; t < total; t += stride) {
    const int64_t r = t / Dp;
    const int32_t c = static_cast<int32_t>(t - r * Dp);
    store_parts<T>(out, t, total, c < D ? widen(x[r * D + c]) : 0.0f);
  }
}

// [rows, D] -> parts of [D, pitch], zeros behind the rows and, with `keep`, in place of rows whose keep[] is negative
// (whatever those hold must not reach the sum over rows)
template <typename T>
__global__ __launch_bounds__(kBlockThreads) void transpose_kernel(const T *x, const int32_t *keep, uint16_t *out,
                                                                  int32_t rows, int32_t D, int64_t pitch) {
  __shared__ float tile[64][65];
  const int r0 = blockIdx.x * 64, c0 = blockIdx.y * 64;
  const int low = threadIdx.x & 63, high = threadIdx.x >> 6;
  for (int k = high; k < 64; k += kWavesPerBlock) {
    const int r = r0 + k, c = c0 + low;
    float v = 0.0f;
    if (r < rows && c < D && (!keep || keep[r] >= 0)) v = widen(x[static_cast<int64_t>(r) * D + c]);
    tile[k][low] = v;
  }
  __syncthreads();
  for (int k = high; k < 64; k += kWavesPerBlock) {
    const int r = r0 + low, c = c0 + k;
    if (c < D && r < pitch) store_parts<T>(out, static_cast<int64_t>(c) * pitch + r, D * pitch, tile[low][k]);
  }
}

template <typename Id>
__global__ __launch_bounds__(kBlockThreads) void labels_kernel(const Id *labels, int32_t n, int64_t V, int32_t *out) {
  const int i = blockIdx.x * kBlockThreads + threadIdx.x;
  if (i < n) {
    const Id y = labels[i];
    out[i] = y >= 0 && static_cast<int64_t>(y) < V ? static_cast<int32_t>(y) : -1;
  }
}

// ------------------------------------------------------------------------------------------------ forward
struct StatsArgs {
  GemmShape g;
  float2 *part;      // [tiles of vocabulary, N]: largest logit, sum of exp(l - largest)
  int32_t tile0;     // first tile of this piece
};

__device__ __forceinline__ float2 join_stats(float2 a, float2 b) {
  const float m = fmaxf(a.x, b.x);
  if (m == -INFINITY) return float2{m, a.y + b.y};
  return float2{m, a.y * __builtin_amdgcn_exp2f((a.x - m) * kLog2e) + b.y * __builtin_amdgcn_exp2f((b.x - m) * kLog2e)};
}

template <typename Tile>
__global__ __launch_bounds__(Tile::kThreads) void stats_kernel(StatsArgs a) {
  __shared__ __attribute__((aligned(1024))) uint16_t lds[Tile::kLds];
  GemmAcc<Tile> acc;
  const GemmPlace at = gemm_place(a.g);
  gemm_tile<Tile>(a.g, at, lds, acc);
  __syncthreads();
  const int lane = threadIdx.x & (kWaveSize - 1), wave = threadIdx.x / kWaveSize;
  const int wm = wave / Tile::WN, wn = wave % Tile::WN;
  const int v0 = at.tm * Tile::BM + wm * (Tile::BM / Tile::WM);
  float2 *stats = reinterpret_cast<float2 *>(lds);  // [WM][BN]
  const bool edge = v0 + Tile::BM / Tile::WM > a.g.a.rows;
#pragma unroll
  for (int j = 0; j < Tile::TN; ++j) {
    if (edge) {
#pragma unroll
      for (int i = 0; i < Tile::TM; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (v0 + 32 * i + acc_row(r, lane) >= a.g.a.rows) acc.c[i][j][r] = -INFINITY;
    }
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < Tile::TM; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) m = fmaxf(m, acc.c[i][j][r]);
    m = fmaxf(m, __shfl_xor(m, 32, kWaveSize));
    const float from = m == -INFINITY ? 0.0f : m;
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < Tile::TM; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) s += __builtin_amdgcn_exp2f((acc.c[i][j][r] - from) * kLog2e);
    s += __shfl_xor(s, 32, kWaveSize);
    if (lane < 32) stats[wm * Tile::BN + wn * (Tile::BN / Tile::WN) + 32 * j + lane] = float2{m, s};
  }
  __syncthreads();
  for (int c = threadIdx.x; c < Tile::BN; c += Tile::kThreads) {
    const int64_t n = static_cast<int64_t>(at.tn) * Tile::BN + c;
    if (n >= a.g.b.rows) continue;
    float2 s = stats[c];
#pragma unroll
    for (int w = 1; w < Tile::WM; ++w) s = join_stats(s, stats[w * Tile::BN + c]);
    a.part[(static_cast<int64_t>(a.tile0) + at.tm) * a.g.b.rows + n] = s;
  }
}

// 64 rows per workgroup: its 16 waves share the tiles of vocabulary, then take four rows' labels each.
constexpr int kLossThreads = 1024;
template <typename T, typename Id>
__global__ __launch_bounds__(kLossThreads) void loss_kernel(const float2 *part, int32_t tiles, const T *h, const T *w,
                                                            const Id *labels, int32_t N, int64_t V, int32_t D,
                                                            float *loss, float *lse) {
  constexpr int kWaves = kLossThreads / kWaveSize;
  __shared__ float2 joined[kWaves][kWaveSize];
  __shared__ float row_lse[kWaveSize];
  const int lane = threadIdx.x & (kWaveSize - 1), wave = threadIdx.x / kWaveSize;
  const int64_t n = static_cast<int64_t>(blockIdx.x) * kWaveSize + lane;
  float2 s{-INFINITY, 0.0f};
  if (n < N)
    for (int32_t t = wave; t < tiles; t += kWaves) s = join_stats(s, part[static_cast<int64_t>(t) * N + n]);
  joined[wave][lane] = s;
  __syncthreads();
  if (wave == 0) {
#pragma unroll
    for (int k = 1; k < kWaves; ++k) s = join_stats(s, joined[k][lane]);
    const float r = s.x + logf(s.y);
    row_lse[lane] = r;
    if (n < N) lse[n] = r;
  }
  __syncthreads();
  for (int k = wave; k < kWaveSize; k += kWaves) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * kWaveSize + k;
    if (i >= N) break;
    const Id y = labels[i];
    const bool there = y >= 0 && static_cast<int64_t>(y) < V;
    float dot = 0.0f;
    if (there) {
      const T *a = h + i * D, *b = w + static_cast<int64_t>(y) * D;
      for (int32_t c = lane; c < D; c += kWaveSize) dot = __builtin_fmaf(widen(a[c]), widen(b[c]), dot);
#pragma unroll
      for (int d = 1; d < kWaveSize; d <<= 1) dot += __shfl_xor(dot, d, kWaveSize);
    }
    if (lane == 0) loss[i] = there ? row_lse[k] - dot : 0.0f;
  }
}

// ------------------------------------------------------------------------------------------------ backward
struct GradArgs {
  GemmShape g;               // a: the piece's rows of w, b: h
  const int32_t *label;      // [N], negative: ignored
  const float *lse, *dloss;  // [N]
  int32_t v0;                // first vocabulary row of the piece
  uint16_t *nv, *vn;         // G as [N, pitch_v] and [rows of the piece, pitch_n], parts apart by *_part
  int64_t nv_part, vn_part;
  int32_t pitch_v, pitch_n;
};

// T: type of the operands, which says how G is stored.
template <typename Tile, typename T>
__global__ __launch_bounds__(Tile::kThreads) void grad_logits_kernel(GradArgs a) {
  __shared__ __attribute__((aligned(1024))) uint16_t lds[Tile::kLds];
  GemmAcc<Tile> acc;
  const GemmPlace at = gemm_place(a.g);
  gemm_tile<Tile>(a.g, at, lds, acc);
  const int lane = threadIdx.x & (kWaveSize - 1), wave = threadIdx.x / kWaveSize;
  const int wm = wave / Tile::WN, wn = wave % Tile::WN;
  const int v0 = at.tm * Tile::BM + wm * (Tile::BM / Tile::WM);
  const int64_t n0 = static_cast<int64_t>(at.tn) * Tile::BN + wn * (Tile::BN / Tile::WN);
#pragma unroll
  for (int j = 0; j < Tile::TN; ++j) {
    const int64_t n = n0 + 32 * j + lane % 32;
    const bool row = n < a.g.b.rows;
    const int32_t label = row ? a.label[n] : -1;
    const float lse = row ? a.lse[n] : 0.0f, dl = label >= 0 ? a.dloss[n] : 0.0f;
    const int32_t hit = label >= 0 ? label - a.v0 - v0 : -1;  // row of this wave's block that is the label's
    const bool any_hit = __any(hit >= 0 && hit < Tile::BM / Tile::WM);
#pragma unroll
    for (int i = 0; i < Tile::TM; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        float x[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int r = 4 * q + k, v = 32 * i + acc_row(r, lane);
          float p = __builtin_amdgcn_exp2f((acc.c[i][j][r] - lse) * kLog2e);
          if (any_hit && v == hit) p -= 1.0f;
          x[k] = label >= 0 && v0 + v < a.g.a.rows ? p * dl : 0.0f;
          if (v0 + v < a.g.a.rows && n < a.pitch_n)
            store_parts<T>(a.vn, static_cast<int64_t>(v0 + v) * a.pitch_n + n, a.vn_part, x[k]);
        }
        const int v = v0 + 32 * i + acc_row(4 * q, lane);
        if (row && v < a.pitch_v) {
          uint16_t *to = a.nv + n * a.pitch_v + v;
          if constexpr (sizeof(T) == 4) {
            Pack<uint16_t, 4> y[kParts];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const Split s = split3(x[k]);
#pragma unroll
              for (int p = 0; p < kParts; ++p) y[p].v[k] = s.part[p];
            }
#pragma unroll
            for (int p = 0; p < kParts; ++p) *reinterpret_cast<Pack<uint16_t, 4> *>(to + p * a.nv_part) = y[p];
          } else {
            Pack<uint16_t, 4> y;
#pragma unroll
            for (int k = 0; k < 4; ++k) y.v[k] = bits_of(x[k]);
            *reinterpret_cast<Pack<uint16_t, 4> *>(to) = y;
          }
        }
      }
  }
}

struct StoreArgs {
  GemmShape g;
  void *out;               // [rows of a, rows of b] of T
  const int32_t *keep;     // rows of a to write as zeros where negative (null: none)
  float *part;             // or float32 sums of each split, [splits, part_stride], added to what is there
  int64_t part_stride;
  int32_t accumulate;
};

// kPartial: the sums go to a.part for join_kernel, else rounded to a.out.
template <typename Tile, typename T, bool kPartial>
__global__ __launch_bounds__(Tile::kThreads) void product_kernel(StoreArgs a) {
  __shared__ __attribute__((aligned(1024))) uint16_t lds[Tile::kLds];
  GemmAcc<Tile> acc;
  const GemmPlace at = gemm_place(a.g);
  gemm_tile<Tile>(a.g, at, lds, acc);
  const int lane = threadIdx.x & (kWaveSize - 1), wave = threadIdx.x / kWaveSize;
  const int wm = wave / Tile::WN, wn = wave % Tile::WN;
  const int64_t m0 = static_cast<int64_t>(at.tm) * Tile::BM + wm * (Tile::BM / Tile::WM);
  const int64_t n0 = static_cast<int64_t>(at.tn) * Tile::BN + wn * (Tile::BN / Tile::WN);
  float *part = kPartial ? a.part + at.split * a.part_stride : nullptr;
#pragma unroll
  for (int i = 0; i < Tile::TM; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int64_t m = m0 + 32 * i + acc_row(r, lane);
      if (m >= a.g.a.rows) continue;
      const bool zero = !kPartial && a.keep && a.keep[m] < 0;
#pragma unroll
      for (int j = 0; j < Tile::TN; ++j) {
        const int64_t n = n0 + 32 * j + lane % 32;
        if (n >= a.g.b.rows) continue;
        const int64_t to = m * a.g.b.rows + n;
        if constexpr (kPartial)
          part[to] = a.accumulate ? part[to] + acc.c[i][j][r] : acc.c[i][j][r];
        else
          static_cast<T *>(a.out)[to] = narrow<T>(zero ? 0.0f : acc.c[i][j][r]);
      }
    }
}

// out = sum over the splits, in order; rows with keep < 0 become zeros
template <typename T>
__global__ __launch_bounds__(kBlockThreads) void join_kernel(const float *part, int64_t part_stride, int32_t splits,
                                                             T *out, int64_t rows, int32_t D, const int32_t *keep) {
  const int64_t total = rows * D, stride = static_cast<int64_t>(gridDim.x) * kBlockThreads;
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * kBlockThreads + threadIdx.x; t < total; t += stride) {
    float s = 0.0f;
    for (int32_t z = 0; z < splits; ++z) s += part[z * part_stride + t];
    if (keep && keep[t / D] < 0) s = 0.0f;
    out[t] = narrow<T>(s);
  }
}

__global__ __launch_bounds__(kBlockThreads) void zero_kernel(uint16_t *out, int64_t n) {
  const int64_t stride = static_cast<int64_t>(gridDim.x) * kBlockThreads;
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * kBlockThreads + threadIdx.x; t < n; t += stride) out[t] = 0;
}

// ------------------------------------------------------------------------------------------------ host side
enum TileKind { kBig, kMid, kFlat, kTall };
struct TileSize {
  int bm, bn, per_cu;
  double rate;  // of the inner loop relative to the large tile
};
constexpr TileSize kTileSize[] = {{256, 256, 1, 1.0}, {128, 128, 2, 0.7}, {64, 256, 2, 0.6}, {256, 64, 2, 0.6}};
constexpr int kCus = 256;

int64_t up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }

// The tile whose rounds of workgroups over the device take the least time; tiles that can share a long k among
// several workgroups (`splittable`) are judged by their total work instead.
TileKind choose_tile(int64_t M, int64_t N, bool splittable) {
  if (const int forced = config().ce_tile) return static_cast<TileKind>(std::min(forced, 4) - 1);
  int best = kBig;
  double least = 0.0;
  for (int k = 0; k < 4; ++k) {
    const TileSize &s = kTileSize[k];
    const double tiles = static_cast<double>((M + s.bm - 1) / s.bm) * static_cast<double>((N + s.bn - 1) / s.bn);
    const double rounds = splittable ? std::max(1.0, tiles / (kCus * s.per_cu)) : std::ceil(tiles / (kCus * s.per_cu));
    const double cost = (splittable ? tiles / kCus : rounds * s.per_cu) * s.bm * s.bn / s.rate;
    if (k == 0 || cost < least) {
      best = k;
      least = cost;
    }
  }
  return static_cast<TileKind>(best);
}

// Workgroups per tile along k: enough to give every CU two, each with eight steps or more.
int choose_splits(TileKind kind, int64_t M, int64_t N, int64_t steps) {
  const TileSize &s = kTileSize[kind];
  const int64_t tiles = ((M + s.bm - 1) / s.bm) * ((N + s.bn - 1) / s.bn);
  const int64_t want = (kCus * s.per_cu + tiles - 1) / tiles;
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(want, steps / 8)));
}

constexpr int64_t kPieceBytes = int64_t{512} << 20;  // copies and G of one piece of the vocabulary

struct Layout {
  int parts, segments;
  bool packed;           // operands copied with k padded (float32, or rows that are no multiple of 64 or 16 bytes)
  int64_t Dp, Np;        // D and N to multiples of 64
  int64_t piece;         // vocabulary rows per piece, a multiple of 256
  TileKind logits, dh, dw;
  int dh_splits, dw_splits;
  int64_t h_pack, w_pack, stats, label, ht, wt, nv, vn, dh_part, dw_part, bytes;
};

Layout layout(int64_t N, int64_t V, int64_t D, int dtype, bool aligned, bool backward) {
  Layout l{};
  l.parts = dtype == FG_F32 ? kParts : 1;
  l.segments = dtype == FG_F32 ? kSegments : 1;
  l.packed = dtype == FG_F32 || D % kStepK != 0 || !aligned;
  l.Dp = up(D, kStepK);
  l.Np = up(N, kStepK);
  int64_t per_row = l.packed ? 2 * l.parts * l.Dp : 0;
  if (backward) per_row += 2 * l.parts * (2 * l.Np + D);
  l.piece = per_row ? std::max<int64_t>(256, std::min(up(V, 256), kPieceBytes / per_row / 256 * 256)) : up(V, 256);
  if (const int64_t rows = config().ce_piece_rows) l.piece = up(rows, 256);
  const int64_t in_piece = std::min(l.piece, V), piece_p = up(in_piece, kStepK);
  l.logits = choose_tile(in_piece, N, false);
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += up(bytes, 1024);
    return here;
  };
  l.h_pack = take(l.packed ? 2 * l.parts * N * l.Dp : 0);
  l.w_pack = take(l.packed ? 2 * l.parts * in_piece * l.Dp : 0);
  if (!backward) {
    const int64_t bm = kTileSize[l.logits].bm;
    l.stats = take(((V + l.piece - 1) / l.piece) * ((l.piece + bm - 1) / bm) * N * 8);
  } else {
    l.dh = choose_tile(N, D, true);
    l.dw = choose_tile(in_piece, D, true);
    l.dh_splits = choose_splits(l.dh, N, D, piece_p / kStepK * l.segments);
    l.dw_splits = choose_splits(l.dw, in_piece, D, l.Np / kStepK * l.segments);
    l.label = take(4 * N);
    l.ht = take(2 * l.parts * D * l.Np);
    l.wt = take(2 * l.parts * D * piece_p);
    l.nv = take(2 * l.parts * N * piece_p);
    l.vn = take(2 * l.parts * in_piece * l.Np);
    l.dh_part = take(l.dh_splits > 1 || V > l.piece ? 4 * l.dh_splits * N * D : 0);
    l.dw_part = take(l.dw_splits > 1 ? 4 * l.dw_splits * in_piece * D : 0);
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

template <typename T>
GemmOperand operand(const T *x, int64_t rows, int64_t D, const Layout &l, uint16_t *copy, hipStream_t stream) {
  GemmOperand o;
  o.rows = static_cast<int32_t>(rows);
  if (l.packed) {
    pack_kernel<T><<<dim3(flat_grid(rows * l.Dp)), dim3(kBlockThreads), 0, stream>>>(x, copy, rows, static_cast<int32_t>(D),
                                                                                    static_cast<int32_t>(l.Dp));
    o.p = copy;
    o.part = rows * l.Dp;
    o.pitch = l.Dp;
  } else {
    o.p = reinterpret_cast<const uint16_t *>(x);
    o.pitch = D;
  }
  return o;
}

template <typename T>
void transpose(const T *x, const int32_t *keep, uint16_t *out, int64_t rows, int64_t D, int64_t pitch, hipStream_t stream) {
  transpose_kernel<T><<<dim3(static_cast<unsigned>((pitch + 63) / 64), static_cast<unsigned>((D + 63) / 64)),
                        dim3(kBlockThreads), 0, stream>>>(x, keep, out, static_cast<int32_t>(rows),
                                                          static_cast<int32_t>(D), pitch);
}

template <typename T, typename Id>
int forward(int64_t N, int64_t V, int64_t D, const T *h, const T *w, const Id *labels, float *loss, float *lse,
            char *ws, const Layout &l, hipStream_t stream) {
  StatsArgs a{};
  a.part = reinterpret_cast<float2 *>(ws + l.stats);
  a.g.steps = static_cast<int32_t>(l.Dp / kStepK);
  a.g.segments = l.segments;
  a.g.b = operand(h, N, D, l, reinterpret_cast<uint16_t *>(ws + l.h_pack), stream);
  for (int64_t v0 = 0; v0 < V; v0 += l.piece) {
    a.g.a = operand(w + v0 * D, std::min(l.piece, V - v0), D, l, reinterpret_cast<uint16_t *>(ws + l.w_pack), stream);
    const int rc = with_tile(l.logits, &a.g, [&](auto tile, dim3 grid) {
      using Tile = decltype(tile);
      stats_kernel<Tile><<<grid, dim3(Tile::kThreads), 0, stream>>>(a);
    });
    if (rc) return rc;
    a.tile0 += a.g.tiles_m;
  }
  loss_kernel<T, Id><<<dim3(static_cast<unsigned>((N + kWaveSize - 1) / kWaveSize)), dim3(kLossThreads), 0, stream>>>(
      a.part, a.tile0, h, w, labels, static_cast<int32_t>(N), V, static_cast<int32_t>(D), loss, lse);
  FG_HIP_TRY(hipGetLastError());
  return FG_OK;
}

// out[M, D] = the product, through partial sums where k is shared or earlier pieces have added to them
template <typename T>
int product(TileKind kind, StoreArgs a, T *out, bool partial, hipStream_t stream) {
  a.out = out;
  return with_tile(kind, &a.g, [&](auto tile, dim3 grid) {
    using Tile = decltype(tile);
    if (partial)
      product_kernel<Tile, T, true><<<grid, dim3(Tile::kThreads), 0, stream>>>(a);
    else
      product_kernel<Tile, T, false><<<grid, dim3(Tile::kThreads), 0, stream>>>(a);
  });
}

template <typename T>
int backward(int64_t N, int64_t V, int64_t D, const T *h, const T *w, const float *lse, const float *dloss, T *dh,
             T *dw, char *ws, const Layout &l, hipStream_t stream) {
  const int32_t *label = reinterpret_cast<const int32_t *>(ws + l.label);
  auto *ht = reinterpret_cast<uint16_t *>(ws + l.ht), *wt = reinterpret_cast<uint16_t *>(ws + l.wt);
  auto *nv = reinterpret_cast<uint16_t *>(ws + l.nv), *vn = reinterpret_cast<uint16_t *>(ws + l.vn);
  GradArgs a{};
  a.label = label;
  a.lse = lse;
  a.dloss = dloss;
  a.nv = nv;
  a.vn = vn;
  a.pitch_n = static_cast<int32_t>(l.Np);
  a.g.steps = static_cast<int32_t>(l.Dp / kStepK);
  a.g.segments = l.segments;
  a.g.b = operand(h, N, D, l, reinterpret_cast<uint16_t *>(ws + l.h_pack), stream);
  transpose(h, label, ht, N, D, l.Np, stream);
  const bool dh_partial = l.dh_splits > 1 || V > l.piece;
  for (int64_t v0 = 0; v0 < V; v0 += l.piece) {
    const int64_t rows = std::min(l.piece, V - v0), rows_p = up(rows, kStepK);
    a.v0 = static_cast<int32_t>(v0);
    a.pitch_v = static_cast<int32_t>(rows_p);
    a.nv_part = N * rows_p;
    a.vn_part = rows * l.Np;
    a.g.a = operand(w + v0 * D, rows, D, l, reinterpret_cast<uint16_t *>(ws + l.w_pack), stream);
    int rc = with_tile(l.logits, &a.g, [&](auto tile, dim3 grid) {
      using Tile = decltype(tile);
      grad_logits_kernel<Tile, T><<<grid, dim3(Tile::kThreads), 0, stream>>>(a);
    });
    if (rc) return rc;
    transpose(w + v0 * D, static_cast<const int32_t *>(nullptr), wt, rows, D, rows_p, stream);

    StoreArgs s{};  // dw[v, d] = sum over n of G[v, n] * h[n, d]
    s.g.segments = l.segments;
    s.g.steps = static_cast<int32_t>(l.Np / kStepK);
    s.g.splits = l.dw_splits;
    s.g.a = GemmOperand{vn, a.vn_part, l.Np, static_cast<int32_t>(rows)};
    s.g.b = GemmOperand{ht, D * l.Np, l.Np, static_cast<int32_t>(D)};
    s.part = reinterpret_cast<float *>(ws + l.dw_part);
    s.part_stride = rows * D;
    rc = product<T>(l.dw, s, dw + v0 * D, l.dw_splits > 1, stream);
    if (rc) return rc;
    if (l.dw_splits > 1)
      join_kernel<T><<<dim3(flat_grid(rows * D)), dim3(kBlockThreads), 0, stream>>>(
          s.part, s.part_stride, l.dw_splits, dw + v0 * D, rows, static_cast<int32_t>(D), nullptr);

    s.g.steps = static_cast<int32_t>(rows_p / kStepK);  // dh[n, d] = sum over v of G[n, v] * w[v, d]
    s.g.splits = l.dh_splits;
    s.g.a = GemmOperand{nv, a.nv_part, rows_p, static_cast<int32_t>(N)};
    s.g.b = GemmOperand{wt, D * rows_p, rows_p, static_cast<int32_t>(D)};
    s.keep = label;
    s.part = reinterpret_cast<float *>(ws + l.dh_part);
    s.part_stride = N * D;
    s.accumulate = v0 > 0;
    rc = product<T>(l.dh, s, dh, dh_partial, stream);
    if (rc) return rc;
  }
  if (dh_partial)
    join_kernel<T><<<dim3(flat_grid(N * D)), dim3(kBlockThreads), 0, stream>>>(
        reinterpret_cast<float *>(ws + l.dh_part), N * D, l.dh_splits, dh, N, static_cast<int32_t>(D), label);
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
  const dim3 grid(static_cast<unsigned>((N + fg::kBlockThreads - 1) / fg::kBlockThreads));
  if (itype == FG_I32)
    fg::labels_kernel<int32_t><<<grid, dim3(fg::kBlockThreads), 0, s>>>(static_cast<const int32_t *>(labels), static_cast<int32_t>(N), V, label);
  else
    fg::labels_kernel<int64_t><<<grid, dim3(fg::kBlockThreads), 0, s>>>(static_cast<const int64_t *>(labels), static_cast<int32_t>(N), V, label);
#define FG_TYPED(T)                                                                                              \
  fg::backward<T>(N, V, D, static_cast<const T *>(hidden), static_cast<const T *>(weight), lse, dloss,           \
                  static_cast<T *>(dhidden), static_cast<T *>(dweight), ws, l, s)
  return dtype == FG_F32 ? FG_TYPED(float) : FG_TYPED(__bf16);
#undef FG_TYPED
}

}  // extern "C"
