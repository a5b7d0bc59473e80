// Embedding lookup with scaling, and its gradient.
//
//   lookup     out[i, :]   = scale * table[id[i], :]
//   gradient   grad[v, :]  = scale * sum over i with id[i] = v of dout[i, :]
//
// An id outside [0, V) is padding: its output row is zero and it adds nothing to the gradient.  Sums are held in
// float32 and rounded once to the element type.
//
// The gradient is a sum over runs of a sorted list, so that no atomic decides an order: the positions are sorted by
// id (stably, so equal ids keep their order), the sorted list is cut into chunks, a group of lanes walks each chunk
// and adds the rows of each run.  A run inside one chunk is written out at once; of a run that crosses a chunk's
// border each chunk leaves a partial row (at most two per chunk: its first and its last run), and the partial rows,
// again a sorted list, are added the same way until few are left.  The order of every sum depends on the ids and the sizes alone.
#include <algorithm>
#include <initializer_list>
#include <type_traits>

#include "element.hpp"

namespace fg {
namespace {

constexpr int kRankSortMost = 12288;  // ids that the one-launch sort takes (48 KB of LDS)
constexpr int kRankThreads = 1024;
constexpr int kRadixBits = 11;        // most bits per pass
constexpr int32_t kSkip = INT32_MIN;  // flag on a partial row's key: nothing there to add

int lanes_per_row(int64_t D, int vec) {
  int l = 1;
  while (l < kWaveSize && static_cast<int64_t>(l) * vec < D) l <<= 1;
  return l;
}

template <typename Id>
__device__ __forceinline__ int32_t key_of(Id id, int32_t V) {
  return id >= 0 && id < static_cast<Id>(V) ? static_cast<int32_t>(id) : V;
}
__device__ __forceinline__ int32_t key_of(int2 entry, int32_t) { return entry.x; }  // of a list sorted before

// ------------------------------------------------------------------------------------------------ lookup
// A group of lpr lanes copies kRows rows at a time, each lane VEC elements of each: all ids first, then all rows,
// so that kRows gathers are in flight per lane.
template <typename T, typename Id, int VEC>
__global__ __launch_bounds__(kBlockThreads) void lookup_kernel(const T *table, const Id *ids, T *out, int64_t n,
                                                               int32_t V, int32_t D, int lpr, float scale) {
  constexpr int kRows = 4;
  using P = Pack<T, VEC>;
  const int sub = threadIdx.x & (lpr - 1);
  const int64_t group = (static_cast<int64_t>(blockIdx.x) * kBlockThreads + threadIdx.x) / lpr;
  const int64_t first = group * kRows;
  if (first >= n) return;
  int32_t key[kRows];
#pragma unroll
  for (int r = 0; r < kRows; ++r) key[r] = first + r < n ? key_of(ids[first + r], V) : V;
  for (int32_t c = (blockIdx.y * lpr + sub) * VEC; c < D; c += gridDim.y * lpr * VEC) {
    P x[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r)
      if (key[r] < V) x[r] = *reinterpret_cast<const P *>(table + static_cast<int64_t>(key[r]) * D + c);
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      if (first + r >= n) break;
      P y;
#pragma unroll
      for (int k = 0; k < VEC; ++k) y.v[k] = key[r] < V ? narrow<T>(widen(x[r].v[k]) * scale) : narrow<T>(0.0f);
      *reinterpret_cast<P *>(out + (first + r) * D + c) = y;
    }
  }
}

// ------------------------------------------------------------------------------------------------ sort
// Up to kRankSortMost ids: the place of id i is the number of ids below it plus the number of equal ids before it,
// counted directly.  A workgroup holds all ids in LDS and places 64 of them; each of its 16 waves counts over a
// sixteenth of the list, four ids per LDS read.  N * N / 64 wave steps, but one launch: whole gradients take 26, 37,
// 44 and 49 us for 4100, 10000, 13978 and 16384 ids where those with the six launches of the radix sort take 41, 42, 43 and 43.
template <typename Id>
__global__ __launch_bounds__(kRankThreads) void rank_sort_kernel(const Id *ids, int32_t n, int32_t V, int2 *sorted) {
  constexpr int kWaves = kRankThreads / kWaveSize;
  __shared__ int4 all[kRankSortMost / 4];
  __shared__ int32_t count[kWaves][kWaveSize];
  int32_t *flat = reinterpret_cast<int32_t *>(all);
  const int padded = (n + 4 * kWaves - 1) / (4 * kWaves) * (4 * kWaves);
  for (int j = threadIdx.x; j < padded; j += kRankThreads) flat[j] = j < n ? key_of(ids[j], V) : INT32_MAX;
  __syncthreads();
  const int lane = threadIdx.x & (kWaveSize - 1), wave = threadIdx.x / kWaveSize;
  const int base = blockIdx.x * kWaveSize, i = base + lane;
  const int32_t mine = i < n ? flat[i] : -1;
  const int quads = padded / 4, share = quads / kWaves;
  int32_t below = 0;
  int q = wave * share;
  const int end = q + share;
  for (; q < min(end, base / 4); ++q) {  // ids before this workgroup's: equal ones count
    const int4 k = all[q];
    below += (k.x <= mine) + (k.y <= mine) + (k.z <= mine) + (k.w <= mine);
  }
  for (; q < min(end, (base + kWaveSize) / 4); ++q) {
    const int4 k = all[q];
    const int j = q * 4;
    below += (k.x < mine || (k.x == mine && j < i)) + (k.y < mine || (k.y == mine && j + 1 < i)) +
             (k.z < mine || (k.z == mine && j + 2 < i)) + (k.w < mine || (k.w == mine && j + 3 < i));
  }
  for (; q < end; ++q) {
    const int4 k = all[q];
    below += (k.x < mine) + (k.y < mine) + (k.z < mine) + (k.w < mine);
  }
  count[wave][lane] = below;
  __syncthreads();
  if (wave == 0 && i < n) {
    int place = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) place += count[w][lane];
    sorted[place] = int2{mine, i};
  }
}

// The sorted list holds {key, position} pairs, which a scatter writes in one piece.
// More ids: least-significant-digit radix sort, digits of up to kRadixBits bits (two passes up to 4M rows), three
// launches per pass: counts per workgroup and digit, a scan of each digit's counts over the workgroups, the scatter.
template <typename Id, int kItems>
__global__ __launch_bounds__(kBlockThreads) void radix_count_kernel(const Id *keys, int32_t n, int32_t V, int shift,
                                                                    int bits, int32_t *counts) {
  __shared__ int32_t hist[1 << kRadixBits];
  const int digits = 1 << bits;
  for (int d = threadIdx.x; d < digits; d += kBlockThreads) hist[d] = 0;
  __syncthreads();
  const int64_t lo = static_cast<int64_t>(blockIdx.x) * kItems;
#pragma unroll
  for (int r = 0; r < kItems / kBlockThreads; ++r) {
    const int64_t i = lo + r * kBlockThreads + threadIdx.x;
    if (i < n) atomicAdd(&hist[(key_of(keys[i], V) >> shift) & (digits - 1)], 1);
  }
  __syncthreads();
  for (int d = threadIdx.x; d < digits; d += kBlockThreads)
    counts[static_cast<int64_t>(d) * gridDim.x + blockIdx.x] = hist[d];
}

// One wave per digit: exclusive scan of its counts over the workgroups, in place, and their total.
__global__ __launch_bounds__(kBlockThreads) void radix_scan_kernel(int32_t *counts, int32_t blocks, int32_t digits,
                                                                   int32_t *totals) {
  const int lane = threadIdx.x & (kWaveSize - 1);
  const int d = blockIdx.x * kWavesPerBlock + threadIdx.x / kWaveSize;
  if (d >= digits) return;
  int32_t *c = counts + static_cast<int64_t>(d) * blocks;
  int32_t before = 0;
  for (int32_t b = 0; b < blocks; b += kWaveSize) {
    const int32_t x = b + lane < blocks ? c[b + lane] : 0;
    int32_t s = x;
#pragma unroll
    for (int k = 1; k < kWaveSize; k <<= 1) {
      const int32_t y = __shfl_up(s, k, kWaveSize);
      if (lane >= k) s += y;
    }
    if (b + lane < blocks) c[b + lane] = before + s - x;
    before += __shfl(s, kWaveSize - 1, kWaveSize);
  }
  if (lane == 0) totals[d] = before;
}

// A wave ranks its consecutive kItems / 4 keys, 64 at a time: lanes of equal digit find each other by one ballot
// per bit, the first of them takes their places from the wave's counter of that digit.
template <typename Id, bool kFirst, int kItems>
__global__ __launch_bounds__(kBlockThreads) void radix_scatter_kernel(const Id *keys, int32_t n, int32_t V, int shift,
                                                                      int bits, const int32_t *counts,
                                                                      const int32_t *totals, int2 *sorted) {
  constexpr int kMost = 1 << kRadixBits, kRounds = kItems / kBlockThreads;
  __shared__ int32_t taken[kWavesPerBlock][kMost];  // per wave and digit: keys ranked so far
  __shared__ int32_t base[kMost];                   // first place of each digit for this workgroup
  __shared__ int32_t sums[kBlockThreads];
  const int digits = 1 << bits, lane = threadIdx.x & (kWaveSize - 1), wave = threadIdx.x / kWaveSize;
  const int64_t lo = static_cast<int64_t>(blockIdx.x) * kItems + wave * (kItems / kWavesPerBlock);
  int32_t key[kRounds], from[kRounds], rank[kRounds];
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const int64_t i = lo + r * kWaveSize + lane;
    key[r] = 0;
    from[r] = -1;
    if (i < n) {
      const Id x = keys[i];
      key[r] = key_of(x, V);
      if constexpr (kFirst) from[r] = static_cast<int32_t>(i);
      else from[r] = x.y;
    }
  }
  for (int d = threadIdx.x; d < digits; d += kBlockThreads) {
    base[d] = totals[d];
#pragma unroll
    for (int w = 0; w < kWavesPerBlock; ++w) taken[w][d] = 0;
  }
  __syncthreads();
  {  // exclusive scan of the totals over the digits: each thread owns `per` neighbouring digits
    const int per = (digits + kBlockThreads - 1) / kBlockThreads, d0 = threadIdx.x * per;
    int32_t s = 0;
    for (int k = 0; k < per; ++k) s += d0 + k < digits ? base[d0 + k] : 0;
    sums[threadIdx.x] = s;
    __syncthreads();
    for (int k = 1; k < kBlockThreads; k <<= 1) {
      const int32_t y = static_cast<int>(threadIdx.x) >= k ? sums[threadIdx.x - k] : 0;
      __syncthreads();
      sums[threadIdx.x] += y;
      __syncthreads();
    }
    int32_t before = threadIdx.x ? sums[threadIdx.x - 1] : 0;
    for (int k = 0; k < per; ++k) {
      if (d0 + k >= digits) break;
      const int32_t x = base[d0 + k];
      base[d0 + k] = before + counts[static_cast<int64_t>(d0 + k) * gridDim.x + blockIdx.x];
      before += x;
    }
  }
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const int d = (key[r] >> shift) & (digits - 1);
    uint64_t peers = __ballot(from[r] >= 0);
    for (int b = 0; b < bits; ++b) {
      const uint64_t set = __ballot((d >> b) & 1);
      peers &= (d >> b) & 1 ? set : ~set;
    }
    const int leader = peers ? __ffsll(static_cast<unsigned long long>(peers)) - 1 : lane;
    int32_t old = 0;
    if (from[r] >= 0 && lane == leader) old = atomicAdd(&taken[wave][d], __popcll(peers));
    rank[r] = __shfl(old, leader, kWaveSize) + __popcll(peers & ((uint64_t{1} << lane) - 1));
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    if (from[r] < 0) continue;
    const int d = (key[r] >> shift) & (digits - 1);
    int32_t place = base[d] + rank[r];
    for (int w = 0; w < wave; ++w) place += taken[w][d];
    sorted[place] = int2{key[r], from[r]};
  }
}

// ------------------------------------------------------------------------------------------------ sums over runs
template <typename T, int VEC>
__device__ __forceinline__ void write_row(T *grad, int64_t at, const float *acc, float scale, int accumulate) {
  using P = Pack<T, VEC>;
  P y;
  if (accumulate) {
    y = *reinterpret_cast<const P *>(grad + at);
#pragma unroll
    for (int k = 0; k < VEC; ++k) y.v[k] = narrow<T>(__builtin_fmaf(acc[k], scale, widen(y.v[k])));
  } else {
#pragma unroll
    for (int k = 0; k < VEC; ++k) y.v[k] = narrow<T>(acc[k] * scale);
  }
  *reinterpret_cast<P *>(grad + at) = y;
}

struct RunArgs {
  const int2 *sorted;   // [n] first level: {key, row}, keys ascending
  const int32_t *keys;  // [n] later levels: keys of the rows, ascending, with kSkip set where there is nothing to add
  int64_t n;
  int32_t chunk;        // entries per group
  int32_t V, D;
  int lpr, accumulate;
  int fill_blocks;      // workgroups ahead of the others that write zeros into the absent rows
  int fill_rows, fill_lpr;  // rows per wave of these, lanes per row (0: ranges)
  float scale;
  float *part;          // [2 * chunks, D] partial rows, slots 2c and 2c + 1 for the first and last run of chunk c
  int32_t *part_keys;   // [2 * chunks]
};

// Zeros in the rows that no id names.  A wave looks `fill_rows` rows up in the sorted ids (one binary search per lane),
// then writes those of them that are absent: row by row where rows are whole 16-byte pieces of memory, else neighbouring
// absent rows as one range, whose pieces are whole but for the first and the last.
template <typename T>
__device__ __forceinline__ void zero_absent(const RunArgs &a, T *grad) {
  const int lane = threadIdx.x & (kWaveSize - 1);
  const int64_t r0 = (static_cast<int64_t>(blockIdx.x) * kWavesPerBlock + threadIdx.x / kWaveSize) * a.fill_rows;
  if (r0 >= a.V) return;
  const int32_t n = static_cast<int32_t>(a.n);
  const bool asks = lane < a.fill_rows && r0 + lane < a.V;
  int32_t lo = 0, hi = asks ? n : 0;
  while (lo < hi) {
    const int32_t m = lo + (hi - lo) / 2;
    if (a.sorted[m].x < r0 + lane) lo = m + 1; else hi = m;
  }
  uint64_t absent = __ballot(asks && !(lo < n && a.sorted[lo].x == r0 + lane));
  constexpr int64_t kPiece = 16 / sizeof(T);
  if (a.fill_lpr) {
    const int sub = lane & (a.fill_lpr - 1);
    for (int r = lane / a.fill_lpr; r < a.fill_rows; r += kWaveSize / a.fill_lpr) {
      if (!((absent >> r) & 1)) continue;
      for (int64_t c = (static_cast<int64_t>(blockIdx.y) * a.fill_lpr + sub) * kPiece; c < a.D;
           c += static_cast<int64_t>(gridDim.y) * a.fill_lpr * kPiece)
        *reinterpret_cast<uint4 *>(grad + (r0 + r) * a.D + c) = uint4{0, 0, 0, 0};
    }
    return;
  }
  const int64_t ahead = reinterpret_cast<uintptr_t>(grad) % 16 / sizeof(T);  // elements between a 16-byte boundary and grad
  while (absent) {
    const int start = __ffsll(static_cast<unsigned long long>(absent)) - 1;
    const uint64_t others = ~(absent >> start);
    const int rows = others ? __ffsll(static_cast<unsigned long long>(others)) - 1 : kWaveSize;
    absent = start + rows < kWaveSize ? absent >> (start + rows) << (start + rows) : 0;
    const int64_t first = (r0 + start) * a.D, last = first + static_cast<int64_t>(rows) * a.D;
    const int64_t begin = (first + ahead) / kPiece * kPiece - ahead;
    for (int64_t c = begin + (static_cast<int64_t>(blockIdx.y) * kWaveSize + lane) * kPiece; c < last;
         c += static_cast<int64_t>(gridDim.y) * kWaveSize * kPiece) {
      if (c >= first && c + kPiece <= last) {
        *reinterpret_cast<uint4 *>(grad + c) = uint4{0, 0, 0, 0};
      } else {
        for (int64_t k = max(c, first); k < min(c + kPiece, last); ++k) grad[k] = narrow<T>(0.0f);
      }
    }
  }
}

// S: element type of the rows that are added (the gradient's own on the first level, then float).
template <typename S, typename T, int VEC, bool kFirst>
__global__ __launch_bounds__(kBlockThreads) void run_sums_kernel(RunArgs a, const S *rows, T *grad) {
  if (static_cast<int>(blockIdx.x) < a.fill_blocks) {
    zero_absent(a, grad);
    return;
  }
  constexpr int kAhead = 8;  // rows under way per lane
  using P = Pack<S, VEC>;
  const int sub = threadIdx.x & (a.lpr - 1);
  const int64_t c = ((static_cast<int64_t>(blockIdx.x) - a.fill_blocks) * kBlockThreads + threadIdx.x) / a.lpr;
  const int64_t lo = c * a.chunk, hi = min(lo + a.chunk, a.n);
  if (lo >= a.n) return;
  const int32_t col = (blockIdx.y * a.lpr + sub) * VEC;
  const bool mine = col < a.D, keeper = blockIdx.y == 0 && sub == 0;
  auto entry = [&](int64_t e) {
    if constexpr (kFirst) return a.sorted[e];
    else return int2{a.keys[e], 0};
  };
  const int32_t prev = lo > 0 ? entry(lo - 1).x & ~kSkip : -1, next = hi < a.n ? entry(hi).x & ~kSkip : -1;
  int32_t cur = entry(lo).x & ~kSkip;
  const int32_t first_key = cur;
  bool first = true, any = false, head = false, tail = false;  // head / tail: the two slots hold something
  float acc[VEC] = {};
  auto flush = [&](bool last) {
    const bool whole = !(first && prev == cur) && !(last && next == cur);
    if (any) {
      if (whole) {
        if (mine) write_row<T, VEC>(grad, static_cast<int64_t>(cur) * a.D + col, acc, a.scale, a.accumulate);
      } else {
        (first ? head : tail) = true;
        if (mine) {
          float *p = a.part + (2 * c + (first ? 0 : 1)) * a.D + col;
#pragma unroll
          for (int k = 0; k < VEC; ++k) p[k] = acc[k];
        }
      }
    }
  };
  for (int64_t e = lo; e < hi; e += kAhead) {
    int32_t key[kAhead], row[kAhead];
    P x[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int2 y = e + u < hi ? entry(e + u) : int2{a.V, 0};
      key[u] = y.x;
      row[u] = y.y;
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (key[u] >= 0 && key[u] < a.V && mine) {
        const int64_t r = kFirst ? row[u] : e + u;
        x[u] = *reinterpret_cast<const P *>(rows + r * a.D + col);
      }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (e + u >= hi) break;
      const int32_t k = key[u] & ~kSkip;
      if (k != cur) {
        flush(false);
        cur = k;
        first = any = false;
#pragma unroll
        for (int j = 0; j < VEC; ++j) acc[j] = 0.0f;
      }
      if (key[u] >= 0 && key[u] < a.V) {
        any = true;
        if (mine) {
#pragma unroll
          for (int j = 0; j < VEC; ++j) acc[j] += widen(x[u].v[j]);
        }
      }
    }
  }
  flush(true);
  if (keeper) {
    a.part_keys[2 * c] = first_key | (head ? 0 : kSkip);
    a.part_keys[2 * c + 1] = cur | (tail ? 0 : kSkip);
  }
}

// The last level: the group at a run's first entry adds the whole run.
template <typename T, int VEC>
__global__ __launch_bounds__(kBlockThreads) void run_join_kernel(RunArgs a, const float *rows, T *grad) {
  const int sub = threadIdx.x & (a.lpr - 1);
  const int64_t e0 = (static_cast<int64_t>(blockIdx.x) * kBlockThreads + threadIdx.x) / a.lpr;
  if (e0 >= a.n) return;
  const int32_t k = a.keys[e0] & ~kSkip;
  if (k >= a.V || (e0 > 0 && (a.keys[e0 - 1] & ~kSkip) == k)) return;
  const int32_t col = (blockIdx.y * a.lpr + sub) * VEC;
  if (col >= a.D) return;
  constexpr int kAhead = 8;
  float acc[VEC] = {};
  bool any = false, more = true;
  for (int64_t e = e0; more && e < a.n; e += kAhead) {
    int32_t key[kAhead];
    Pack<float, VEC> x[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      key[u] = e + u < a.n ? a.keys[e + u] : -1;
      if (e + u < a.n) x[u] = *reinterpret_cast<const Pack<float, VEC> *>(rows + (e + u) * a.D + col);
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      more = more && e + u < a.n && (key[u] & ~kSkip) == k;
      if (!more || key[u] < 0) continue;
      any = true;
#pragma unroll
      for (int j = 0; j < VEC; ++j) acc[j] += x[u].v[j];
    }
  }
  if (any) write_row<T, VEC>(grad, static_cast<int64_t>(k) * a.D + col, acc, a.scale, a.accumulate);
}

// ------------------------------------------------------------------------------------------------ host side
int64_t align256(int64_t b) { return (b + 255) & ~int64_t{255}; }

// Ids per workgroup of the radix sort: few for a short list, which would not fill the device, more for a long one, whose
// counts per workgroup and digit are traffic (164,864 ids: 36 us with 1024, 44 with 2048; 1,000,003: 150 and 120).
int radix_items(int64_t n) { return n <= 524288 ? 1024 : 4096; }

// Entries per group on the first level: short chunks where the list is short (more groups in flight), longer ones
// where it is long (fewer partial rows).
int32_t chunk_of(int64_t n) { return n <= 8192 ? 4 : n <= 65536 ? 8 : n <= 524288 ? 16 : 64; }
constexpr int32_t kNextChunk = 8;    // ... on the levels after it
constexpr int64_t kJoinMost = 2048;  // partial rows that one group may have to join at the end (all ids equal)
constexpr int64_t kFillWaves = 512;  // below which a wave takes fewer rows to zero
constexpr int kMostLevels = 14;      // each leaves a quarter of the partial rows

struct GradLayout {
  int64_t sorted[2], counts, totals, bytes;
  int levels;
  int64_t chunks[kMostLevels], part[kMostLevels], part_keys[kMostLevels];
};

GradLayout grad_layout(int64_t n, int64_t D) {
  GradLayout g{};
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += align256(bytes);
    return here;
  };
  const int64_t blocks = (n + radix_items(n) - 1) / radix_items(n);
  for (int k = 0; k < 2; ++k) g.sorted[k] = take(n * 8);
  g.counts = take(n > kRankSortMost ? blocks * (int64_t{4} << kRadixBits) : 0);
  g.totals = take(int64_t{4} << kRadixBits);
  int64_t entries = n;
  while (g.levels == 0 || entries > kJoinMost) {
    const int32_t chunk = g.levels ? kNextChunk : chunk_of(n);
    g.chunks[g.levels] = (entries + chunk - 1) / chunk;
    entries = 2 * g.chunks[g.levels];
    g.part[g.levels] = take(entries * D * 4);
    g.part_keys[g.levels] = take(entries * 4);
    ++g.levels;
  }
  g.bytes = at;
  return g;
}

unsigned blocks_for(int64_t groups, int lpr) {
  const int64_t per = kBlockThreads / lpr;
  return static_cast<unsigned>((groups + per - 1) / per);
}

template <typename Id>
int sort_ids(const Id *ids, int32_t n, int32_t V, char *ws, const GradLayout &g, const int2 **sorted, hipStream_t stream) {
  auto *s0 = reinterpret_cast<int2 *>(ws + g.sorted[0]), *s1 = reinterpret_cast<int2 *>(ws + g.sorted[1]);
  if (n <= kRankSortMost) {
    rank_sort_kernel<Id><<<dim3((n + kWaveSize - 1) / kWaveSize), dim3(kRankThreads), 0, stream>>>(ids, n, V, s0);
    FG_HIP_TRY(hipGetLastError());
    *sorted = s0;
    return FG_OK;
  }
  int total_bits = 1;
  while (total_bits < 31 && (V >> total_bits) != 0) ++total_bits;  // keys 0 .. V
  const int passes = (total_bits + kRadixBits - 1) / kRadixBits, bits = (total_bits + passes - 1) / passes;
  const int32_t blocks = static_cast<int32_t>((static_cast<int64_t>(n) + radix_items(n) - 1) / radix_items(n));
  auto *counts = reinterpret_cast<int32_t *>(ws + g.counts), *totals = reinterpret_cast<int32_t *>(ws + g.totals);
  auto sort = [&](auto items) {
    constexpr int kItems = decltype(items)::value;
    for (int p = 0; p < passes; ++p) {
      const int shift = p * bits;
      if (p == 0)
        radix_count_kernel<Id, kItems><<<dim3(blocks), dim3(kBlockThreads), 0, stream>>>(ids, n, V, shift, bits, counts);
      else
        radix_count_kernel<int2, kItems><<<dim3(blocks), dim3(kBlockThreads), 0, stream>>>(s0, n, V, shift, bits, counts);
      radix_scan_kernel<<<dim3(((1 << bits) + kWavesPerBlock - 1) / kWavesPerBlock), dim3(kBlockThreads), 0, stream>>>(
          counts, blocks, 1 << bits, totals);
      if (p == 0)
        radix_scatter_kernel<Id, true, kItems><<<dim3(blocks), dim3(kBlockThreads), 0, stream>>>(
            ids, n, V, shift, bits, counts, totals, s1);
      else
        radix_scatter_kernel<int2, false, kItems><<<dim3(blocks), dim3(kBlockThreads), 0, stream>>>(
            s0, n, V, shift, bits, counts, totals, s1);
      std::swap(s0, s1);
    }
  };
  if (radix_items(n) == 1024) sort(std::integral_constant<int, 1024>{});
  else sort(std::integral_constant<int, 4096>{});
  FG_HIP_TRY(hipGetLastError());
  *sorted = s0;
  return FG_OK;
}

template <typename T, int VEC>
int grad_rows(const int2 *sorted, int64_t n, int64_t V, int64_t D, const T *dout, T *grad,
              float scale, int accumulate, char *ws, const GradLayout &g, hipStream_t stream) {
  const int lpr = lanes_per_row(D, VEC);
  const unsigned tiles = static_cast<unsigned>((D + lpr * VEC - 1) / (lpr * VEC));
  RunArgs a{};
  a.sorted = sorted;
  a.n = n;
  a.V = static_cast<int32_t>(V);
  a.D = static_cast<int32_t>(D);
  a.lpr = lpr;
  a.accumulate = accumulate;
  a.scale = scale;
  // a wave takes 64 rows, fewer where that leaves few waves: more waves search longer than they write (with 512, 1024 and
  // 2048 as the limit: 4 ids into 104,121 x 201 float16 13.6, 14.0, 16.3 us; 13,978 into 48,525 x 161 bfloat16 51, 54, 55;
  // 2 into 1105 x 971 float16 13 with each, 40 with 64 rows a wave and stores of single elements)
  a.fill_rows = kWaveSize;
  while (a.fill_rows > 4 && V < a.fill_rows * kFillWaves) a.fill_rows /= 4;
  a.fill_lpr = VEC * sizeof(T) == 16 ? lpr : 0;
  const int64_t fill_rows = static_cast<int64_t>(a.fill_rows) * kWavesPerBlock;
  a.fill_blocks = accumulate ? 0 : static_cast<int>((V + fill_rows - 1) / fill_rows);
  const float *rows = nullptr;
  for (int k = 0; k < g.levels; ++k) {
    a.chunk = k ? kNextChunk : chunk_of(n);
    a.part = reinterpret_cast<float *>(ws + g.part[k]);
    a.part_keys = reinterpret_cast<int32_t *>(ws + g.part_keys[k]);
    const dim3 grid(a.fill_blocks + blocks_for(g.chunks[k], lpr), tiles);
    if (k == 0)
      run_sums_kernel<T, T, VEC, true><<<grid, dim3(kBlockThreads), 0, stream>>>(a, dout, grad);
    else
      run_sums_kernel<float, T, VEC, false><<<grid, dim3(kBlockThreads), 0, stream>>>(a, rows, grad);
    if (n == 0) {
      FG_HIP_TRY(hipGetLastError());
      return FG_OK;
    }
    rows = a.part;
    a.keys = a.part_keys;
    a.n = 2 * g.chunks[k];
    a.fill_blocks = 0;
  }
  run_join_kernel<T, VEC><<<dim3(blocks_for(a.n, lpr), tiles), dim3(kBlockThreads), 0, stream>>>(a, rows, grad);
  FG_HIP_TRY(hipGetLastError());
  return FG_OK;
}

template <typename T>
int grad_typed(const int2 *sorted, int64_t n, int64_t V, int64_t D, const void *dout, void *grad,
               float scale, int accumulate, char *ws, const GradLayout &g, hipStream_t stream) {
  const T *d = static_cast<const T *>(dout);
  T *o = static_cast<T *>(grad);
  switch (vector_elements(D, sizeof(T), {dout, grad})) {
    case 8:
      if constexpr (sizeof(T) == 2) return grad_rows<T, 8>(sorted, n, V, D, d, o, scale, accumulate, ws, g, stream);
      [[fallthrough]];
    case 4: return grad_rows<T, 4>(sorted, n, V, D, d, o, scale, accumulate, ws, g, stream);
    case 2: return grad_rows<T, 2>(sorted, n, V, D, d, o, scale, accumulate, ws, g, stream);
    default: return grad_rows<T, 1>(sorted, n, V, D, d, o, scale, accumulate, ws, g, stream);
  }
}

template <typename T, typename Id>
int lookup_typed(const void *table, const void *ids, void *out, int64_t n, int64_t V, int64_t D, float scale,
                 hipStream_t stream) {
  const T *t = static_cast<const T *>(table);
  const int vec = vector_elements(D, sizeof(T), {table, out}), lpr = lanes_per_row(D, vec);
  // A launch has fewer than 2^32 threads along x, and a row takes up to 16: 2^26 ids (2^30 threads) at a time.
  constexpr int64_t kMostIds = 1 << 26;
  for (int64_t from = 0; from < n; from += kMostIds) {
    const Id *i = static_cast<const Id *>(ids) + from;
    T *o = static_cast<T *>(out) + from * D;
    const int64_t count = std::min(kMostIds, n - from);
    const dim3 grid(blocks_for((count + 3) / 4, lpr),
                    static_cast<unsigned>(std::min<int64_t>(16, (D + lpr * vec - 1) / (lpr * vec))));
#define FG_LOOKUP(VEC)                                                                                          \
  lookup_kernel<T, Id, VEC><<<grid, dim3(kBlockThreads), 0, stream>>>(t, i, o, count, static_cast<int32_t>(V),  \
                                                                      static_cast<int32_t>(D), lpr, scale)
    if constexpr (sizeof(T) == 2) {
      if (vec == 8) FG_LOOKUP(8);
    }
    if (vec == 4) FG_LOOKUP(4);
    if (vec == 2) FG_LOOKUP(2);
    if (vec == 1) FG_LOOKUP(1);
#undef FG_LOOKUP
  }
  FG_HIP_TRY(hipGetLastError());
  return FG_OK;
}

// Sizes shared by the entry points: rows and columns that int32 counts, ids that int32 places.
int check_sizes(int64_t V, int64_t D, int64_t n, int32_t dtype, int32_t itype) {
  if (V < 1 || V >= 0x7fffffffLL) return fail(FG_EINVAL, "n_rows = %lld is out of range", (long long)V);
  if (D < 1 || D > (1 << 20)) return fail(FG_EINVAL, "D = %lld is out of range", (long long)D);
  if (n < 0 || n > 0x7fff0000LL) return fail(FG_EINVAL, "n_ids = %lld is out of range", (long long)n);
  if (!element_type_ok(dtype)) return fail(FG_EINVAL, "dtype code %d is unknown", dtype);
  if (!index_type_ok(itype)) return fail(FG_EINVAL, "index type code %d is unknown", itype);
  return FG_OK;
}

}  // namespace
}  // namespace fg

extern "C" {

int fg_embedding_lookup(int64_t n_rows, int64_t D, int64_t n_ids, const void *table, const void *ids, void *out,
                        float scale, int32_t dtype, int32_t itype, void *stream) {
  if (int rc = fg::check_sizes(n_rows, D, n_ids, dtype, itype)) return rc;
  if (n_ids == 0) return FG_OK;
  if (!table || !ids || !out) return fg::fail(FG_EINVAL, "a data pointer is null");
  hipStream_t s = static_cast<hipStream_t>(stream);
#define FG_TYPED(T)                                                                                     \
  (itype == FG_I32 ? fg::lookup_typed<T, int32_t>(table, ids, out, n_ids, n_rows, D, scale, s)          \
                   : fg::lookup_typed<T, int64_t>(table, ids, out, n_ids, n_rows, D, scale, s))
  if (dtype == FG_F32) return FG_TYPED(float);
  if (dtype == FG_BF16) return FG_TYPED(__bf16);
  return FG_TYPED(_Float16);
#undef FG_TYPED
}

int fg_embedding_grad_workspace(int64_t n_rows, int64_t D, int64_t n_ids, int64_t *bytes) {
  if (int rc = fg::check_sizes(n_rows, D, n_ids, FG_F32, FG_I32)) return rc;
  if (!bytes) return fg::fail(FG_EINVAL, "bytes is null");
  *bytes = fg::grad_layout(n_ids, D).bytes;
  return FG_OK;
}

int fg_embedding_grad(int64_t n_rows, int64_t D, int64_t n_ids, const void *ids, const void *dout, void *grad,
                      float scale, int32_t accumulate, int32_t dtype, int32_t itype, void *workspace,
                      int64_t workspace_bytes, void *stream) {
  if (int rc = fg::check_sizes(n_rows, D, n_ids, dtype, itype)) return rc;
  if (n_ids == 0 && accumulate) return FG_OK;
  const fg::GradLayout g = fg::grad_layout(n_ids, D);
  if (!grad || (n_ids > 0 && (!ids || !dout))) return fg::fail(FG_EINVAL, "a data pointer is null");
  if (!workspace || !fg::aligned_to(workspace, 256) || workspace_bytes < g.bytes)
    return fg::fail(FG_EINVAL, "the workspace needs %lld bytes at a multiple of 256", (long long)g.bytes);
  hipStream_t s = static_cast<hipStream_t>(stream);
  char *ws = static_cast<char *>(workspace);
  const int2 *sorted = nullptr;
  if (n_ids > 0) {
    const int32_t n = static_cast<int32_t>(n_ids), V = static_cast<int32_t>(n_rows);
    const int rc = itype == FG_I32 ? fg::sort_ids(static_cast<const int32_t *>(ids), n, V, ws, g, &sorted, s)
                                   : fg::sort_ids(static_cast<const int64_t *>(ids), n, V, ws, g, &sorted, s);
    if (rc) return rc;
  }
#define FG_TYPED(T) fg::grad_typed<T>(sorted, n_ids, n_rows, D, dout, grad, scale, accumulate, ws, g, s)
  if (dtype == FG_F32) return FG_TYPED(float);
  if (dtype == FG_BF16) return FG_TYPED(__bf16);
  return FG_TYPED(_Float16);
#undef FG_TYPED
}

}  // extern "C"
