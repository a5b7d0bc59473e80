// Global norm of many gradients, and their clipping by it:
//
//   norm = sqrt(sum over tensors t, elements i of g_t[i]^2)      c = min(1, max_norm / (norm + eps))
//   out_t[i] = c * g_t[i]
//
// All tensors of a call are one list of 8 KB pieces.  A workgroup takes a contiguous range of the list, so that it
// looks its first tensor up once and then moves on; it adds squares in float64 (no overflow for any float32, and the
// device's double rate is far above what memory delivers) and leaves one partial sum.  The scaling kernel's
// workgroups each add the partial sums again, in the same order, which costs less than a launch between the two.
// The scaling goes through each workgroup's range from its end: what the first pass read last is still in the last-level
// cache.  Small lists (the layers of a small model) run in one workgroup and one launch.  The tensors' addresses travel in
// the kernel arguments, so a call can be captured into a graph and needs no copy to the device.
#include <algorithm>
#include <initializer_list>

#include "element.hpp"

namespace fg {
namespace {

constexpr int kTensors = 96;          // per launch: 29 bytes each, within the 4 KB of kernel arguments
constexpr int kPieceBytes = 8192;
constexpr int kMostBlocks = 2048;     // partial sums over all launches of a call
constexpr int kSmallPieces = 16;      // pieces up to which one workgroup does everything, a wave each
constexpr int kSmallThreads = 1024;

struct TensorList {
  const void *in[kTensors];
  void *out[kTensors];
  int64_t n[kTensors];
  int32_t first[kTensors + 1];  // first piece of each tensor
  uint8_t type[kTensors];       // element type, + 4 when not 16-byte aligned
  int32_t count;
};

int64_t pieces_of(int64_t n, int dtype) { return (n * element_bytes(dtype) + kPieceBytes - 1) / kPieceBytes; }

template <int THREADS>
__device__ __forceinline__ double block_sum(double x, double *lds) {
  constexpr int kWaves = THREADS / kWaveSize;
  for (int d = 1; d < kWaveSize; d <<= 1) x += __shfl_xor(x, d, kWaveSize);
  if ((threadIdx.x & (kWaveSize - 1)) == 0) lds[threadIdx.x / kWaveSize] = x;
  __syncthreads();
  double s = 0.0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) s += lds[w];
  __syncthreads();
  return s;
}

template <typename T, int N>
__device__ __forceinline__ double square_sum(const Pack<T, N> &p) {
  double s = 0.0;
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const double d = static_cast<double>(widen(p.v[k]));
    s = __builtin_fma(d, d, s);
  }
  return s;
}

// Sum of squares of elements [lo, hi) of one tensor, this thread's share.
template <typename T, int THREADS>
__device__ __forceinline__ double squares(const void *in, int64_t lo, int64_t hi, bool aligned) {
  constexpr int kVec = 16 / sizeof(T);
  using P = Pack<T, kVec>;
  const T *x = static_cast<const T *>(in);
  double s = 0.0;
  int64_t i = lo;
  if (aligned) {
    const int64_t whole = lo + (hi - lo) / kVec * kVec;
    constexpr int kUnroll = 4;
    int64_t j = lo + threadIdx.x * kVec;
    for (; j + THREADS * kVec * (kUnroll - 1) < whole; j += THREADS * kVec * kUnroll) {
      P p[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) p[u] = *reinterpret_cast<const P *>(x + j + THREADS * kVec * u);
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) s += square_sum(p[u]);
    }
    for (; j < whole; j += THREADS * kVec) s += square_sum(*reinterpret_cast<const P *>(x + j));
    i = whole;
  }
  for (int64_t j = i + threadIdx.x; j < hi; j += THREADS) {
    const double d = static_cast<double>(widen(x[j]));
    s = __builtin_fma(d, d, s);
  }
  return s;
}

// A store that leaves the last-level cache to the gradients that are still to be read (3% of the two passes together).
template <typename T, typename P>
__device__ __forceinline__ void store_past(T *to, const P &p) {
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  __builtin_nontemporal_store(__builtin_bit_cast(u32x4, p), reinterpret_cast<u32x4 *>(to));
}

template <typename T, int THREADS>
__device__ __forceinline__ void scale_out(const void *in, void *out, int64_t lo, int64_t hi, bool aligned, float c) {
  constexpr int kVec = 16 / sizeof(T), kUnroll = 4;
  using P = Pack<T, kVec>;
  const T *x = static_cast<const T *>(in);
  T *y = static_cast<T *>(out);
  if (aligned) {
    const int64_t whole = lo + (hi - lo) / kVec * kVec;
    for (int64_t j = whole + threadIdx.x; j < hi; j += THREADS) y[j] = narrow<T>(widen(x[j]) * c);
    int64_t end = whole;
    for (; end - lo >= THREADS * kVec * kUnroll; end -= THREADS * kVec * kUnroll) {
      P p[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
        p[u] = *reinterpret_cast<const P *>(x + end - (THREADS * (u + 1) - threadIdx.x) * kVec);
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
#pragma unroll
        for (int k = 0; k < kVec; ++k) p[u].v[k] = narrow<T>(widen(p[u].v[k]) * c);
        store_past(y + end - (THREADS * (u + 1) - threadIdx.x) * kVec, p[u]);
      }
    }
    for (int64_t j = lo + threadIdx.x * kVec; j < end; j += THREADS * kVec) {
      P p = *reinterpret_cast<const P *>(x + j);
#pragma unroll
      for (int k = 0; k < kVec; ++k) p.v[k] = narrow<T>(widen(p.v[k]) * c);
      *reinterpret_cast<P *>(y + j) = p;
    }
    return;
  }
  for (int64_t j = lo + threadIdx.x; j < hi; j += THREADS) y[j] = narrow<T>(widen(x[j]) * c);
}

// Calls f(tensor, first element, one past the last) for this workgroup's share of the list, tensor by tensor, from the
// last tensor to the first with kBack.
template <bool kBack, typename F>
__device__ __forceinline__ void for_share(const TensorList &l, F &&f) {
  const int32_t total = l.first[l.count];
  const int32_t lo = static_cast<int32_t>(static_cast<int64_t>(total) * blockIdx.x / gridDim.x);
  const int32_t hi = static_cast<int32_t>(static_cast<int64_t>(total) * (blockIdx.x + 1) / gridDim.x);
  if (lo >= hi) return;
  int a = 0, b = l.count - 1;  // last tensor that starts at or before `lo`
  while (a < b) {
    const int m = (a + b + 1) / 2;
    if (l.first[m] <= lo) a = m; else b = m - 1;
  }
  int z = a;  // one past the last tensor that starts below `hi`
  while (z < l.count && l.first[z] < hi) ++z;
  for (int k = a; k < z; ++k) {
    const int t = kBack ? z - 1 - (k - a) : k;
    const int32_t p0 = max(lo, l.first[t]), p1 = min(hi, l.first[t + 1]);
    if (p0 >= p1) continue;
    const int64_t per = kPieceBytes / ((l.type[t] & 3) == FG_F32 ? 4 : 2);
    f(t, (p0 - l.first[t]) * per, min((p1 - l.first[t]) * per, l.n[t]));
  }
}

template <int THREADS>
__device__ __forceinline__ double share_squares(const TensorList &l) {
  double s = 0.0;
  for_share<false>(l, [&](int t, int64_t lo, int64_t hi) {
    const int type = l.type[t] & 3;
    const bool aligned = l.type[t] < 4;
    if (type == FG_F32) s += squares<float, THREADS>(l.in[t], lo, hi, aligned);
    else if (type == FG_BF16) s += squares<__bf16, THREADS>(l.in[t], lo, hi, aligned);
    else s += squares<_Float16, THREADS>(l.in[t], lo, hi, aligned);
  });
  return s;
}

template <int THREADS>
__device__ __forceinline__ void share_scale(const TensorList &l, float c) {
  for_share<true>(l, [&](int t, int64_t lo, int64_t hi) {
    const int type = l.type[t] & 3;
    const bool aligned = l.type[t] < 4;
    if (l.out[t] == l.in[t] && c == 1.0f) return;  // in place and nothing to clip
    if (type == FG_F32) scale_out<float, THREADS>(l.in[t], l.out[t], lo, hi, aligned, c);
    else if (type == FG_BF16) scale_out<__bf16, THREADS>(l.in[t], l.out[t], lo, hi, aligned, c);
    else scale_out<_Float16, THREADS>(l.in[t], l.out[t], lo, hi, aligned, c);
  });
}

// The coefficient in double: a norm beyond float32 still clips to max_norm.  A norm that is NaN or infinite gives
// NaN and 0, as the formula says (fmin would drop the NaN).
__device__ __forceinline__ float coefficient(double norm, float max_norm, float eps) {
  const double c = static_cast<double>(max_norm) / (norm + static_cast<double>(eps));
  return c < 1.0 || c != c ? static_cast<float>(c) : 1.0f;
}

// One wave per piece.  The piece stays in registers between the two passes (eight loads of 16 bytes per lane, all under way
// at once); only a tensor off its alignment is read again.
__global__ __launch_bounds__(kSmallThreads) void small_kernel(TensorList l, int clip, float max_norm, float eps,
                                                              float *norm_out) {
  constexpr int kHeld = kPieceBytes / (kWaveSize * 16);
  static_assert(kSmallPieces == kSmallThreads / kWaveSize, "a wave per piece");
  __shared__ double lds[kSmallThreads / kWaveSize];
  const int lane = threadIdx.x & (kWaveSize - 1), piece = threadIdx.x / kWaveSize;
  const bool busy = piece < l.first[l.count];
  int t = 0;  // tensors that end at or before this piece: counted by the lanes together
  for (int k = 0; k < l.count; k += kWaveSize)
    t += __popcll(__ballot(k + lane < l.count && l.first[k + lane + 1] <= piece));
  t = busy ? t : 0;
  const int type = busy ? l.type[t] & 3 : 0, bytes = type == FG_F32 ? 4 : 2;
  const bool aligned = busy && l.type[t] < 4;
  const int64_t per = kPieceBytes / bytes, lo = busy ? (piece - l.first[t]) * per : 0;
  const int count = busy ? static_cast<int>(min(per, l.n[t] - lo)) : 0;  // elements of this piece
  const int vectors = aligned ? count * bytes / 16 : 0;                  // whole 16-byte vectors of it
  const int loose = vectors * 16 / bytes;                                // first element behind them
  const char *in = busy ? static_cast<const char *>(l.in[t]) + lo * bytes : nullptr;
  char *out = busy && clip ? static_cast<char *>(l.out[t]) + lo * bytes : nullptr;
  uint4 held[kHeld];
#pragma unroll
  for (int u = 0; u < kHeld; ++u)
    held[u] = u * kWaveSize + lane < vectors ? reinterpret_cast<const uint4 *>(in)[u * kWaveSize + lane] : uint4{0, 0, 0, 0};
  auto typed = [&](auto &&f) {  // f(a value of the tensor's type)
    if (type == FG_F32) f(0.0f);
    else if (type == FG_BF16) f(__bf16{});
    else f(_Float16{});
  };
  double s = 0.0;
  typed([&](auto kind) {
    using T = decltype(kind);
#pragma unroll
    for (int u = 0; u < kHeld; ++u) s += square_sum(__builtin_bit_cast(Pack<T, 16 / sizeof(T)>, held[u]));
    for (int j = loose + lane; j < count; j += kWaveSize) {
      const double d = static_cast<double>(widen(reinterpret_cast<const T *>(in)[j]));
      s = __builtin_fma(d, d, s);
    }
  });
  const double norm = sqrt(block_sum<kSmallThreads>(s, lds));
  if (threadIdx.x == 0) *norm_out = static_cast<float>(norm);
  if (!clip || !busy) return;
  const float c = coefficient(norm, max_norm, eps);
  if (in == out && c == 1.0f) return;  // in place and nothing to clip
  typed([&](auto kind) {
    using T = decltype(kind);
    constexpr int kVec = 16 / sizeof(T);
#pragma unroll
    for (int u = 0; u < kHeld; ++u) {
      auto p = __builtin_bit_cast(Pack<T, kVec>, held[u]);
#pragma unroll
      for (int k = 0; k < kVec; ++k) p.v[k] = narrow<T>(widen(p.v[k]) * c);
      if (u * kWaveSize + lane < vectors) reinterpret_cast<Pack<T, kVec> *>(out)[u * kWaveSize + lane] = p;
    }
    for (int j = loose + lane; j < count; j += kWaveSize)
      reinterpret_cast<T *>(out)[j] = narrow<T>(widen(reinterpret_cast<const T *>(in)[j]) * c);
  });
}

__global__ __launch_bounds__(kBlockThreads) void squares_kernel(TensorList l, double *partial) {
  __shared__ double lds[kWavesPerBlock];
  const double s = block_sum<kBlockThreads>(share_squares<kBlockThreads>(l), lds);
  if (threadIdx.x == 0) partial[blockIdx.x] = s;
}

__device__ __forceinline__ double norm_of(const double *partial, int partials, double *lds) {
  double s = 0.0;
  for (int i = threadIdx.x; i < partials; i += kBlockThreads) s += partial[i];
  return sqrt(block_sum<kBlockThreads>(s, lds));
}

__global__ __launch_bounds__(kBlockThreads) void norm_kernel(const double *partial, int partials, float *norm_out) {
  __shared__ double lds[kWavesPerBlock];
  const double norm = norm_of(partial, partials, lds);
  if (threadIdx.x == 0) *norm_out = static_cast<float>(norm);
}

__global__ __launch_bounds__(kBlockThreads) void scale_kernel(TensorList l, const double *partial, int partials,
                                                              float max_norm, float eps, float *norm_out) {
  __shared__ double lds[kWavesPerBlock];
  const double norm = norm_of(partial, partials, lds);
  if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = static_cast<float>(norm);
  share_scale<kBlockThreads>(l, coefficient(norm, max_norm, eps));
}

// Fills `l` with up to kTensors tensors from `from` on that have elements; returns where the next launch goes on.
int fill(const fg_tensor *t, int32_t count, int32_t from, TensorList *l) {
  l->count = 0;
  int64_t piece = 0;
  int32_t i = from;
  for (; i < count && l->count < kTensors; ++i) {
    if (t[i].n == 0) continue;
    const int64_t more = pieces_of(t[i].n, t[i].dtype);
    if (piece + more > 0x7fffffffLL) break;
    const int k = l->count++;
    l->in[k] = t[i].in;
    l->out[k] = t[i].out;
    l->n[k] = t[i].n;
    l->first[k] = static_cast<int32_t>(piece);
    l->type[k] = static_cast<uint8_t>(
        t[i].dtype + (aligned_to(t[i].in, 16) && (!t[i].out || aligned_to(t[i].out, 16)) ? 0 : 4));
    piece += more;
  }
  l->first[l->count] = static_cast<int32_t>(piece);
  return i;
}

int run(const fg_tensor *t, int32_t count, int clip, float max_norm, float eps, float *norm_out, double *partial,
        hipStream_t stream) {
  int launches = 0;
  TensorList l;
  int32_t at = 0;
  do {
    at = fill(t, count, at, &l);
    if (launches == 0 && at == count && l.first[l.count] <= kSmallPieces) {  // an empty list too: norm 0
      small_kernel<<<dim3(1), dim3(kSmallThreads), 0, stream>>>(l, clip, max_norm, eps, norm_out);
      FG_HIP_TRY(hipGetLastError());
      return FG_OK;
    }
    ++launches;
  } while (at < count);
  // every launch has as many workgroups as the partial sums' room allows
  const int most = std::max(1, kMostBlocks / std::max(1, launches));
  int partials = 0;
  for (int32_t i = 0; i < count;) {
    i = fill(t, count, i, &l);
    if (l.count == 0) break;
    const int blocks = std::min(most, l.first[l.count]);
    squares_kernel<<<dim3(blocks), dim3(kBlockThreads), 0, stream>>>(l, partial + partials);
    partials += blocks;
  }
  if (!clip) {
    norm_kernel<<<dim3(1), dim3(kBlockThreads), 0, stream>>>(partial, partials, norm_out);
  } else {
    float *norm_to = norm_out;
    for (int32_t i = 0; i < count;) {
      i = fill(t, count, i, &l);
      if (l.count == 0) break;
      scale_kernel<<<dim3(std::min(kMostBlocks, l.first[l.count])), dim3(kBlockThreads), 0, stream>>>(
          l, partial, partials, max_norm, eps, norm_to);
      norm_to = nullptr;
    }
  }
  FG_HIP_TRY(hipGetLastError());
  return FG_OK;
}

constexpr int32_t kMostTensors = kTensors * kMostBlocks;  // one partial sum per launch is the least

int check(int32_t count, const fg_tensor *t, bool clip, const float *norm, const void *workspace,
          int64_t workspace_bytes) {
  if (count < 0 || count > kMostTensors) return fail(FG_EINVAL, "count = %d is out of range", count);
  if (!norm) return fail(FG_EINVAL, "norm is null");
  if (count > 0 && !t) return fail(FG_EINVAL, "tensors is null");
  for (int32_t i = 0; i < count; ++i) {
    if (t[i].n < 0 || t[i].n > (int64_t{1} << 40)) return fail(FG_EINVAL, "tensor %d has %lld elements", i, (long long)t[i].n);
    if (!element_type_ok(t[i].dtype)) return fail(FG_EINVAL, "tensor %d has the unknown dtype code %d", i, t[i].dtype);
    if (t[i].n > 0 && (!t[i].in || (clip && !t[i].out))) return fail(FG_EINVAL, "tensor %d has a null pointer", i);
  }
  if (!workspace || !aligned_to(workspace, 256) || workspace_bytes < int64_t{kMostBlocks} * 8)
    return fail(FG_EINVAL, "the workspace needs %d bytes at a multiple of 256", kMostBlocks * 8);
  return FG_OK;
}

}  // namespace
}  // namespace fg

extern "C" {

int fg_grad_norm_workspace(int64_t *bytes) {
  if (!bytes) return fg::fail(FG_EINVAL, "bytes is null");
  *bytes = int64_t{fg::kMostBlocks} * 8;
  return FG_OK;
}

int fg_grad_norm(int32_t count, const fg_tensor *tensors, float *norm, void *workspace, int64_t workspace_bytes,
                 void *stream) {
  if (int rc = fg::check(count, tensors, false, norm, workspace, workspace_bytes)) return rc;
  return fg::run(tensors, count, 0, 1.0f, 0.0f, norm, static_cast<double *>(workspace), static_cast<hipStream_t>(stream));
}

int fg_grad_clip(int32_t count, const fg_tensor *tensors, float max_norm, float eps, float *norm, void *workspace,
                 int64_t workspace_bytes, void *stream) {
  if (int rc = fg::check(count, tensors, true, norm, workspace, workspace_bytes)) return rc;
  if (!(max_norm >= 0.0f) || !(eps >= 0.0f)) return fg::fail(FG_EINVAL, "max_norm and eps must not be negative");
  return fg::run(tensors, count, 1, max_norm, eps, norm, static_cast<double *>(workspace), static_cast<hipStream_t>(stream));
}

}  // extern "C"
