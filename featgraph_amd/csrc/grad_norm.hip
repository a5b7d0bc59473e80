// Global norm of many gradients, and their clipping by it:
//
//   norm = sqrt(sum over tensors t, elements i of g_t[i]^2)      c = min(1, max_norm / (norm + eps))
//   out_t[i] = c * g_t[i]
//
// All tensors of a call are one list of 16 KB pieces.  A workgroup takes a contiguous range of the list, so that it
// looks its first tensor up once and then moves on; it adds squares in float64 (no overflow for any float32, and the
// device's double rate is far above what memory delivers) and leaves one partial sum.  The scaling kernel's
// workgroups each add the partial sums again, in the same order, which costs less than a launch between the two.
// Small lists (the layers of a small model) run in one workgroup and one launch.  The tensors' addresses travel in
// the kernel arguments, so a call can be captured into a graph and needs no copy to the device.
#include <algorithm>
#include <initializer_list>

#include "element.hpp"

namespace fg {
namespace {

constexpr int kTensors = 96;          // per launch: 29 bytes each, within the 4 KB of kernel arguments
constexpr int kPieceBytes = 16384;
constexpr int kMostBlocks = 2048;     // partial sums over all launches of a call
constexpr int kSmallPieces = 16;      // pieces up to which one workgroup does everything
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
    for (int64_t j = lo + threadIdx.x * kVec; j < whole; j += THREADS * kVec) {
      const P p = *reinterpret_cast<const P *>(x + j);
#pragma unroll
      for (int k = 0; k < kVec; ++k) {
        const double d = static_cast<double>(widen(p.v[k]));
        s = __builtin_fma(d, d, s);
      }
    }
    i = whole;
  }
  for (int64_t j = i + threadIdx.x; j < hi; j += THREADS) {
    const double d = static_cast<double>(widen(x[j]));
    s = __builtin_fma(d, d, s);
  }
  return s;
}

template <typename T, int THREADS>
__device__ __forceinline__ void scale_out(const void *in, void *out, int64_t lo, int64_t hi, bool aligned, float c) {
  constexpr int kVec = 16 / sizeof(T);
  using P = Pack<T, kVec>;
  const T *x = static_cast<const T *>(in);
  T *y = static_cast<T *>(out);
  int64_t i = lo;
  if (aligned) {
    const int64_t whole = lo + (hi - lo) / kVec * kVec;
    for (int64_t j = lo + threadIdx.x * kVec; j < whole; j += THREADS * kVec) {
      P p = *reinterpret_cast<const P *>(x + j);
#pragma unroll
      for (int k = 0; k < kVec; ++k) p.v[k] = narrow<T>(widen(p.v[k]) * c);
      *reinterpret_cast<P *>(y + j) = p;
    }
    i = whole;
  }
  for (int64_t j = i + threadIdx.x; j < hi; j += THREADS) y[j] = narrow<T>(widen(x[j]) * c);
}

// Calls f(tensor, first element, one past the last) for this workgroup's share of the list, tensor by tensor.
template <typename F>
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
  for (int t = a; t < l.count && l.first[t] < hi; ++t) {
    const int32_t p0 = max(lo, l.first[t]), p1 = min(hi, l.first[t + 1]);
    if (p0 >= p1) continue;
    const int64_t per = kPieceBytes / ((l.type[t] & 3) == FG_F32 ? 4 : 2);
    f(t, (p0 - l.first[t]) * per, min((p1 - l.first[t]) * per, l.n[t]));
  }
}

template <int THREADS>
__device__ __forceinline__ double share_squares(const TensorList &l) {
  double s = 0.0;
  for_share(l, [&](int t, int64_t lo, int64_t hi) {
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
  for_share(l, [&](int t, int64_t lo, int64_t hi) {
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

__global__ __launch_bounds__(kSmallThreads) void small_kernel(TensorList l, int clip, float max_norm, float eps,
                                                              float *norm_out) {
  __shared__ double lds[kSmallThreads / kWaveSize];
  const double norm = sqrt(block_sum<kSmallThreads>(share_squares<kSmallThreads>(l), lds));
  if (threadIdx.x == 0) *norm_out = static_cast<float>(norm);
  if (clip) share_scale<kSmallThreads>(l, coefficient(norm, max_norm, eps));
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
