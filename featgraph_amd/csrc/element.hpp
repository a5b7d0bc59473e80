// Element types of the training operators: float32, bfloat16 and float16 in memory, float32 in registers.
#pragma once

#include "common.hpp"

namespace fg {

template <typename T>
__device__ __forceinline__ float widen(T x) {
  return static_cast<float>(x);
}
// one rounding to nearest even (v_cvt_pk_bf16_f32 / v_cvt_f16_f32); float32 stays as it is
template <typename T>
__device__ __forceinline__ T narrow(float x) {
  return static_cast<T>(x);
}

// N consecutive elements that one lane loads or stores at once
template <typename T, int N>
struct alignas(sizeof(T) * N) Pack {
  T v[N];
};

inline int element_bytes(int dtype) { return dtype == FG_F32 ? 4 : 2; }
inline bool element_type_ok(int dtype) { return dtype == FG_F32 || dtype == FG_BF16 || dtype == FG_F16; }
inline bool index_type_ok(int itype) { return itype == FG_I32 || itype == FG_I64; }

// Elements per 16-byte (or narrower) access that divides rows of D elements and fits the alignment of every
// pointer in `ptrs`: the largest power of two up to 16 bytes.
inline int vector_elements(int64_t D, int bytes, std::initializer_list<const void *> ptrs) {
  int v = 16 / bytes;
  while (v > 1) {
    bool ok = D % v == 0;
    for (const void *p : ptrs) ok = ok && aligned_to(p, static_cast<uintptr_t>(v) * bytes);
    if (ok) break;
    v >>= 1;
  }
  return v;
}

}  // namespace fg
