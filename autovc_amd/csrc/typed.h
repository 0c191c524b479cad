// Element types of the sequence-model operators (recurrence.hip, class_probs.hip, dropout.hip):
// fp32, bf16 or fp16 in memory, fp32 in registers.  Vectors are loaded and stored at the
// alignment of one element: the global memory instructions take any alignment, so a row may begin
// anywhere (odd widths, column slices of a wider buffer) without a variant of its own.
#pragma once

#include "common.h"

namespace avc {

template <typename E, int N>
struct Vec {
  E v[N];
};

// N consecutive elements at p (element-aligned), one memory instruction of N * sizeof(E) bytes
template <typename E, int N>
__device__ __forceinline__ Vec<E, N> vload(const E* p) {
  Vec<E, N> r;
  __builtin_memcpy(&r, p, sizeof(r));
  return r;
}
// rounded to the element type once, to nearest even
template <typename E, int N>
__device__ __forceinline__ void vstore(E* p, const float (&x)[N]) {
  Vec<E, N> r;
#pragma unroll
  for (int i = 0; i < N; ++i) r.v[i] = static_cast<E>(x[i]);
  __builtin_memcpy(p, &r, sizeof(r));
}

// calls f(E{}) with the element type of an AVC_DTYPE_* code, which the caller has checked
template <typename F>
inline int with_dtype(int dtype, F f) {
  switch (dtype) {
    case AVC_DTYPE_BF16: return f(__bf16{});
    case AVC_DTYPE_F16: return f(_Float16{});
    default: return f(float{});
  }
}
inline bool dtype_ok(int dtype) { return dtype >= AVC_DTYPE_F32 && dtype <= AVC_DTYPE_F16; }

}  // namespace avc
