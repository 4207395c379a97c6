// The element types the training-side operators take (float32, float16, bfloat16) and their vector accesses; sums and statistics are never held in them.
#pragma once
#include "common.h"

namespace casmvs {
namespace elem {

typedef _Float16 f16;
typedef __bf16 bf16;

inline size_t size_of(int dtype) { return dtype == CASMVS_DTYPE_F32 ? 4 : 2; }
inline bool known(int dtype) { return dtype == CASMVS_DTYPE_F32 || dtype == CASMVS_DTYPE_F16 || dtype == CASMVS_DTYPE_BF16; }

// V consecutive elements as one access of V * sizeof(T) bytes (the caller checks the alignment on the host)
template <class T, int V>
struct alignas(sizeof(T) * V) Vec {
  T v[V];
};
template <class T, int V>
__device__ __forceinline__ Vec<T, V> load(const T *p) {
  return *reinterpret_cast<const Vec<T, V> *>(p);
}
template <class T, int V>
__device__ __forceinline__ void store(T *p, const Vec<T, V> &v) {
  *reinterpret_cast<Vec<T, V> *>(p) = v;
}

}  // namespace elem
}  // namespace casmvs

// Runs `...` with `T` bound to the element type of `dtype` (checked before).
#define CASMVS_WITH_DTYPE(dtype, ...)                                                        \
  do {                                                                                       \
    if ((dtype) == CASMVS_DTYPE_F32) { using T = float; __VA_ARGS__; }                       \
    else if ((dtype) == CASMVS_DTYPE_F16) { using T = casmvs::elem::f16; __VA_ARGS__; }      \
    else { using T = casmvs::elem::bf16; __VA_ARGS__; }                                      \
  } while (0)
