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
// The same past the caches, for an output that will not be in them when it is read next (streams() on the host)
template <class T, int V>
__device__ __forceinline__ void store_past(T *p, const Vec<T, V> &v) {
  if constexpr (sizeof(T) * V >= 4) {
    typedef unsigned U __attribute__((ext_vector_type(sizeof(T) * V / 4)));
    __builtin_nontemporal_store(__builtin_bit_cast(U, v), reinterpret_cast<U *>(p));
  } else {
    store<T, V>(p, v);
  }
}
// Whether an output of so many bytes is written past the caches: from half of the 256 MB that lie before the memory on.  Smaller ones find their reader's data
// evicted for nothing (a training step at 640x512 with every output written past them: 10.73 -> 10.85 ms).
inline bool streams(size_t bytes) { return bytes >= ((size_t)128 << 20); }

// V consecutive floats on any 4-byte boundary, still as one access
template <int V>
struct __attribute__((packed, aligned(4))) Floats {
  float v[V];
};

// a / b and a % b; in 32 bits where both fit (a 64-bit division is some 100 instructions)
__device__ __forceinline__ void divide(size_t a, size_t b, size_t &quotient, size_t &rest) {
  if (((a | b) >> 32) == 0) {
    quotient = (unsigned)a / (unsigned)b;
    rest = (unsigned)a - (unsigned)quotient * (unsigned)b;
  } else {
    quotient = a / b;
    rest = a - quotient * b;
  }
}

// The value of lane (own ^ d), d = 1, 2, 4 .. 32: inside a row of 16 lanes by data-parallel moves (quad permutes; 4 and 8 after the smaller steps of a sum, where
// the mirror of 8 / 16 lanes holds the same value), beyond by the LDS crossbar.  For sums over lanes in the order 1, 2, 4, ..; all lanes active.
__device__ __forceinline__ double lane_xor(double v, int d) {
  const unsigned long long u = __builtin_bit_cast(unsigned long long, v);
  int lo = (int)(unsigned)u, hi = (int)(unsigned)(u >> 32);
  switch (d) {
    case 1: lo = __builtin_amdgcn_update_dpp(0, lo, 0xB1, 0xF, 0xF, false); hi = __builtin_amdgcn_update_dpp(0, hi, 0xB1, 0xF, 0xF, false); break;
    case 2: lo = __builtin_amdgcn_update_dpp(0, lo, 0x4E, 0xF, 0xF, false); hi = __builtin_amdgcn_update_dpp(0, hi, 0x4E, 0xF, 0xF, false); break;
    case 4: lo = __builtin_amdgcn_update_dpp(0, lo, 0x141, 0xF, 0xF, false); hi = __builtin_amdgcn_update_dpp(0, hi, 0x141, 0xF, 0xF, false); break;
    case 8: lo = __builtin_amdgcn_update_dpp(0, lo, 0x140, 0xF, 0xF, false); hi = __builtin_amdgcn_update_dpp(0, hi, 0x140, 0xF, 0xF, false); break;
    default: {
      const int from = (int)((threadIdx.x & 63) ^ d) * 4;
      lo = __builtin_amdgcn_ds_bpermute(from, lo);
      hi = __builtin_amdgcn_ds_bpermute(from, hi);
    }
  }
  return __builtin_bit_cast(double, (unsigned long long)(unsigned)hi << 32 | (unsigned)lo);
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
