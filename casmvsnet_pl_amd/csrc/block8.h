// The 8-bit checkpoint format, one block = 32 consecutive values of a plane = eight lanes with four values each.
//
//   e = max(floor(log2 max |v|), -127),  step = 2^(e - 6),  code = sign bit | min(127, rint(|v| / step)),  scale byte = e + 127
//   a block that holds an Inf or a NaN: scale byte 255, and it reads back as NaN.
//
// A power-of-two step makes every operation but the one rounding exact: what a block holds does not depend on who computed it, and code * step is exact in
// float32 (and in float64 for the statistics).  The price against max / 127 as the step is up to one bit: an error of at most 2^-7 of the block's largest
// power of two.  Rounding: half to even; values between 127.5 and 128 steps saturate.
#pragma once
#include "elem_types.h"

namespace casmvs {
namespace block8 {

constexpr int kBlock = 32;
constexpr int kLanes = 8;   // lanes per block

// exchanges inside groups of eight lanes: xor 1, xor 2 (quad permutes), then the mirror of eight.  All eight lanes have to be active.
template <class F>
__device__ __forceinline__ unsigned over_block(unsigned v, F f) {
  v = f(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, false));
  v = f(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, false));
  return f(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xF, 0xF, false));
}

__device__ __forceinline__ unsigned high_word(double v) { return (unsigned)(__builtin_bit_cast(unsigned long long, v) >> 32); }
// 2^e for -1022 <= e <= 1023
__device__ __forceinline__ double power_of_two(int e) { return __builtin_bit_cast(double, (unsigned long long)(unsigned)(e + 1023) << 52); }

// Four values of a lane -> its four code bytes; `scale`: the block's scale byte (the same in its eight lanes).
__device__ __forceinline__ unsigned quantise(const double (&v)[4], unsigned &scale) {
  unsigned top = 0;   // the largest magnitude's high word: its exponent is the block's, and Inf / NaN have the largest exponent field there is
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const unsigned h = high_word(v[i]) & 0x7FFFFFFFu;
    top = h > top ? h : top;
  }
  top = over_block(top, [](unsigned a, unsigned b) { return a > b ? a : b; });
  int e = (int)(top >> 20) - 1023;
  e = e < -127 ? -127 : e;
  const bool finite = e <= 127;   // (a float32 is below 2^128)
  scale = finite ? (unsigned)(e + 127) : 255u;
  const double per_step = power_of_two(finite ? 6 - e : 0);
  unsigned codes = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    // |v| / step < 128: adding 1.5 * 2^52 rounds it to an integer, half to even, in the low bits of the sum
    const double t = __builtin_fabs(v[i]) * per_step + 6755399441055744.0;
    unsigned q = (unsigned)__builtin_bit_cast(unsigned long long, t);
    q = q > 127u ? 127u : q;
    q = finite ? q : 0u;
    codes |= (q | (high_word(v[i]) >> 31 << 7)) << (8 * i);
  }
  return codes;
}

// The value of code byte `i` of `codes`.  step of the block: step_of(scale byte); 0 * NaN = NaN for a block that is not finite.
__device__ __forceinline__ float step_of(unsigned scale) {
  return scale == 255u ? __builtin_nanf("") : __builtin_ldexpf(1.0f, (int)scale - 133);
}
__device__ __forceinline__ float value_of(unsigned codes, int i, float step) {
  const unsigned byte = codes >> (8 * i);
  const float m = (float)(byte & 127u) * step;   // exact, subnormal steps included
  return (byte & 128u) ? -m : m;
}

}  // namespace block8
}  // namespace casmvs
