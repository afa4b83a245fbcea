// Codes of the 8-bit cache -> fp16, exactly: int8 and e4m3 both fit its 11 bits.
//
// e4m3 is converted.  Widening it with shifts and masks instead (sign, exponent and mantissa moved to where fp16 has them are the code times
// 2^-8) was slower in both attention kernels, where it lengthens the chain of the warps that convert: decode of 64 requests of 4000 tokens
// 103 -> 119 us, chunks of queries 350 -> 366.
#pragma once

#include <cuda_fp16.h>
#include <stdint.h>

namespace tfa_b200 {

// Four codes of a word -> two pairs of halves.  int8: 0x6400 | (code ^ 0x80) is 1024 + 128 + code.
template <bool kInt8>
__device__ __forceinline__ void widen(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (kInt8) {
    w ^= 0x80808080u;
    const uint32_t a = __byte_perm(w, 0x64646464u, 0x4140), b = __byte_perm(w, 0x64646464u, 0x4342);
    const __half2 off = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));
    const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&a), off), y = __hsub2(*reinterpret_cast<const __half2*>(&b), off);
    lo = *reinterpret_cast<const uint32_t*>(&x);
    hi = *reinterpret_cast<const uint32_t*>(&y);
  } else {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}" : "=r"(lo), "=r"(hi) : "r"(w));
  }
}
// Sums over V refer to a scale of V that is no smaller than this: 2^4 times its reciprocal is a float, and 2^-4 of it almost a normal one (scales go
// down to 2^-126).
constexpr float kSmallestVRef = 1e-37f;

// Rows of queries become fp16 with a power of two taken out, which brings the row's largest element into [2^13, 2^14): what is lost lies
// 2^-31 below that element.  `largest`: exponent bits of the largest element, in place; the factors stay
// inside what a float's exponent holds.
template <bool kBf16>
__device__ __forceinline__ void row_scale(uint32_t largest, float& up, float& down) {
  const int e = kBf16 ? min(max((int)(largest >> 7), 14), 253) : min(max((int)(largest >> 10), 1), 30) + 112;  // exponent field of a float
  up = __int_as_float((267 - e) << 23);  // 2^(140 - e)
  down = __int_as_float((e - 13) << 23);
}
template <bool kBf16>
constexpr uint32_t exponent_bits() {
  return kBf16 ? 0x7F80u : 0x7C00u;
}
template <bool kBf16>
__device__ __forceinline__ uint32_t scale_to_half2(uint32_t x, float up) {
  float2 f;
  if constexpr (kBf16) {
    f = make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xFFFF0000u));
  } else {
    f = __half22float2(*reinterpret_cast<const __half2*>(&x));
  }
  const __half2 v = __floats2half2_rn(f.x * up, f.y * up);
  return *reinterpret_cast<const uint32_t*>(&v);
}

}  // namespace tfa_b200
