// Codes of the 8-bit cache -> fp16, exactly: int8 and e4m3 both fit its 11 bits.
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

// bf16 rows become fp16 with a power of two taken out: e, the largest exponent field of the row -> the factor that brings its largest
// element into [2^13, 2^14), and its inverse.  What is lost lies 2^-31 below that element.  (Kept inside what a float's exponent holds.)
__device__ __forceinline__ void row_scale(uint32_t largest /* exponent bits of a bf16, in place */, float& up, float& down) {
  const int e = min(max((int)(largest >> 7), 14), 253);
  up = __int_as_float((267 - e) << 23);    // 2^(140 - e)
  down = __int_as_float((e - 13) << 23);
}
__device__ __forceinline__ uint32_t bf16_to_half2(uint32_t x, float up) {
  __half2 v = __floats2half2_rn(__uint_as_float(x << 16) * up, __uint_as_float(x & 0xFFFF0000u) * up);
  return *reinterpret_cast<uint32_t*>(&v);
}

}  // namespace tfa_b200
