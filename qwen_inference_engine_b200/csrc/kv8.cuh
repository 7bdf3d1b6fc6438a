// kv8.cuh -- a cache in 8 bits: of each token and kv head a vector of codes (e4m3 or int8) and a power of two, for keys and for values.
//
// The scale is the smallest power of two with which the vector's largest element is no more than the largest code (448, 127).  As one token of a head has its own, nothing that a
// later token brings revises it.  As it is a power of two, a code times its scale is a bf16 number (of 4 or 7 bits), products of codes with queries are exact in fp32, and e4m3, which
// has an exponent of its own, loses nothing by it; int8 loses up to one of its bits.
#pragma once
#include <cuda_fp16.h>

#include "common.cuh"
#include "kernels.h"

namespace qie {

// the scale's byte for a largest element of `amax` (fp32 bits of a number that is not below 0): 2^(byte - 127); 0 for a vector of zeros, 255 for one that has an infinity or no number
template <int CODE>
__device__ __forceinline__ uint32_t kv8_scale_byte(uint32_t amax) {
  if (amax == 0) return 0;
  if (amax >= 0x7f800000u) return 255;
  // 448 = 1.75 * 2^8, 127 = 1.984375 * 2^6: the exponent is one more where the mantissa is above those
  const int b = CODE == KV8_E4M3 ? (int)((amax + 0x1fffffu) >> 23) - 8 : (int)((amax + 0x01ffffu) >> 23) - 6;
  return (uint32_t)max(b, 1);
}
// what a vector with this byte is multiplied with to give codes; bytes of 0 and 255 have codes of 0
__device__ __forceinline__ float kv8_inverse(uint32_t byte) { return byte == 0 || byte == 255 ? 0.f : __uint_as_float((254u - byte) << 23); }
// and its codes, to give values (255: no numbers)
__device__ __forceinline__ float kv8_scale(uint32_t byte) { return __uint_as_float(byte == 255 ? 0x7fc00000u : byte << 23); }

// four numbers within the codes' range, rounded to nearest even
template <int CODE>
__device__ __forceinline__ uint32_t kv8_pack(float a, float b, float c, float d) {
  if constexpr (CODE == KV8_E4M3) {
    uint32_t r;
    asm("{\n\t.reg .b16 lo, hi;\n\tcvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n\tcvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n\tmov.b32 %0, {lo, hi};\n\t}"
        : "=r"(r) : "f"(a), "f"(b), "f"(c), "f"(d));
    return r;
  } else {
    // the units of 1.5 * 2^23 + x are whole numbers: the low byte of its bits is x in two's complement
    constexpr float M = 12582912.f;
    const uint32_t lo = __byte_perm(__float_as_uint(a + M), __float_as_uint(b + M), 0x0040), hi = __byte_perm(__float_as_uint(c + M), __float_as_uint(d + M), 0x0040);
    return __byte_perm(lo, hi, 0x5410);
  }
}
// the codes in the bytes 0 and 1 (and 2 and 3) of w as fp16, exactly
template <int CODE>
__device__ __forceinline__ void kv8_unpack(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (CODE == KV8_E4M3) {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}" : "=r"(lo), "=r"(hi) : "r"(w));
  } else {
    // 1024 + (x + 128) has x + 128 in its low byte
    const uint32_t u = w ^ 0x80808080u;
    lo = __byte_perm(u, 0x64646464u, 0x4140), hi = __byte_perm(u, 0x64646464u, 0x4342);
    asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(lo) : "r"(0x64806480u));
    asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(hi) : "r"(0x64806480u));
  }
}
__device__ __forceinline__ float h_lo(uint32_t p) { return __half2float(__ushort_as_half((unsigned short)(p & 0xffffu))); }
__device__ __forceinline__ float h_hi(uint32_t p) { return __half2float(__ushort_as_half((unsigned short)(p >> 16))); }
// bytes that are e4m3's code for no number (sign aside): 0x80 in their place, 0 elsewhere
__device__ __forceinline__ uint32_t kv8_nans(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

}  // namespace qie
