// The 4-bit format of cached key and value rows.  A head's row of 128 numbers is 8 blocks of 16; a block is 16 codes in e2m1 (sign, then a magnitude of
// 0, 0.5, 1, 1.5, 2, 3, 4, 6) and one scale byte b: the fp16 number with the bits b << 7 (5 bits of exponent, 3 of mantissa, no sign).  A number is code * scale: 2 + 4
// significant bits, so that it is exact in fp16, where the products below read it.  The scale reaches from 2^-17 to 10 240 (6 * 10 240 is the last that fits fp16)
// without a second one per tensor, and costs the reader a shift.
//   scale = nearest(max|x| / 6), half way to the even mantissa, at most 10 240;  code = nearest(x / scale), half way to the smaller magnitude, at most 6.
// 255, a NaN as fp16, is the scale of a block that holds an infinity or a NaN: all its numbers read as NaN.
#pragma once
#include "common.cuh"
#include "fp8.cuh"          // DeviceGuard

constexpr int kFp4Codes = 64;          // bytes of a row's codes: number 2i in the low half of byte i, 2i + 1 in the high half
constexpr int kFp4Scales = 8;          // bytes of its scales
constexpr int kFp4MostScale = 226;     // 10 240

#ifdef __CUDACC__
// max(|x|) of a block as bf16 bits -> its scale byte
__device__ __forceinline__ uint32_t fp4_scale_byte(uint32_t amax_bits) {
  if (amax_bits >= 0x7f80u) return 255u;
  const float s = __fdiv_rn(__uint_as_float(amax_bits << 16), 6.0f);       // correctly rounded: a quotient half way between two scales is a float
  if (s < 6.103515625e-05f) return (uint32_t)__float2int_rn(s * 131072.0f);  // below 2^-14: steps of 2^-17
  const uint32_t u = __float_as_uint(s);
  const uint32_t r = ((u + 0x7ffffu + ((u >> 20) & 1u)) >> 20) - ((127 - 15) << 3);
  return r > kFp4MostScale ? kFp4MostScale : r;
}
__device__ __forceinline__ float fp4_scale(uint32_t byte) { return __half2float(__ushort_as_half((unsigned short)(byte << 7))); }
// 1 / scale, a millionth part smaller: a quotient of a bf16 number (8 bits) and a scale (4 bits) is at a border between codes or at least 2^-9 of its value away
// from it, so that this moves the ones at a border to the smaller magnitude, and no other
__device__ __forceinline__ float fp4_inverse(uint32_t byte) {
  return byte == 0 || byte == 255u ? 0.f : __fdiv_rn(1.0f, fp4_scale(byte)) * (1.0f - 9.5367431640625e-07f);
}
// eight numbers (bf16 pairs) -> eight codes, the first in the lowest four bits; a NaN's code is any
__device__ __forceinline__ uint32_t fp4_codes8(const uint4& x, float inv) {
  uint32_t r;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(r)
      : "f"(bf16_lo(x.x) * inv), "f"(bf16_hi(x.x) * inv), "f"(bf16_lo(x.y) * inv), "f"(bf16_hi(x.y) * inv), "f"(bf16_lo(x.z) * inv), "f"(bf16_hi(x.z) * inv),
        "f"(bf16_lo(x.w) * inv), "f"(bf16_hi(x.w) * inv));
  return r;
}
// the largest magnitude of eight numbers, as bf16 bits
__device__ __forceinline__ uint32_t fp4_amax8(const uint4& x) {
  const uint32_t m = __vmaxu2(__vmaxu2(x.x & 0x7fff7fffu, x.y & 0x7fff7fffu), __vmaxu2(x.z & 0x7fff7fffu, x.w & 0x7fff7fffu));
  return max(m & 0xffffu, m >> 16);
}
__device__ __forceinline__ void fp4_prefetch(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }
// eight codes -> four pairs of fp16 numbers
__device__ __forceinline__ uint4 fp4_halves8(uint32_t codes) {
  uint4 r;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "mov.b32 {a, b, c, d}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, a;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, c;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
      : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(codes));
  return r;
}
#endif
// n / d for n < 2^31 and a d of the host's: d's inverse, rounded up, with as many bits as that takes
struct Fp4Div {
  unsigned long long mul;
  int shift;
  __device__ __forceinline__ int operator()(int n) const { return (int)((unsigned long long)(unsigned)n * mul >> shift); }
};
inline Fp4Div fp4_div(int d) {
  int s = 0;
  while ((1ll << s) < d) ++s;
  return Fp4Div{((1ull << (32 + s)) + (unsigned long long)d - 1) / (unsigned long long)d, 32 + s};
}

