// The 8-bit format of rows and weights: e4m3 numbers q and an fp32 scale for a block of 128 numbers along a row (of 128 x 128 in a weight); a number is
// q * scale.  scale = max(amax / 448, 2^-126) with the block's largest magnitude amax, so that the largest number becomes 448, e4m3's last, and 1 / scale
// is finite for a block of zeros too; q = x * (1 / scale), rounded to nearest even.  A NaN stays with its number and counts for no scale; an infinity
// makes its block's scale infinite, and what is computed from the block NaN.
#pragma once
#include "typed.cuh"

constexpr int kFp8Block = 128;

// Calls may come while another device is the current one.
struct DeviceGuard {
  int before = -1;
  explicit DeviceGuard(int device) {
    int now = -1;
    if (cudaGetDevice(&now) == cudaSuccess && now != device && cudaSetDevice(device) == cudaSuccess) before = now;
  }
  ~DeviceGuard() {
    if (before >= 0) cudaSetDevice(before);
  }
};

#ifdef __CUDACC__
__device__ __forceinline__ float fp8_scale(float amax) { return fmaxf(amax / 448.0f, 1.17549435e-38f); }
// four numbers -> four bytes, the first in the lowest; beyond 448 (a unit in the last place, from the two roundings above) 448, NaN 0x7f
__device__ __forceinline__ uint32_t fp8_pack4(float a, float b, float c, float d) {
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
  return (uint32_t)lo | ((uint32_t)hi << 16);
}
__device__ __forceinline__ uint4 fp8_pack16(const float* f, float inv) {
  uint4 u;
  u.x = fp8_pack4(f[0] * inv, f[1] * inv, f[2] * inv, f[3] * inv);
  u.y = fp8_pack4(f[4] * inv, f[5] * inv, f[6] * inv, f[7] * inv);
  u.z = fp8_pack4(f[8] * inv, f[9] * inv, f[10] * inv, f[11] * inv);
  u.w = fp8_pack4(f[12] * inv, f[13] * inv, f[14] * inv, f[15] * inv);
  return u;
}
// largest magnitude of 16 numbers in each of eight neighbouring lanes: a block (fmaxf passes NaN over)
__device__ __forceinline__ float fp8_amax8(const float* f) {
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) m = fmaxf(m, fabsf(f[i]));
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  return m;
}
// 16 consecutive numbers that are read once (16-byte aligned)
__device__ __forceinline__ void load16(const __nv_bfloat16* p, float* f) {
  const uint4 a = ld_once_u4(p), b = ld_once_u4(p + 8);
  unpack8(a, f);
  unpack8(b, f + 8);
}
__device__ __forceinline__ void load16(const float* p, float* f) {
  uint4 u[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) u[i] = ld_once_u4(p + 4 * i);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[4 * i] = __uint_as_float(u[i].x); f[4 * i + 1] = __uint_as_float(u[i].y);
    f[4 * i + 2] = __uint_as_float(u[i].z); f[4 * i + 3] = __uint_as_float(u[i].w);
  }
}
#endif
