// Rows and weights in 8 bits (fp8.cuh):
//   nvc_quant_fp8_rows     rows as they are or through an activation unit, gathered or not
//   nvc_add_rmsnorm_fp8    the residual sum and RMS norm in front of a product
//   nvc_quant_fp8_blocks   weights, once at load time
// All three are bound by the bytes they move.  A thread holds 16 neighbouring numbers, eight lanes a block of 128: two or four 16-byte loads per operand in
// flight, one 16-byte store, and the block's largest magnitude in three shuffles.
#include "fp8.cuh"
#include "internal.h"
#include "ptx.cuh"

#include <algorithm>

namespace {

constexpr int kRowsPerCta = 8;        // warps of quant_rows_kernel, one stretch of 512 columns each

// Two numbers at a time: the same fp32 operations, half the instructions
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\tfma.rn.f32x2 x, x, y, z;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// z sigmoid(w) = z c / (c (1 + exp(-w))), where w < 0 wherever z is far below 0: exp(-w) = 2^d exp(r), after Cody and Waite: d the multiple of 2^-11 next to -w / ln 2,
// r = -w - d ln 2 with ln 2 in two parts (to fp32, and the rest), exp(r) = 1 + r as |r| < 2^-12.4.  d and d + log2 c are exact, so the exponential has the hardware's 2^-22, at any w;
// with it the reciprocal's 2^-23, r^2 / 2 < 2^-25.8 and four roundings: below 2^-20.
// c = 2^-32 for w <= -1, so that neither the hardware's exponential nor its reciprocal, which know no denormals here, leave the normal numbers where the result has not; there z is no small
// number, and z c has all its digits.  c = 1 elsewhere, where z may be as small or large as a number can be, and the sigmoid is a quarter or more.  w is held where the result is
// z or 0 (an infinite z stays one).
// These units bound their passes: 34 instructions for a number, with exponential and reciprocal for denormals and one number at a time, took 119 us for 8 191 x 12 288
// gated rows, these 91 (gelu 98; without a choice of c 86, but there 1e-36 had no digits left).
__device__ __forceinline__ float2 times_sigmoid(float2 z, float2 w) {
  const float2 v = make_float2(fminf(fmaxf(w.x, -120.0f), 88.0f), fminf(fmaxf(w.y, -120.0f), 88.0f));
  float2 near;                                   // 0 for w <= -1, else 1: no number lies between -1 and -1 + 2^-40
  asm("fma.rn.sat.f32 %0, %1, 0f53800000, 0f53800000;" : "=f"(near.x) : "f"(v.x));
  asm("fma.rn.sat.f32 %0, %1, 0f53800000, 0f53800000;" : "=f"(near.y) : "f"(v.y));
  const float2 c = add2(near, both(2.32830644e-10f)), shift = fma2(near, both(32.0f), both(-32.0f));
  const float2 d = add2(fma2(v, both(-1.44269502f), both(6144.0f)), both(-6144.0f)), h = add2(d, shift);          // a number from 4 096 on has whole multiples of 2^-11
  const float2 n = make_float2(-v.x, -v.y);
  const float2 r = fma2(d, both(1.90465421e-9f), fma2(d, both(-0.693147182f), n));
  float2 e, q;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(h.x));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(h.y));
  e = fma2(e, add2(r, both(1.0f)), c);
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(q.x) : "f"(e.x));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(q.y) : "f"(e.y));
  return mul2(mul2(z, c), q);
}
// gated units of 16 numbers; gelu: 0.5 z (1 + tanh(a)) = z sigmoid(2 a), a = sqrt(2 / pi) (z + 0.044715 z^3): no digits are lost where tanh is near -1
template <int kAct>
__device__ __forceinline__ void gate16(float* y, const float* u) {
#pragma unroll
  for (int i = 0; i < 16; i += 2) {
    const float2 z = make_float2(y[i], y[i + 1]);
    const float2 w = kAct == NVC_ACT_SILU_MUL ? z : mul2(z, fma2(mul2(z, z), both(0.0713548163f), both(1.59576912f)));
    const float2 t = mul2(times_sigmoid(z, w), make_float2(u[i], u[i + 1]));
    y[i] = t.x;
    y[i + 1] = t.y;
  }
}

// 16 numbers as they were read
struct Packed16 {
  uint4 u[2];
  __device__ __forceinline__ void load(const __nv_bfloat16* p) {
    u[0] = ld_once_u4(p);
    u[1] = ld_once_u4(p + 8);
  }
  __device__ __forceinline__ void get(float* f) const {
    unpack8(u[0], f);
    unpack8(u[1], f + 8);
  }
};
struct Plain16 {
  float v[16];
  __device__ __forceinline__ void load(const float* p) { load16(p, v); }
  __device__ __forceinline__ void get(float* f) const {
#pragma unroll
    for (int i = 0; i < 16; ++i) f[i] = v[i];
  }
};

template <typename T> struct HeldOf { using type = Plain16; };
template <> struct HeldOf<__nv_bfloat16> { using type = Packed16; };

// A warp takes a stretch of 512 columns of a row, or, kLoop, one after the other, with the next stretch's numbers under way while it works on one.
// kFlat: blocks of all rows one behind the other, four to a warp, where stretches would leave lanes without columns (8 191 x 1 040: 6.7 us in stretches).
template <typename T, int kAct, bool kLoop, bool kFlat>
__global__ void __launch_bounds__(32 * kRowsPerCta)
quant_rows_kernel(const T* x, int64_t ldx, int x_rows, int up_off, const int32_t* rows, const int32_t* num_rows, uint8_t* __restrict__ q, int64_t ldq,
                  float* __restrict__ scale, int64_t lds, int N, int H, int parts) {
  using Held = typename HeldOf<T>::type;
  constexpr bool kGated = kAct == NVC_ACT_SILU_MUL || kAct == NVC_ACT_GELU_TANH_MUL;
  pdl_trigger();
  const int lane = threadIdx.x & 31;
  const int64_t step = (int64_t)gridDim.x * kRowsPerCta;
  int64_t unit = (int64_t)blockIdx.x * kRowsPerCta + (threadIdx.x >> 5);
  pdl_wait();
  // parts of a row: stretches, or blocks
  const int n = num_rows ? min(N, max(*num_rows, 0)) : N;
  const int64_t units = kFlat ? ((int64_t)n * parts + 3) / 4 : (int64_t)n * parts;
  Held y_next, u_next;
  int64_t r_next = 0;
  int col_next = 0;
  bool there = false;
  auto fetch = [&](int64_t at) {
    if (at >= units) return;                     // the same for a whole warp
    if (kFlat) {
      const uint32_t b = (uint32_t)at * 4 + (lane >> 3), r = b / (uint32_t)parts;      // fewer than 2^32 blocks
      r_next = r;
      col_next = r < (uint32_t)n ? (int)(b - r * parts) * kFp8Block + (lane & 7) * 16 : H;
    } else {
      r_next = at / parts;
      col_next = (int)(at - r_next * parts) * 512 + lane * 16;
    }
    there = col_next < H;
    if (!there) return;
    const int64_t src = rows ? rows[r_next] : r_next;
    there = src >= 0 && (!rows || src < x_rows);
    if (there) {
      const T* p = x + src * ldx + col_next;
      y_next.load(p);
      if (kGated) u_next.load(p + up_off);
    }
  };
  fetch(unit);
  while (unit < units) {
    float y[16] = {};
    if (there) {
      y_next.get(y);
      if (kGated) {
        float u[16];
        u_next.get(u);
        gate16<kAct>(y, u);
      } else if (kAct == NVC_ACT_RELU2) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          float v;                                 // a NaN stays one (8 191 x 12 288 53.0 us; by a comparison 57.0)
          asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(v) : "f"(y[i]));
          y[i] = v * v;
        }
      }
    }
    const int64_t r = r_next;
    const int col = col_next;
    if (kLoop) {
      unit += step;
      fetch(unit);
    }
    const float s = fp8_scale(fp8_amax8(y));
    if (col < H) {
      *reinterpret_cast<uint4*>(q + r * ldq + col) = fp8_pack16(y, 1.0f / s);
      if ((lane & 7) == 0) scale[r * lds + col / kFp8Block] = s;
    }
    if (!kLoop) break;
  }
}

// One CTA per row, which stays in registers between the sum of squares and the way out.
template <typename T, typename W>
__global__ void __launch_bounds__(1024)
add_rmsnorm_fp8_kernel(const T* x, const float* res_in, float* res_out, const W* w, float eps, uint8_t* __restrict__ q, int64_t ldq,
                       float* __restrict__ scale, int64_t lds, nvc_bf16* __restrict__ out, int H) {
  __shared__ float part[32];
  pdl_trigger();
  const int col = threadIdx.x * 16, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const int64_t r = blockIdx.x, at = r * H + col;
  const bool in = col < H;
  float g[16] = {}, y[16] = {};
  pdl_wait();
  float ss = 0.f;
  if (in) {
    load16(w + col, g);
    load16(x + at, y);
    if (res_in) {
      float a[16];
      load16(res_in + at, a);
#pragma unroll
      for (int i = 0; i < 16; ++i) y[i] += a[i];
    }
    if (res_out) {
#pragma unroll
      for (int i = 0; i < 4; ++i) *reinterpret_cast<float4*>(res_out + at + 4 * i) = make_float4(y[4 * i], y[4 * i + 1], y[4 * i + 2], y[4 * i + 3]);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) ss += y[i] * y[i];
  }
  ss = warp_sum(ss);
  if (lane == 0) part[threadIdx.x >> 5] = ss;
  __syncthreads();
  const float total = warp_sum(lane < warps ? part[lane] : 0.f);
  const float rstd = 1.0f / sqrtf(total / (float)H + eps);
#pragma unroll
  for (int i = 0; i < 16; ++i) y[i] = y[i] * rstd * g[i];
  const float s = fp8_scale(fp8_amax8(y));
  if (!in) return;
  *reinterpret_cast<uint4*>(q + r * ldq + col) = fp8_pack16(y, 1.0f / s);
  if ((lane & 7) == 0) scale[r * lds + col / kFp8Block] = s;
  if (out) {
    *reinterpret_cast<uint4*>(out + at) = pack8(y);
    *reinterpret_cast<uint4*>(out + at + 8) = pack8(y + 8);
  }
}

// Many rows: CTAs that go from row to row, with the next rows on their way into a ring in shared memory, one copy per row and operand.  The barrier inside the sum of
// squares is also the one behind which the row's place is free again.  A lane holds four neighbouring numbers of each of its warp's four blocks, so that every access of
// a warp is to neighbouring bytes.
// 16 000 x 4 096 bf16 with residual and bf16 rows beside (852 MB, floor 130 us): a CTA per row with the loads in front 164 us, this 146.
template <typename T>
__device__ __forceinline__ float4 lds4(const uint8_t* p);
template <>
__device__ __forceinline__ float4 lds4<float>(const uint8_t* p) { return *reinterpret_cast<const float4*>(p); }
template <>
__device__ __forceinline__ float4 lds4<__nv_bfloat16>(const uint8_t* p) {
  const uint2 u = *reinterpret_cast<const uint2*>(p);
  return make_float4(bf16_lo(u.x), bf16_hi(u.x), bf16_lo(u.y), bf16_hi(u.y));
}

template <typename T, typename W>
__global__ void __launch_bounds__(1024)
add_rmsnorm_fp8_ring_kernel(const T* x, const float* res_in, float* res_out, const W* w, float eps, uint8_t* __restrict__ q, int64_t ldq,
                            float* __restrict__ scale, int64_t lds, nvc_bf16* __restrict__ out, int N, int H, int stages) {
  extern __shared__ __align__(16) uint8_t ring[];
  __shared__ float part[2][32];
  __shared__ __align__(8) uint64_t bars[4];
  pdl_trigger();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const uint32_t x_bytes = H * sizeof(T), row_bytes = x_bytes + (res_in ? H * 4 : 0);
  const uint32_t bar0 = smem_u32(bars), ring0 = smem_u32(ring);
  auto fetch = [&](int64_t r, int s) {
    ptx::mbar_arrive_expect_tx(bar0 + 8 * s, row_bytes);
    ptx::bulk_load(ring0 + s * row_bytes, x + r * H, x_bytes, bar0 + 8 * s);
    if (res_in) ptx::bulk_load(ring0 + s * row_bytes + x_bytes, res_in + r * H, H * 4, bar0 + 8 * s);
  };
  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) ptx::mbar_init(bar0 + 8 * s, 1);
    ptx::fence_barrier_init();
  }
  __syncthreads();
  pdl_wait();
  if (threadIdx.x == 0)
    for (int s = 0; s < stages; ++s)
      if ((int64_t)blockIdx.x + (int64_t)s * gridDim.x < N) fetch((int64_t)blockIdx.x + (int64_t)s * gridDim.x, s);
  float4 g[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int col = warp * 512 + i * 128 + lane * 4;
    g[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (col < H) g[i] = lds4<W>(reinterpret_cast<const uint8_t*>(w + col));
  }
  // this thread's first number of a row in every operand; its four blocks are 128 numbers apart
  const int col0 = warp * 512 + lane * 4;
  uint32_t in = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) in |= (col0 + i * 128 < H ? 1u : 0u) << i;
  const float inv_h = 1.0f / (float)H;
  const int64_t step = gridDim.x;
  uint8_t* q_at = q + blockIdx.x * ldq + col0;
  float* scale_at = scale + blockIdx.x * lds + warp * 4 + lane;
  float* res_at = res_out + blockIdx.x * (int64_t)H + col0;
  nvc_bf16* out_at = out + blockIdx.x * (int64_t)H + col0;
  const bool writes_scale = lane < 4 && warp * 512 + lane * 128 < H;
  int it = 0, s = 0, phase = 0;
  for (int64_t r = blockIdx.x; r < N; r += step, ++it) {
    float4 y[4];
    float2 ss = both(0.f);
    ptx::mbar_wait(bar0 + 8 * s, phase);
    const uint8_t* xs = ring + s * row_bytes + col0 * sizeof(T);
    const uint8_t* rs = ring + s * row_bytes + x_bytes + col0 * 4;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      y[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (in >> i & 1) {
        y[i] = lds4<T>(xs + i * 128 * sizeof(T));
        if (res_in) {
          const float4 a = lds4<float>(rs + i * 512);
          y[i].x += a.x; y[i].y += a.y; y[i].z += a.z; y[i].w += a.w;
        }
        if (res_out) *reinterpret_cast<float4*>(res_at + i * 128) = y[i];
      }
      const float2 lo = make_float2(y[i].x, y[i].y), hi = make_float2(y[i].z, y[i].w);
      ss = fma2(hi, hi, fma2(lo, lo, ss));
    }
    const float sum = warp_sum(ss.x + ss.y);
    if (lane == 0) part[it & 1][warp] = sum;
    __syncthreads();
    if (threadIdx.x == 0 && r + stages * step < N) fetch(r + stages * step, s);
    if (++s == stages) { s = 0; phase ^= 1; }
    const float v = fmaf(warp_sum(lane < warps ? part[it & 1][lane] : 0.f), inv_h, eps);
    float rstd = rsqrtf(v);                      // off by two units at most; a Newton step leaves one
    rstd = v < 1e38f && v > 1e-30f ? fmaf(rstd * 0.5f, fmaf(-v * rstd, rstd, 1.0f), rstd) : 1.0f / sqrtf(v);
    // a lane takes the scale of one of the four blocks: its two divisions are as long as all else that is done for four numbers
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 lo = mul2(mul2(make_float2(y[i].x, y[i].y), both(rstd)), make_float2(g[i].x, g[i].y)), hi = mul2(mul2(make_float2(y[i].z, y[i].w), both(rstd)), make_float2(g[i].z, g[i].w));
      y[i] = make_float4(lo.x, lo.y, hi.x, hi.y);
      // magnitudes' bits are in the order of the magnitudes; four NaN are none
      const float m = fmaxf(fmaxf(fmaxf(fabsf(y[i].x), fabsf(y[i].y)), fmaxf(fabsf(y[i].z), fabsf(y[i].w))), 0.f);
      const uint32_t all = __reduce_max_sync(0xffffffffu, __float_as_uint(m));
      if ((lane & 3) == i) top = __uint_as_float(all);
    }
    const float mine = fp8_scale(top), my_inv = 1.0f / mine;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float inv = __shfl_sync(0xffffffffu, my_inv, i);
      if (in >> i & 1) {
        const float2 lo = mul2(make_float2(y[i].x, y[i].y), both(inv)), hi = mul2(make_float2(y[i].z, y[i].w), both(inv));
        *reinterpret_cast<uint32_t*>(q_at + i * 128) = fp8_pack4(lo.x, lo.y, hi.x, hi.y);
        if (out) *reinterpret_cast<uint2*>(out_at + i * 128) = make_uint2(pack_bf16(y[i].x, y[i].y), pack_bf16(y[i].z, y[i].w));
      }
    }
    if (writes_scale) *scale_at = mine;
    q_at += step * ldq;
    scale_at += step * lds;
    res_at += step * H;
    out_at += step * H;
  }
}

// One CTA per block of 128 x 128: 32 rows at a time, eight threads each, four times; the numbers stay in registers, bf16 ones as they are (unpacked they took 87
// registers, two CTAs per SM and 1.8 times as long).  Four CTAs (three for fp32) share an SM: 24 576 x 4 096 bf16 47.6 us.
template <typename T, typename Held>
__global__ void __launch_bounds__(256, (sizeof(T) == 2 ? 4 : 3))
quant_blocks_kernel(const T* w, uint8_t* __restrict__ q, float* __restrict__ scale, int N, int K) {
  __shared__ float part[8];
  pdl_wait();
  const int col = blockIdx.x * kFp8Block + (threadIdx.x & 7) * 16, row0 = blockIdx.y * kFp8Block + (threadIdx.x >> 3);
  const int64_t first = (int64_t)blockIdx.z * N;               // the group's first row
  Held y[4] = {};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (col < K && row0 + 32 * i < N) y[i].load(w + (first + row0 + 32 * i) * K + col);
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float f[16];
    y[i].get(f);
#pragma unroll
    for (int j = 0; j < 16; ++j) m = fmaxf(m, fabsf(f[j]));
  }
  m = warp_max(m);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = m;
  __syncthreads();
  m = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = fmaxf(m, part[i]);
  const float s = fp8_scale(m), inv = 1.0f / s;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (col < K && row0 + 32 * i < N) {
      float f[16];
      y[i].get(f);
      *reinterpret_cast<uint4*>(q + (first + row0 + 32 * i) * K + col) = fp8_pack16(f, inv);
    }
  }
  if (threadIdx.x == 0) scale[((int64_t)blockIdx.z * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x] = s;
}

template <typename T, bool kFlat>
auto* rows_kernel(int act) {
  return act == NVC_ACT_SILU_MUL ? quant_rows_kernel<T, NVC_ACT_SILU_MUL, true, kFlat>
         : act == NVC_ACT_GELU_TANH_MUL ? quant_rows_kernel<T, NVC_ACT_GELU_TANH_MUL, true, kFlat>
         : act == NVC_ACT_RELU2 ? quant_rows_kernel<T, NVC_ACT_RELU2, false, kFlat> : quant_rows_kernel<T, NVC_ACT_NONE, false, kFlat>;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
bool dtype_ok(int dt) { return dt == NVC_DT_BF16 || dt == NVC_DT_F32; }

}  // namespace

extern "C" int nvc_quant_fp8_rows(nvc_ctx* ctx, const void* x, int x_dtype, int ldx, int x_rows, int act, int up_off, const int32_t* rows, const int32_t* num_rows, nvc_fp8* q,
                                  int ldq, float* scale, int lds, int N, int H, void* stream) {
  NVC_REQUIRE(ctx, ctx && (x || x_rows == 0) && q && scale, NVC_EINVAL, "null pointer");
  NVC_REQUIRE(ctx, N >= 0 && H > 0 && x_rows >= 0 && dtype_ok(x_dtype), NVC_EINVAL, "bad sizes or dtype");
  NVC_REQUIRE(ctx, rows || N <= x_rows, NVC_EINVAL, "more rows than x has");
  NVC_REQUIRE(ctx, act == NVC_ACT_NONE || act == NVC_ACT_RELU2 || act == NVC_ACT_GELU_TANH_MUL || act == NVC_ACT_SILU_MUL, NVC_EINVAL,
              "act must be NVC_ACT_NONE, _RELU2, _GELU_TANH_MUL or _SILU_MUL");
  const bool gated = act == NVC_ACT_GELU_TANH_MUL || act == NVC_ACT_SILU_MUL;
  NVC_REQUIRE(ctx, H <= 0x7fffffff - 512, NVC_ESHAPE, "too many rows or too wide");          // column numbers of the last stretch
  NVC_REQUIRE(ctx, H % 16 == 0, NVC_ESHAPE, "H must be a multiple of 16");
  NVC_REQUIRE(ctx, !gated || (up_off >= H && up_off % 16 == 0), NVC_ESHAPE, "the second half must start at a multiple of 16 behind the first");
  NVC_REQUIRE(ctx, ldx % 8 == 0 && ldx >= (gated ? (int64_t)up_off + H : H) && ldq % 16 == 0 && ldq >= H && lds >= (H + kFp8Block - 1) / kFp8Block, NVC_ESHAPE,
              "row strides must cover the rows, x's be a multiple of 8 and q's of 16");
  NVC_REQUIRE(ctx, aligned16(x) && aligned16(q), NVC_EINVAL, "pointers must be 16-byte aligned");
  if (N == 0) return NVC_OK;
  const int stretches = (H + 511) / 512, blocks = (H + kFp8Block - 1) / kFp8Block;
  // lanes without columns in more than a tenth of the stretches
  const bool flat = 40 * stretches > 11 * blocks && (int64_t)N * blocks < 0xfffffff0LL;
  const int64_t ctas = ((flat ? ((int64_t)N * blocks + 3) / 4 : (int64_t)N * stretches) + kRowsPerCta - 1) / kRowsPerCta;
  NVC_REQUIRE(ctx, ctas <= 0x7fffffffLL, NVC_ESHAPE, "too many rows");
  // gated units of large inputs go on from stretch to stretch (with a lighter unit 64 x 12 288 bf16 2.7 us for 3.5, 8 191 x 12 288 87 for 89); nothing to gain where nothing is computed (49 for 55)
  const int64_t grid = gated && ctas > (int64_t)ctx->num_sms * 16 ? (int64_t)ctx->num_sms * 16 : ctas;
  DeviceGuard guard(ctx->device);
  NVC_DISPATCH_DT(x_dtype, T, {
    auto* kernel = flat ? rows_kernel<T, true>(act) : rows_kernel<T, false>(act);
    NVC_CUDA_CHECK(ctx, nvc_launch(ctx, kernel, dim3((unsigned)grid), dim3(32 * kRowsPerCta), 0, nvc_stream(stream), static_cast<const T*>(x), (int64_t)ldx, x_rows, up_off, rows,
                                   num_rows, q, (int64_t)ldq, scale, (int64_t)lds, N, H, flat ? blocks : stretches));
  });
  NVC_CUDA_CHECK(ctx, cudaGetLastError());
  ctx->launches++;
  return NVC_OK;
}

extern "C" int nvc_add_rmsnorm_fp8(nvc_ctx* ctx, const void* x, int x_dtype, const float* residual_in, float* residual_out, const void* w, int w_dtype, float eps, nvc_fp8* q,
                                   int ldq, float* scale, int lds, nvc_bf16* out, int N, int H, void* stream) {
  NVC_REQUIRE(ctx, ctx && x && w && q && scale, NVC_EINVAL, "null pointer");
  NVC_REQUIRE(ctx, N >= 0 && H > 0 && dtype_ok(x_dtype) && dtype_ok(w_dtype), NVC_EINVAL, "bad sizes or dtype");
  NVC_REQUIRE(ctx, H % 16 == 0 && H <= 16384, NVC_ESHAPE, "H must be a multiple of 16 and <= 16384");
  NVC_REQUIRE(ctx, ldq % 16 == 0 && ldq >= H && lds >= (H + kFp8Block - 1) / kFp8Block, NVC_ESHAPE, "row strides must cover the rows, q's be a multiple of 16");
  NVC_REQUIRE(ctx, aligned16(x) && aligned16(residual_in) && aligned16(residual_out) && aligned16(w) && aligned16(q) && aligned16(out), NVC_EINVAL,
              "pointers must be 16-byte aligned");
  if (N == 0) return NVC_OK;
  DeviceGuard guard(ctx->device);
  // One way for every combination of types
  auto run = [&](auto* one, auto* ring, auto* xt, auto* wt) -> int {
    const int threads = (H / 16 + 31) / 32 * 32;                           // of either kernel
    const int row = H * ((x_dtype == NVC_DT_F32 ? 4 : 2) + (residual_in ? 4 : 0));
    const int stages = std::max(1, std::min(4, std::max(200 * 1024 / row / std::max(1024 / threads, 1), 200 * 1024 / row >= 2 ? 2 : 1)));
    const int per_sm = std::max(1, std::min({1024 / threads, 24, 200 * 1024 / (stages * row)}));
    const int64_t places = std::min<int64_t>((int64_t)ctx->num_sms * per_sm, N);
    // a ring where SMs have several rows and half a million numbers to go through (a CTA per row / ring, us: 148 x 4 096 3.2 / 4.5, 300 5.7 / 5.2, 1 200 13.7 / 10.5; 300 x 1 024
    // 2.8 / 3.3, 600 4.1 / 3.9; 1 800 x 256 4.25 / 4.06, 5 000 8.1 / 6.4)
    if (N < 2 * ctx->num_sms || (int64_t)N * H < (1 << 19)) {
      NVC_CUDA_CHECK(ctx, nvc_launch(ctx, one, dim3(N), dim3(threads), 0, nvc_stream(stream), xt, residual_in, residual_out, wt, eps, q, (int64_t)ldq, scale, (int64_t)lds, out, H));
      return NVC_OK;
    }
    NVC_CUDA_CHECK(ctx, nvc_launch(ctx, ring, dim3((unsigned)places), dim3(threads), stages * row, nvc_stream(stream), xt, residual_in, residual_out, wt, eps, q, (int64_t)ldq,
                                   scale, (int64_t)lds, out, N, H, stages));
    return NVC_OK;
  };
  int rc = NVC_OK;
  NVC_DISPATCH_DT(x_dtype, T, {
    if (w_dtype == NVC_DT_F32) rc = run(add_rmsnorm_fp8_kernel<T, float>, add_rmsnorm_fp8_ring_kernel<T, float>, static_cast<const T*>(x), static_cast<const float*>(w));
    else rc = run(add_rmsnorm_fp8_kernel<T, __nv_bfloat16>, add_rmsnorm_fp8_ring_kernel<T, __nv_bfloat16>, static_cast<const T*>(x), static_cast<const __nv_bfloat16*>(w));
  });
  if (rc) return rc;
  NVC_CUDA_CHECK(ctx, cudaGetLastError());
  ctx->launches++;
  return NVC_OK;
}

extern "C" int nvc_fp8_rows_init(nvc_ctx* ctx) {
#define X(T, W) NVC_CUDA_CHECK(ctx, (cudaFuncSetAttribute(add_rmsnorm_fp8_ring_kernel<T, W>, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024)));
  X(float, float) X(float, __nv_bfloat16) X(__nv_bfloat16, float) X(__nv_bfloat16, __nv_bfloat16)
#undef X
  return NVC_OK;
}

extern "C" int nvc_quant_fp8_blocks(nvc_ctx* ctx, const void* w, int w_dtype, nvc_fp8* q, float* scale, int groups, int N, int K, void* stream) {
  NVC_REQUIRE(ctx, ctx && w && q && scale, NVC_EINVAL, "null pointer");
  NVC_REQUIRE(ctx, groups >= 0 && N > 0 && K > 0 && dtype_ok(w_dtype), NVC_EINVAL, "bad sizes or dtype");
  NVC_REQUIRE(ctx, N <= 65535 * kFp8Block && K <= 0x7fffffff - kFp8Block && groups <= 65535, NVC_ESHAPE, "too many rows or too wide: groups and N / 128 are at most 65 535");
  NVC_REQUIRE(ctx, K % 16 == 0, NVC_ESHAPE, "K must be a multiple of 16");
  const int rows = (N + kFp8Block - 1) / kFp8Block;
  NVC_REQUIRE(ctx, aligned16(w) && aligned16(q), NVC_EINVAL, "pointers must be 16-byte aligned");
  if (groups == 0) return NVC_OK;
  const dim3 grid((K + kFp8Block - 1) / kFp8Block, rows, groups);
  DeviceGuard guard(ctx->device);
  if (w_dtype == NVC_DT_F32)
    NVC_CUDA_CHECK(ctx, nvc_launch(ctx, quant_blocks_kernel<float, Plain16>, grid, dim3(256), 0, nvc_stream(stream), static_cast<const float*>(w), q, scale, N, K));
  else
    NVC_CUDA_CHECK(ctx, nvc_launch(ctx, quant_blocks_kernel<__nv_bfloat16, Packed16>, grid, dim3(256), 0, nvc_stream(stream), static_cast<const __nv_bfloat16*>(w), q, scale, N, K));
  NVC_CUDA_CHECK(ctx, cudaGetLastError());
  ctx->launches++;
  return NVC_OK;
}
