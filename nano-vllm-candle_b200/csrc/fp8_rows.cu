// Rows and weights in 8 bits (fp8.cuh):
//   nvc_quant_fp8_rows     rows as they are or through an activation unit, gathered or not
//   nvc_add_rmsnorm_fp8    the residual sum and RMS norm in front of a product
//   nvc_quant_fp8_blocks   weights, once at load time
// All three are bound by the bytes they move.  A thread holds 16 neighbouring numbers, eight lanes a block of 128: two or four 16-byte loads per operand in
// flight, one 16-byte store, and the block's largest magnitude in three shuffles.
#include "fp8.cuh"

namespace {

constexpr int kRowsPerCta = 8;        // warps of quant_rows_kernel, one stretch of 512 columns each

// z sigmoid(z) with two to four units in the last place: exp(-z) as 2^h (1 + l ln 2), h + l = -z log2(e) with the product's rounding and the constant's in l
__device__ __forceinline__ float silu_f32(float z) {
  const float h = z * -1.44269502f, l = fmaf(z, -1.44269502f, -h) + z * -1.92596299e-8f;
  float e, r;
  asm("ex2.approx.f32 %0, %1;" : "=f"(e) : "f"(h));
  if (fabsf(h) < 126.0f) e = fmaf(e, l * 0.693147181f, e);      // beyond, 1 + e is 1 or too large to count; infinities stay clear of l
  asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
  return z * r;
}

template <typename T, int kAct>
__global__ void __launch_bounds__(32 * kRowsPerCta)
quant_rows_kernel(const T* x, int64_t ldx, int up_off, const int32_t* rows, const int32_t* num_rows, uint8_t* __restrict__ q, int64_t ldq,
                  float* __restrict__ scale, int64_t lds, int N, int H, int stretches) {
  pdl_trigger();
  const int lane = threadIdx.x & 31;
  const int64_t unit = (int64_t)blockIdx.x * kRowsPerCta + (threadIdx.x >> 5);
  const int64_t r = unit / stretches;
  const int col = (int)(unit - r * stretches) * 512 + lane * 16;
  pdl_wait();
  if (r >= N || (num_rows && r >= *num_rows)) return;          // the same for a whole warp
  const int64_t src = rows ? rows[r] : r;
  float y[16] = {};
  if (src >= 0 && col < H) {
    const T* p = x + src * ldx + col;
    load16(p, y);
    if (kAct == NVC_ACT_SILU_MUL || kAct == NVC_ACT_GELU_TANH_MUL) {
      float u[16];
      load16(p + up_off, u);
#pragma unroll
      for (int i = 0; i < 16; ++i) y[i] = (kAct == NVC_ACT_SILU_MUL ? silu_f32(y[i]) : gelu_tanh_f32(y[i])) * u[i];
    } else if (kAct == NVC_ACT_RELU2) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float v = fmaxf(y[i], 0.f);
        y[i] = v * v;
      }
    }
  }
  const float s = fp8_scale(fp8_amax8(y));
  if (col >= H) return;
  *reinterpret_cast<uint4*>(q + r * ldq + col) = fp8_pack16(y, 1.0f / s);
  if ((lane & 7) == 0) scale[r * lds + col / kFp8Block] = s;
}

// One CTA per row, which stays in registers between the sum of squares and the way out.
template <typename T, typename W>
__global__ void __launch_bounds__(1024)
add_rmsnorm_fp8_kernel(const T* x, const float* res_in, float* res_out, const W* __restrict__ w, float eps, uint8_t* __restrict__ q, int64_t ldq,
                       float* __restrict__ scale, int64_t lds, nvc_bf16* __restrict__ out, int H) {
  __shared__ float part[32];
  pdl_trigger();
  const int col = threadIdx.x * 16, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const int64_t r = blockIdx.x, at = r * H + col;
  const bool in = col < H;
  float g[16] = {}, y[16] = {};
  if (in) load16(reinterpret_cast<const W*>(w) + col, g);      // never written by a kernel: in front of the wait
  pdl_wait();
  float ss = 0.f;
  if (in) {
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

// One CTA per block of 128 x 128: 32 rows at a time, eight threads each, four times; the numbers stay in registers.
template <typename T>
__global__ void __launch_bounds__(256)
quant_blocks_kernel(const T* w, uint8_t* __restrict__ q, float* __restrict__ scale, int N, int K) {
  __shared__ float part[8];
  const int col = blockIdx.x * kFp8Block + (threadIdx.x & 7) * 16, row0 = blockIdx.y * kFp8Block + (threadIdx.x >> 3);
  const int64_t first = (int64_t)blockIdx.z * N;               // the group's first row
  float y[4][16] = {};
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (col < K && row0 + 32 * i < N) load16(w + (first + row0 + 32 * i) * K + col, y[i]);
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 16; ++j) m = fmaxf(m, fabsf(y[i][j]));
  m = warp_max(m);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = m;
  __syncthreads();
  m = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = fmaxf(m, part[i]);
  const float s = fp8_scale(m), inv = 1.0f / s;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (col < K && row0 + 32 * i < N) *reinterpret_cast<uint4*>(q + (first + row0 + 32 * i) * K + col) = fp8_pack16(y[i], inv);
  if (threadIdx.x == 0) scale[((int64_t)blockIdx.z * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x] = s;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
bool dtype_ok(int dt) { return dt == NVC_DT_BF16 || dt == NVC_DT_F32; }

}  // namespace

extern "C" int nvc_quant_fp8_rows(nvc_ctx* ctx, const void* x, int x_dtype, int ldx, int act, int up_off, const int32_t* rows, const int32_t* num_rows, nvc_fp8* q,
                                  int ldq, float* scale, int lds, int N, int H, void* stream) {
  NVC_REQUIRE(ctx, ctx && x && q && scale, NVC_EINVAL, "null pointer");
  NVC_REQUIRE(ctx, N >= 0 && H > 0 && dtype_ok(x_dtype), NVC_EINVAL, "bad sizes or dtype");
  NVC_REQUIRE(ctx, act == NVC_ACT_NONE || act == NVC_ACT_RELU2 || act == NVC_ACT_GELU_TANH_MUL || act == NVC_ACT_SILU_MUL, NVC_EINVAL,
              "act must be NVC_ACT_NONE, _RELU2, _GELU_TANH_MUL or _SILU_MUL");
  const bool gated = act == NVC_ACT_GELU_TANH_MUL || act == NVC_ACT_SILU_MUL;
  NVC_REQUIRE(ctx, H % 16 == 0, NVC_ESHAPE, "H must be a multiple of 16");
  NVC_REQUIRE(ctx, !gated || (up_off >= H && up_off % 16 == 0), NVC_ESHAPE, "the second half must start at a multiple of 16 behind the first");
  NVC_REQUIRE(ctx, ldx % 8 == 0 && ldx >= (gated ? (int64_t)up_off + H : H) && ldq % 16 == 0 && ldq >= H && lds >= (H + kFp8Block - 1) / kFp8Block, NVC_ESHAPE,
              "row strides must cover the rows, x's be a multiple of 8 and q's of 16");
  NVC_REQUIRE(ctx, aligned16(x) && aligned16(q), NVC_EINVAL, "pointers must be 16-byte aligned");
  if (N == 0) return NVC_OK;
  const int stretches = (H + 511) / 512;
  const int64_t ctas = ((int64_t)N * stretches + kRowsPerCta - 1) / kRowsPerCta;
  NVC_REQUIRE(ctx, ctas <= 0x7fffffffLL, NVC_ESHAPE, "too many rows");
  DeviceGuard guard(ctx->device);
  NVC_DISPATCH_DT(x_dtype, T, {
    auto* kernel = act == NVC_ACT_SILU_MUL ? quant_rows_kernel<T, NVC_ACT_SILU_MUL>
                   : act == NVC_ACT_GELU_TANH_MUL ? quant_rows_kernel<T, NVC_ACT_GELU_TANH_MUL>
                   : act == NVC_ACT_RELU2 ? quant_rows_kernel<T, NVC_ACT_RELU2> : quant_rows_kernel<T, NVC_ACT_NONE>;
    NVC_CUDA_CHECK(ctx, nvc_launch(ctx, kernel, dim3((unsigned)ctas), dim3(32 * kRowsPerCta), 0, nvc_stream(stream), static_cast<const T*>(x), (int64_t)ldx, up_off, rows,
                                   num_rows, q, (int64_t)ldq, scale, (int64_t)lds, N, H, stretches));
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
  const int threads = (H / 16 + 31) / 32 * 32;
  DeviceGuard guard(ctx->device);
  NVC_DISPATCH_DT(x_dtype, T, {
    const T* xt = static_cast<const T*>(x);
    if (w_dtype == NVC_DT_F32)
      NVC_CUDA_CHECK(ctx, nvc_launch(ctx, add_rmsnorm_fp8_kernel<T, float>, dim3(N), dim3(threads), 0, nvc_stream(stream), xt, residual_in, residual_out,
                                     static_cast<const float*>(w), eps, q, (int64_t)ldq, scale, (int64_t)lds, out, H));
    else
      NVC_CUDA_CHECK(ctx, nvc_launch(ctx, add_rmsnorm_fp8_kernel<T, __nv_bfloat16>, dim3(N), dim3(threads), 0, nvc_stream(stream), xt, residual_in, residual_out,
                                     static_cast<const __nv_bfloat16*>(w), eps, q, (int64_t)ldq, scale, (int64_t)lds, out, H));
  });
  NVC_CUDA_CHECK(ctx, cudaGetLastError());
  ctx->launches++;
  return NVC_OK;
}

// Launched without an early start of its own and without one for the kernel behind it: its results are weights, which the products read ahead of their wait.
extern "C" int nvc_quant_fp8_blocks(nvc_ctx* ctx, const void* w, int w_dtype, nvc_fp8* q, float* scale, int groups, int N, int K, void* stream) {
  NVC_REQUIRE(ctx, ctx && w && q && scale, NVC_EINVAL, "null pointer");
  NVC_REQUIRE(ctx, groups >= 0 && N > 0 && K > 0 && dtype_ok(w_dtype), NVC_EINVAL, "bad sizes or dtype");
  const int rows = (N + kFp8Block - 1) / kFp8Block;
  NVC_REQUIRE(ctx, K % 16 == 0 && rows <= 65535 && groups <= 65535, NVC_ESHAPE, "K must be a multiple of 16, groups and N / 128 at most 65 535");
  NVC_REQUIRE(ctx, aligned16(w) && aligned16(q), NVC_EINVAL, "pointers must be 16-byte aligned");
  if (groups == 0) return NVC_OK;
  const dim3 grid((K + kFp8Block - 1) / kFp8Block, rows, groups);
  DeviceGuard guard(ctx->device);
  NVC_DISPATCH_DT(w_dtype, T, { quant_blocks_kernel<T><<<grid, 256, 0, nvc_stream(stream)>>>(static_cast<const T*>(w), q, scale, N, K); });
  NVC_CUDA_CHECK(ctx, cudaGetLastError());
  ctx->launches++;
  return NVC_OK;
}
