// Products of 8-bit rows and weights (fp8.cuh), dense and grouped by expert:
//   C[m, n] = sum over k-blocks b of a_scale[m, b] * w_scale[n / 128, b] * (sum over the block's k of A[m, k] * W[n, k]),  bf16 or fp32
// The inner sums run on the tensor cores (e4m3 products are exact in fp32) in an accumulator of their own per k-block; the outer sums, whose factors differ
// from block to block, in fp32 registers.
//
// A persistent grid, one CTA per SM, walks tiles of 128 x BN:
//   warp 0     TMA producer: 128 x 128 bytes of A and BN x 128 of W per k-block into a ring that runs on into the next tile
//   warp 1     tcgen05.mma M 128, N BN, K 32, four per k-block, into one of two (BN 256) or four accumulators in tensor memory
//   warps 4-11 two per quadrant of tensor memory, one for either half of the columns: accumulator times scales onto registers, rows through a staging buffer
#include "fp8.cuh"
#include "ptx.cuh"
#include "internal.h"
#include "gemm_epilogue.cuh"

namespace {

constexpr int BM = 128, BK = 128;

// e4m3 x e4m3 -> fp32: D format fp32, A and B formats 0, both K-major
__host__ __device__ constexpr uint32_t idesc_fp8(int M, int N) { return (1u << 4) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24); }

__device__ __forceinline__ void umma_fp8_ss(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate) : "memory");
}

// (a0, a1) += (d0, d1) * (s, s), both in one instruction
__device__ __forceinline__ void fma2(float2& a, uint32_t d0, uint32_t d1, float s) {
  asm("{\n\t.reg .b64 x, y, z;\n\t"
      "mov.b64 x, {%0, %1};\n\tmov.b64 y, {%2, %3};\n\tmov.b64 z, {%4, %4};\n\t"
      "fma.rn.f32x2 x, y, z, x;\n\t"
      "mov.b64 {%0, %1}, x;\n\t}"
      : "+f"(a.x), "+f"(a.y) : "r"(d0), "r"(d1), "f"(s));
}

template <int BN>
struct Cfg {
  static constexpr int kBytesA = BM * BK, kBytesB = BN * BK, kStageBytes = kBytesA + kBytesB;
  static constexpr int kStages = BN == 256 ? 4 : (BN == 128 ? 6 : 8);        // 192 KB
  static constexpr int kAcc = BN == 256 ? 2 : 4;                             // accumulators
  static constexpr int kTmemCols = kAcc * BN;
  static constexpr int kThreads = 384;
  static constexpr int kOffStaging = kStages * kStageBytes;                  // 4 KB per epilogue warp
  static constexpr int kOffBar = kOffStaging + 8 * 4096;
  static constexpr int kNumBars = 2 * kStages + 2 * kAcc;
  static constexpr int kSmemBytes = kOffBar + kNumBars * 8 + 16 + 1024;      // 1024: alignment by hand
  static_assert(kSmemBytes <= 232448, "shared memory per CTA");
};

struct Args {
  void* C;
  const float* a_scale;
  const float* w_scale;
  const int32_t* tile_group;        // nullptr: dense
  int64_t ldc, lds;
  int out_f32, M, N, num_kb, num_tiles, n_tiles, m_tiles, band, zero;
};

// Tile number -> row tile, column tile: bands of `band` row tiles, the row tiles of a band fastest (band 1: column tiles fastest)
__device__ __forceinline__ int2 tile_at(int tile, const Args& a) {
  if (a.band == 1) return make_int2(tile / a.n_tiles, tile % a.n_tiles);
  const int b = tile / (a.band * a.n_tiles), rest = tile - b * a.band * a.n_tiles, rows = min(a.band, a.m_tiles - b * a.band), n = rest / rows;
  return make_int2(b * a.band + rest - n * rows, n);
}

template <int BN, bool kGrouped>
__global__ void __launch_bounds__(Cfg<BN>::kThreads, 1)
gemm_fp8_kernel(const __grid_constant__ CUtensorMap tma_a, const __grid_constant__ CUtensorMap tma_b, const Args a) {
  using cfg = Cfg<BN>;
  pdl_trigger();
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* gen = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t bar0 = base + cfg::kOffBar;
  auto full_bar = [&](int s) { return bar0 + 8u * s; };
  auto empty_bar = [&](int s) { return bar0 + 8u * (cfg::kStages + s); };
  auto acc_full = [&](int i) { return bar0 + 8u * (2 * cfg::kStages + i); };
  auto acc_empty = [&](int i) { return bar0 + 8u * (2 * cfg::kStages + cfg::kAcc + i); };
  const uint32_t tmem_slot = bar0 + 8u * cfg::kNumBars;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp == 0) {
    if (lane == 0) {
      ptx::tma_prefetch_desc(&tma_a);
      ptx::tma_prefetch_desc(&tma_b);
      for (int s = 0; s < cfg::kStages; ++s) {
        ptx::mbar_init(full_bar(s), 1);
        ptx::mbar_init(empty_bar(s), 1);
      }
      for (int i = 0; i < cfg::kAcc; ++i) {
        ptx::mbar_init(acc_full(i), 1);
        ptx::mbar_init(acc_empty(i), 8);
      }
      ptx::fence_barrier_init();
    }
    __syncwarp();
  } else if (warp == 1) {
    ptx::tmem_alloc(tmem_slot, cfg::kTmemCols);
    ptx::tmem_relinquish();
  }
  ptx::tcgen05_fence_before();
  __syncthreads();
  ptx::tcgen05_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(gen + cfg::kOffBar + cfg::kNumBars * 8);
  pdl_wait();
  // every role walks the same tiles; the group of the next one is fetched a tile ahead (past L1: an earlier kernel of the stream wrote the table)
  auto group_of = [&](int tile) { return !kGrouped ? 0 : (tile < a.num_tiles ? __ldcg(a.tile_group + tile / a.n_tiles) : -1); };
  int next = group_of(blockIdx.x);
  // registers: the epilogue's two warpgroups hold up to 128 sums each thread, the first warpgroup next to nothing: 128 x 72 + 256 x 216 = 384 x 168
  if (warp < 4) asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
  if (warp == 0) {
    uint32_t it = 0;
    for (int tile = blockIdx.x; tile < a.num_tiles; tile += gridDim.x) {
      const int grp = next;
      const int2 at = tile_at(tile, a);
      next = group_of(tile + gridDim.x);
      if (kGrouped && grp < 0) continue;
      for (int kb = 0; kb < a.num_kb; ++kb, ++it) {
        const int s = it % cfg::kStages;
        ptx::mbar_wait(empty_bar(s), ((it / cfg::kStages) & 1) ^ 1u);      // first lap: falls through
        if (ptx::elect_one()) {
          ptx::mbar_arrive_expect_tx(full_bar(s), cfg::kStageBytes);
          const uint32_t dst = base + s * cfg::kStageBytes;
          ptx::tma_load_2d(dst + cfg::kBytesA, &tma_b, full_bar(s), kb * BK, grp * a.N + at.y * BN);
          ptx::tma_load_2d(dst, &tma_a, full_bar(s), kb * BK, at.x * BM);
        }
        __syncwarp();
      }
    }
  } else if (warp == 1) {
    constexpr uint32_t idesc = idesc_fp8(BM, BN), desc_hi = ptx::umma_desc_hi_sw128(1024);
    const uint32_t a_lo0 = ptx::umma_desc_lo(base, 16);
    uint32_t it = 0;
    for (int tile = blockIdx.x; tile < a.num_tiles; tile += gridDim.x) {
      const int grp = next;
      next = group_of(tile + gridDim.x);
      if (kGrouped && grp < 0) continue;
      for (int kb = 0; kb < a.num_kb; ++kb, ++it) {
        const int s = it % cfg::kStages, acc = it % cfg::kAcc;
        ptx::mbar_wait(acc_empty(acc), ((it / cfg::kAcc) & 1) ^ 1u);       // its last k-block has been read out
        ptx::mbar_wait(full_bar(s), (it / cfg::kStages) & 1);
        ptx::tcgen05_fence_after();
        if (ptx::elect_one()) {
          const uint32_t a_lo = a_lo0 + ((s * cfg::kStageBytes) >> 4), b_lo = a_lo + (cfg::kBytesA >> 4);
#pragma unroll
          for (int k = 0; k < BK / 32; ++k)        // 32 numbers are 32 bytes along K inside the 128-byte swizzle span: +2 in the address field
            umma_fp8_ss(tmem + acc * BN, ptx::umma_desc(a_lo + 2 * k, desc_hi), ptx::umma_desc(b_lo + 2 * k, desc_hi), idesc, k != 0 ? 1u : 0u);
          ptx::umma_commit(empty_bar(s));
          ptx::umma_commit(acc_full(acc));
        }
        __syncwarp();
      }
    }
  } else if (warp >= 4) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    constexpr int kCols = BN / 2, kChunk = 16, kChunks = kCols / kChunk;   // this thread's columns, and those of one read of tensor memory
    const int quad = warp & 3, side = (warp - 4) >> 2;
    const uint32_t taddr = tmem + ((uint32_t)(quad * 32) << 16) + side * kCols;
    const int w_blocks = (a.N + kFp8Block - 1) / kFp8Block;
    uint32_t it = 0;
    for (int tile = blockIdx.x; tile < a.num_tiles; tile += gridDim.x) {
      const int grp = next;
      const int2 at = tile_at(tile, a);
      next = group_of(tile + gridDim.x);
      if (kGrouped && grp < 0 && !a.zero) continue;
      const int row0 = at.x * BM + quad * 32, n0 = at.y * BN + side * kCols;
      RowStage st = make_row_stage(gen + cfg::kOffStaging + (warp - 4) * 4096, a.C, a.out_f32, NVC_EPI_NONE, a.ldc, row0, a.M, n0, kCols, a.N);
      float2 acc[kCols / 2];
#pragma unroll
      for (int j = 0; j < kCols / 2; ++j) acc[j] = make_float2(0.f, 0.f);
      if (!kGrouped || grp >= 0) {                                         // else rows that no group computes: zeros
        // rows and columns behind the last have the last one's scales, and are not stored
        const float* sa = a.a_scale + (int64_t)min(row0 + lane, a.M - 1) * a.lds;
        const float* sw = a.w_scale + ((int64_t)grp * w_blocks + min(n0 / kFp8Block, w_blocks - 1)) * a.num_kb;
        float next_a = sa[0], next_w = sw[0];
        for (int kb = 0; kb < a.num_kb; ++kb, ++it) {
          const float s = next_a * next_w;
          if (kb + 1 < a.num_kb) {
            next_a = sa[kb + 1];
            next_w = sw[kb + 1];
          }
          const int i = it % cfg::kAcc;
          ptx::mbar_wait(acc_full(i), (it / cfg::kAcc) & 1);
          ptx::tcgen05_fence_after();
          uint32_t v[2][kChunk];
          ptx::tmem_ld_32x32b_x16(taddr + i * BN, v[0]);
#pragma unroll
          for (int c = 0; c < kChunks; ++c) {
            ptx::tmem_ld_wait();
            if (c + 1 < kChunks) ptx::tmem_ld_32x32b_x16(taddr + i * BN + (c + 1) * kChunk, v[(c + 1) & 1]);
            if (c + 1 == kChunks) {                                        // read out: the accumulator may be written again
              ptx::tcgen05_fence_before();
              __syncwarp();
              if (lane == 0) ptx::mbar_arrive(acc_empty(i));
            }
#pragma unroll
            for (int j = 0; j < kChunk / 2; ++j) fma2(acc[c * (kChunk / 2) + j], v[c & 1][2 * j], v[c & 1][2 * j + 1], s);
          }
        }
      }
#pragma unroll
      for (int c = 0; c < kCols; c += 32) {
        float f[32];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          f[2 * j] = acc[c / 2 + j].x;
          f[2 * j + 1] = acc[c / 2 + j].y;
        }
        st.emit32(lane, a.out_f32, NVC_EPI_NONE, f);
      }
      st.finish(lane);
    }
  }
  ptx::tcgen05_fence_before();
  __syncthreads();
  if (warp == 1) {
    ptx::tcgen05_fence_after();
    ptx::tmem_dealloc(tmem, cfg::kTmemCols);
  }
}

int make_map(nvc_ctx* ctx, CUtensorMap* map, const void* base, uint64_t inner, uint64_t rows, uint64_t row_bytes, uint32_t box_rows) {
  cuuint64_t gdim[2] = {inner, rows}, gstr[1] = {row_bytes};
  cuuint32_t box[2] = {BK, box_rows}, estr[2] = {1, 1};
  const CUresult r = ctx->encode_tiled(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), gdim, gstr, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                       CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r == CUDA_SUCCESS) return NVC_OK;
  nvc_set_error(ctx, "cuTensorMapEncodeTiled failed with CUresult " + std::to_string((int)r));
  return NVC_EINVAL;
}

template <int BN, bool kGrouped>
int launch(nvc_ctx* ctx, const nvc_fp8* A, int lda, const nvc_fp8* W, int K, int groups, Args a, cudaStream_t st) {
  CUtensorMap ta, tb;
  int rc = make_map(ctx, &ta, A, (uint64_t)K, (uint64_t)a.M, (uint64_t)lda, BM);
  if (!rc) rc = make_map(ctx, &tb, W, (uint64_t)K, (uint64_t)a.N * groups, (uint64_t)K, BN);
  if (rc) return rc;
  a.n_tiles = (a.N + BN - 1) / BN;
  a.m_tiles = (a.M + BM - 1) / BM;
  const int64_t tiles = (int64_t)a.m_tiles * a.n_tiles;
  NVC_REQUIRE(ctx, tiles <= 0x7fffffffLL - ctx->num_sms, NVC_ESHAPE, "too many tiles");
  a.num_tiles = (int)tiles;
  const int grid = (int)(tiles < ctx->num_sms ? tiles : ctx->num_sms);
  NVC_CUDA_CHECK(ctx, nvc_launch(ctx, gemm_fp8_kernel<BN, kGrouped>, dim3(grid), dim3(Cfg<BN>::kThreads), Cfg<BN>::kSmemBytes, st, ta, tb, a));
  NVC_CUDA_CHECK(ctx, cudaGetLastError());
  ctx->launches++;
  return NVC_OK;
}

// What both products ask of their arguments.
int nvc_gemm_fp8_check(nvc_ctx* ctx, const nvc_fp8* A, int lda, const float* a_scale, int lds, const nvc_fp8* W, const float* w_scale, void* C, int ldc, int out_dtype, int M, int Nout,
          int K, int groups) {
  NVC_REQUIRE(ctx, ctx && A && a_scale && W && w_scale && C, NVC_EINVAL, "null pointer");
  NVC_REQUIRE(ctx, M >= 0 && Nout > 0 && K > 0 && groups > 0, NVC_EINVAL, "bad sizes");
  NVC_REQUIRE(ctx, K % 16 == 0 && Nout % 16 == 0, NVC_ESHAPE, "K and Nout must be multiples of 16");
  NVC_REQUIRE(ctx, lda % 16 == 0 && lda >= K && ldc % 8 == 0 && ldc >= Nout && lds >= (K + BK - 1) / BK, NVC_ESHAPE,
              "row strides must cover the rows, A's be a multiple of 16 and C's of 8");
  NVC_REQUIRE(ctx, out_dtype == NVC_DT_BF16 || out_dtype == NVC_DT_F32, NVC_EINVAL, "bad out_dtype");
  NVC_REQUIRE(ctx, ((uintptr_t)A % 16) == 0 && ((uintptr_t)W % 16) == 0 && ((uintptr_t)C % 16) == 0, NVC_EINVAL, "pointers must be 16-byte aligned");
  NVC_REQUIRE(ctx, (int64_t)Nout * groups <= 0x7fffffffLL && M <= 0x7fffffff - BM, NVC_ESHAPE, "too many rows");
  NVC_REQUIRE(ctx, ctx->encode_tiled != nullptr, NVC_EDEVICE, "cuTensorMapEncodeTiled unavailable");
  return NVC_OK;
}

}  // namespace

extern "C" int nvc_gemm_fp8_init(nvc_ctx* ctx) {
#define X(BN, G) NVC_CUDA_CHECK(ctx, (cudaFuncSetAttribute(gemm_fp8_kernel<BN, G>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<BN>::kSmemBytes)));
  X(256, false) X(128, false) X(64, false) X(256, true) X(128, true) X(64, true)
#undef X
  return NVC_OK;
}

extern "C" int nvc_gemm_fp8(nvc_ctx* ctx, const nvc_fp8* A, int lda, const float* a_scale, int lds, const nvc_fp8* W, const float* w_scale, void* C, int ldc, int out_dtype,
                            int M, int Nout, int K, void* stream) {
  int rc = nvc_gemm_fp8_check(ctx, A, lda, a_scale, lds, W, w_scale, C, ldc, out_dtype, M, Nout, K, 1);
  if (rc || M == 0) return rc;
  DeviceGuard guard(ctx->device);
  Args a = {C, a_scale, w_scale, nullptr, ldc, lds, out_dtype == NVC_DT_F32, M, Nout, (K + BK - 1) / BK, 0, 0, 0, 1, 0};
  const int64_t m_tiles = (M + BM - 1) / BM;
  if (m_tiles * ((Nout + 127) / 128) <= ctx->num_sms / 2) return launch<64, false>(ctx, A, lda, W, K, 1, a, nvc_stream(stream));
  if (m_tiles * ((Nout + 255) / 256) <= ctx->num_sms) return launch<128, false>(ctx, A, lda, W, K, 1, a, nvc_stream(stream));
  return launch<256, false>(ctx, A, lda, W, K, 1, a, nvc_stream(stream));
}

extern "C" int nvc_gemm_fp8_grouped(nvc_ctx* ctx, const nvc_fp8* A, int lda, const float* a_scale, int lds, const nvc_fp8* W, const float* w_scale, void* C, int ldc,
                                    int out_dtype, int M_cap, int Nout, int K, const int32_t* tile_group, int groups, int zero, void* stream) {
  int rc = nvc_gemm_fp8_check(ctx, A, lda, a_scale, lds, W, w_scale, C, ldc, out_dtype, M_cap, Nout, K, groups);
  if (rc) return rc;
  NVC_REQUIRE(ctx, tile_group, NVC_EINVAL, "null pointer");
  NVC_REQUIRE(ctx, M_cap % BM == 0, NVC_EINVAL, "M_cap must be a multiple of 128");
  if (M_cap == 0) return NVC_OK;
  DeviceGuard guard(ctx->device);
  Args a = {C, a_scale, w_scale, tile_group, ldc, lds, out_dtype == NVC_DT_F32, M_cap, Nout, (K + BK - 1) / BK, 0, 0, 0, 1, zero != 0};
  const int64_t m_tiles = M_cap / BM;
  if (m_tiles * ((Nout + 127) / 128) <= ctx->num_sms / 2) return launch<64, true>(ctx, A, lda, W, K, groups, a, nvc_stream(stream));
  if (m_tiles * ((Nout + 255) / 256) <= ctx->num_sms) return launch<128, true>(ctx, A, lda, W, K, groups, a, nvc_stream(stream));
  return launch<256, true>(ctx, A, lda, W, K, groups, a, nvc_stream(stream));
}
