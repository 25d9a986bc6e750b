// Products of 8-bit rows and weights (fp8.cuh), dense and grouped by expert:
//   C[m, n] = sum over k-blocks b of a_scale[m, b] * w_scale[n / 128, b] * (sum over the block's k of A[m, k] * W[n, k]),  bf16 or fp32
// The inner sums run on the tensor cores (e4m3 products are exact in fp32) in an accumulator of their own per k-block; the outer sums, whose factors differ
// from block to block, in fp32 registers.
//
// A persistent grid, one CTA per SM, walks tiles of 128 x BN:
//   warp 0     TMA producer: 128 x 128 bytes of A and BN x 128 of W per k-block into a ring that runs on into the next tile
//   warp 1     tcgen05.mma M 128, N BN, K 32, four per k-block, into one of two (BN 256) or four accumulators in tensor memory
//   warps 4-11 two per quadrant of tensor memory, one for either half of the columns: accumulator times scales onto registers, rows through shared memory and TMA
#include "fp8.cuh"
#include "ptx_pair.cuh"
#include "internal.h"

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
  asm volatile("{\n\t.reg .b64 x, y, z;\n\t"        // volatile: not in front of the wait for d0, d1
      "mov.b64 x, {%0, %1};\n\tmov.b64 y, {%2, %3};\n\tmov.b64 z, {%4, %4};\n\t"
      "fma.rn.f32x2 x, y, z, x;\n\t"
      "mov.b64 {%0, %1}, x;\n\t}"
      : "+f"(a.x), "+f"(a.y) : "r"(d0), "r"(d1), "f"(s));
}

__device__ __forceinline__ void umma_fp8_ss_pair(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate) : "memory");
}

__device__ __forceinline__ void mbar_arrive_cluster_relaxed(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}

__device__ __forceinline__ bool mbar_test(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
  return ok != 0;
}

// A thread's kCols sums over all k-blocks: accumulator it % kAcc of tensor memory (kStride columns each), times the row's and the weight block's scales.  Two warps
// of a quarter of the SM share its 512 cycles per k-block, of which the sums take 330 and the reads 256; one after the other in a warp they take longer than that.  So reads
// of 32 columns are under way two at a time, the next k-block's first two between the sums of this one's last, and whether it is there is asked for ahead of time (a
// barrier's answer takes 100 to 200 cycles beside the tensor core's own reads of shared memory).  8 192 x 24 576 x 4 096, us, numbers of zero, which leave the power cap
// out: 640 with wait, reads and sums in order, 597 with the reads ahead, 555 with the question ahead; the tensor pipe alone, without sums, 383.
// release(i): the accumulator has been read out.
template <int kCols, int kAcc, int kStride, typename Full, typename Release>
__device__ __forceinline__ void scaled_sums(float2* acc, const float* sa, const float* sw, int num_kb, uint32_t& it, uint32_t taddr, Full full, Release release) {
  static_assert(kCols == 64 || kCols == 128, "two or four reads");
  uint32_t v[2][32];
  float next_a = sa[0], next_w = sw[0];
  auto sums = [&](int c, float s) {
#pragma unroll
    for (int j = 0; j < 16; ++j) fma2(acc[c * 16 + j], v[c & 1][2 * j], v[c & 1][2 * j + 1], s);
  };
  ptx::mbar_wait(full(it % kAcc), (it / kAcc) & 1);
  ptx::tcgen05_fence_after();
  uint32_t t = taddr + it % kAcc * kStride;
  ptx::tmem_ld_32x32b_x32(t, v[0]);
  ptx::tmem_ld_32x32b_x32(t + 32, v[1]);
  for (int kb = 0; kb < num_kb; ++kb) {
    const float s = next_a * next_w;
    const bool more = kb + 1 < num_kb;
    if (more) {
      next_a = sa[kb + 1];
      next_w = sw[kb + 1];
    }
    const uint32_t next_bar = full((it + 1) % kAcc), next_parity = ((it + 1) / kAcc) & 1;
    ptx::tmem_ld_wait();
    if (kCols == 128) {
      sums(0, s);
      ptx::tmem_ld_32x32b_x32(t + 64, v[0]);
      sums(1, s);
      ptx::tmem_ld_32x32b_x32(t + 96, v[1]);
    }
    const bool ready = mbar_test(next_bar, next_parity);
    if (kCols == 128) ptx::tmem_ld_wait();
    ptx::tcgen05_fence_before();
    release(it % kAcc);
    ++it;
    sums(kCols / 32 - 2, s);
    if (more) {
      if (!ready) ptx::mbar_wait(next_bar, next_parity);
      ptx::tcgen05_fence_after();
      t = taddr + it % kAcc * kStride;
      ptx::tmem_ld_32x32b_x32(t, v[0]);
    }
    sums(kCols / 32 - 1, s);
    if (more) ptx::tmem_ld_32x32b_x32(t + 32, v[1]);
  }
}

// ---- the way out: 32 rows x 128 bytes at a time into one of the warp's kBufs buffers (16-byte chunks XOR-swizzled by row, as TMA reads them), from there by TMA, which
// knows where C ends.  The warp goes on while the copies run.
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* m, uint32_t smem_src, int32_t c0, int32_t c1) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(reinterpret_cast<uint64_t>(m)), "r"(smem_src), "r"(c0), "r"(c1) : "memory");
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
template <int kPending>
__device__ __forceinline__ void bulk_wait_read() {
  asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(kPending) : "memory");
}
__device__ __forceinline__ void bulk_wait_all() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

template <int kCols, int kBufs>
__device__ __forceinline__ void store_sums(const CUtensorMap* tma_c, uint32_t buf, uint32_t& filled, int lane, int out_f32, int row0, int M, int n0, int N, const float2* acc) {
#pragma unroll
  for (int c = 0; c < kCols / 32; ++c) {
    const bool first = out_f32 || c % 2 == 0, last = out_f32 || c % 2 == 1;       // 32 fp32 or 64 bf16 columns are 128 bytes
    if (first) {
      if (lane == 0) bulk_wait_read<kBufs - 1>();
      __syncwarp();
    }
    const uint32_t b = buf + (kBufs == 1 ? 0 : filled % kBufs * 4096), row = b + lane * 128;
    auto put = [&](int chunk, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
      asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(row + ((chunk ^ (lane & 7)) << 4)), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
    };
    const float2* f = acc + c * 16;
    if (out_f32) {
#pragma unroll
      for (int k = 0; k < 8; ++k) put(k, __float_as_uint(f[2 * k].x), __float_as_uint(f[2 * k].y), __float_as_uint(f[2 * k + 1].x), __float_as_uint(f[2 * k + 1].y));
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        put(c % 2 * 4 + k, pack_bf16(f[4 * k].x, f[4 * k].y), pack_bf16(f[4 * k + 1].x, f[4 * k + 1].y), pack_bf16(f[4 * k + 2].x, f[4 * k + 2].y),
            pack_bf16(f[4 * k + 3].x, f[4 * k + 3].y));
    }
    if (last) {
      ptx::fence_proxy_async_smem();
      __syncwarp();
      const int n = n0 + (out_f32 ? c : c - 1) * 32;
      if (lane == 0 && n < N && row0 < M) tma_store_2d(tma_c, b, n, row0);
      ++filled;
    }
  }
}

template <int BN>
struct Cfg {
  static constexpr int kBytesA = BM * BK, kBytesB = BN * BK, kStageBytes = kBytesA + kBytesB;
  static constexpr int kStages = BN == 256 ? 4 : 6;                          // 192 KB
  static constexpr int kAcc = BN == 256 ? 2 : 4;                             // accumulators
  static constexpr int kTmemCols = kAcc * BN;
  static constexpr int kThreads = 384;
  static constexpr int kBufs = 1;                                            // 4 KB each, per epilogue warp
  static constexpr int kOffStaging = kStages * kStageBytes;
  static constexpr int kOffBar = kOffStaging + 8 * kBufs * 4096;
  static constexpr int kNumBars = 2 * kStages + 2 * kAcc;
  static constexpr int kSmemBytes = kOffBar + kNumBars * 8 + 16 + 1024;      // 1024: alignment by hand
  static_assert(kSmemBytes <= 232448, "shared memory per CTA");
};

struct Args {
  const float* a_scale;
  const float* w_scale;
  const int32_t* tile_group;        // nullptr: dense
  int64_t lds;
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
gemm_fp8_kernel(const __grid_constant__ CUtensorMap tma_a, const __grid_constant__ CUtensorMap tma_b, const __grid_constant__ CUtensorMap tma_c, const Args a) {
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
  // registers: the epilogue's two warpgroups hold up to 128 sums each thread, the first warpgroup next to nothing: 128 x 56 + 256 x 224 = 384 x 168
  if (warp < 4) asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
  if (warp == 0 && ptx::elect_one()) {
    uint32_t it = 0;
    for (int tile = blockIdx.x; tile < a.num_tiles; tile += gridDim.x) {
      const int grp = next;
      const int2 at = tile_at(tile, a);
      next = group_of(tile + gridDim.x);
      if (kGrouped && grp < 0) continue;
      for (int kb = 0; kb < a.num_kb; ++kb, ++it) {
        const int s = it % cfg::kStages;
        ptx::mbar_wait(empty_bar(s), ((it / cfg::kStages) & 1) ^ 1u);      // first lap: falls through
        ptx::mbar_arrive_expect_tx(full_bar(s), cfg::kStageBytes);
        const uint32_t dst = base + s * cfg::kStageBytes;
        ptx::tma_load_2d(dst + cfg::kBytesA, &tma_b, full_bar(s), kb * BK, grp * a.N + at.y * BN);
        ptx::tma_load_2d(dst, &tma_a, full_bar(s), kb * BK, at.x * BM);
      }
    }
  } else if (warp == 1 && ptx::elect_one()) {
    constexpr uint32_t idesc = idesc_fp8(BM, BN), desc_hi = ptx::umma_desc_hi_sw128(1024);
    const uint32_t a_lo0 = ptx::umma_desc_lo(base, 16);
    uint32_t it = 0;
    for (int tile = blockIdx.x; tile < a.num_tiles; tile += gridDim.x) {
      const int grp = next;
      next = group_of(tile + gridDim.x);
      if (kGrouped && grp < 0) continue;
      for (int kb = 0; kb < a.num_kb; ++kb, ++it) {
        const int s = it % cfg::kStages, acc = it % cfg::kAcc;
        ptx::mbar_wait(full_bar(s), (it / cfg::kStages) & 1);
        ptx::mbar_wait(acc_empty(acc), ((it / cfg::kAcc) & 1) ^ 1u);       // its last k-block has been read out
        ptx::tcgen05_fence_after();
        const uint32_t a_lo = a_lo0 + ((s * cfg::kStageBytes) >> 4), b_lo = a_lo + (cfg::kBytesA >> 4);
#pragma unroll
        for (int k = 0; k < BK / 32; ++k)          // 32 numbers are 32 bytes along K inside the 128-byte swizzle span: +2 in the address field
          umma_fp8_ss(tmem + acc * BN, ptx::umma_desc(a_lo + 2 * k, desc_hi), ptx::umma_desc(b_lo + 2 * k, desc_hi), idesc, k != 0 ? 1u : 0u);
        ptx::umma_commit(empty_bar(s));
        ptx::umma_commit(acc_full(acc));
      }
    }
  } else if (warp >= 4) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
    constexpr int kCols = BN / 2;                                          // this thread's columns
    const int quad = warp & 3, side = (warp - 4) >> 2;
    const uint32_t taddr = tmem + ((uint32_t)(quad * 32) << 16) + side * kCols;
    const int w_blocks = (a.N + kFp8Block - 1) / kFp8Block;
    const uint32_t buf = base + cfg::kOffStaging + (warp - 4) * cfg::kBufs * 4096;
    uint32_t it = 0, filled = 0;
    for (int tile = blockIdx.x; tile < a.num_tiles; tile += gridDim.x) {
      const int grp = next;
      const int2 at = tile_at(tile, a);
      next = group_of(tile + gridDim.x);
      if (kGrouped && grp < 0 && !a.zero) continue;
      const int row0 = at.x * BM + quad * 32, n0 = at.y * BN + side * kCols;
      float2 acc[kCols / 2];
#pragma unroll
      for (int j = 0; j < kCols / 2; ++j) acc[j] = make_float2(0.f, 0.f);
      if (!kGrouped || grp >= 0) {                                         // else rows that no group computes: zeros
        // rows and columns behind the last have the last one's scales, and are not stored
        const float* sa = a.a_scale + (int64_t)min(row0 + lane, a.M - 1) * a.lds;
        const float* sw = a.w_scale + ((int64_t)grp * w_blocks + min(n0 / kFp8Block, w_blocks - 1)) * a.num_kb;
        scaled_sums<kCols, cfg::kAcc, BN>(acc, sa, sw, a.num_kb, it, taddr, acc_full, [&](int i) {
          if (lane == 0) ptx::mbar_arrive(acc_empty(i));
        });
      }
      store_sums<kCols, cfg::kBufs>(&tma_c, buf, filled, lane, a.out_f32, row0, a.M, n0, a.N, acc);
    }
    if (lane == 0) bulk_wait_all();
  }
  __syncwarp();
  ptx::tcgen05_fence_before();
  __syncthreads();
  if (warp == 1) {
    ptx::tcgen05_fence_after();
    ptx::tmem_dealloc(tmem, cfg::kTmemCols);
  }
}

// Tiles of 256 x 256 on CTA pairs: each CTA brings 128 rows of A and 128 of W, the leader's tcgen05.mma.cta_group::2 read both CTAs' shared memory and write 128 rows into
// either's tensor memory.  A k-block brings 32 KB per SM where the 1-CTA tile brings 48 KB, for the same 512 cycles of the tensor pipe.
// Tensor memory holds two k-blocks of 256 columns; the way from the last product over commit, reads and release back to the next product takes longer than the other
// k-block's 512 cycles, so a k-block is two products of 128 columns, handed over by themselves: then 768 cycles lie in between.  The left half's columns 0 .. 63 come from
// the leader's rows of W, 64 .. 127 from the other's, and so on for the right.
// Each half has a warp of the leader's that issues it: a k-block's two waits, products and commits take one thread 600 to 800 cycles (handed over but never read, 581 us
// of 8 192 x 24 576 x 4 096 with one issuing warp, 382 with two, where the tensor pipe is full).
// Stages and accumulators are handed over by barriers of the leader - relaxed: a release at cluster scope waits for the warp's loads of scales, 2 000 cycles per
// k-block (1 454 us) - results by barriers of both.
struct PairCfg {
  static constexpr int kBytesA = BM * BK, kBytesB = 128 * BK, kStageBytes = kBytesA + kBytesB;
  static constexpr int kStages = 5, kBufs = 2;                               // 160 KB and 64 KB
  static constexpr int kSlots = 4;                                           // 128 columns each
  static constexpr int kThreads = 384;
  static constexpr int kOffStaging = kStages * kStageBytes;
  static constexpr int kOffBar = kOffStaging + 8 * kBufs * 4096;
  static constexpr int kNumBars = 2 * kStages + 2 * kSlots;
  static constexpr int kSmemBytes = kOffBar + kNumBars * 8 + 16 + 1024;
  static_assert(kSmemBytes <= 232448, "shared memory per CTA");
};

__global__ void __launch_bounds__(PairCfg::kThreads, 1)
gemm_fp8_pair_kernel(const __grid_constant__ CUtensorMap tma_a, const __grid_constant__ CUtensorMap tma_b, const __grid_constant__ CUtensorMap tma_c, const Args a) {
  using cfg = PairCfg;
  pdl_trigger();
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* gen = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t bar0 = base + cfg::kOffBar;
  auto full_bar = [&](int s) { return bar0 + 8u * s; };
  auto empty_bar = [&](int s) { return bar0 + 8u * (cfg::kStages + s); };
  auto acc_full = [&](int i) { return bar0 + 8u * (2 * cfg::kStages + i); };         // slot i: k-block i / 2 mod 2, half i & 1
  auto acc_empty = [&](int i) { return bar0 + 8u * (2 * cfg::kStages + cfg::kSlots + i); };
  const uint32_t tmem_slot = bar0 + 8u * cfg::kNumBars;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int h = (int)ptx::cluster_ctarank();
  const int cluster = blockIdx.x >> 1, clusters = gridDim.x >> 1;
  if (warp == 0) {
    if (lane == 0) {
      ptx::tma_prefetch_desc(&tma_a);
      ptx::tma_prefetch_desc(&tma_b);
      for (int s = 0; s < cfg::kStages; ++s) {
        ptx::mbar_init(full_bar(s), 1);          // the leader's expect_tx; the bytes of both CTAs complete there
        ptx::mbar_init(empty_bar(s), 2);         // two commits of the leader's, to both CTAs
      }
      for (int i = 0; i < cfg::kSlots; ++i) {
        ptx::mbar_init(acc_full(i), 1);          // the leader's commit, to both CTAs
        ptx::mbar_init(acc_empty(i), 8);         // four warps of either CTA, on the leader's
      }
      ptx::fence_barrier_init();
    }
    __syncwarp();
  } else if (warp == 1) {
    tmem_alloc_pair(tmem_slot, 512);
    tmem_relinquish_pair();
  }
  ptx::tcgen05_fence_before();
  __syncthreads();
  ptx::tcgen05_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(gen + cfg::kOffBar + cfg::kNumBars * 8);
  ptx::cluster_sync_all();                       // both CTAs' barriers exist before the other's copies and commits reach them
  pdl_wait();
  if (warp < 4) asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
  if (warp == 0 && ptx::elect_one()) {
    const uint32_t leader_full0 = ptx::mapa_u32(full_bar(0), 0);
    uint32_t it = 0;
    for (int tile = cluster; tile < a.num_tiles; tile += clusters) {
      const int2 at = tile_at(tile, a);
      for (int kb = 0; kb < a.num_kb; ++kb, ++it) {
        const int s = it % cfg::kStages;
        ptx::mbar_wait(empty_bar(s), ((it / cfg::kStages) & 1) ^ 1u);
        if (h == 0) ptx::mbar_arrive_expect_tx(full_bar(s), 2 * cfg::kStageBytes);
        const uint32_t dst = base + s * cfg::kStageBytes;
        tma_load_2d_pair(dst, &tma_a, leader_full0 + 8u * s, kb * BK, at.x * 2 * BM + h * BM);
        tma_load_2d_pair(dst + cfg::kBytesA, &tma_b, leader_full0 + 8u * s, kb * BK, at.y * 256 + h * 64);
        tma_load_2d_pair(dst + cfg::kBytesA + 64 * BK, &tma_b, leader_full0 + 8u * s, kb * BK, at.y * 256 + 128 + h * 64);
      }
    }
  } else if ((warp == 1 || warp == 2) && h == 0 && ptx::elect_one()) {
    constexpr uint32_t idesc = idesc_fp8(2 * BM, 128), desc_hi = ptx::umma_desc_hi_sw128(1024);
    const int half = warp - 1;
    const uint32_t a_lo0 = ptx::umma_desc_lo(base, 16), b_lo0 = ptx::umma_desc_lo(base + cfg::kBytesA + half * 64 * BK, 16);
    uint32_t it = 0;
    for (int tile = cluster; tile < a.num_tiles; tile += clusters) {
      for (int kb = 0; kb < a.num_kb; ++kb, ++it) {
        const uint32_t s = it % cfg::kStages, slot = (it & 1) * 2 + half, step = (s * cfg::kStageBytes) >> 4;
        ptx::mbar_wait(full_bar(s), (it / cfg::kStages) & 1);
        ptx::mbar_wait(acc_empty(slot), ((it >> 1) & 1) ^ 1u);
        ptx::tcgen05_fence_after();
#pragma unroll
        for (int k = 0; k < BK / 32; ++k)
          umma_fp8_ss_pair(tmem + slot * 128, ptx::umma_desc(a_lo0 + step + 2 * k, desc_hi), ptx::umma_desc(b_lo0 + step + 2 * k, desc_hi), idesc, k != 0 ? 1u : 0u);
        umma_commit_pair_mcast(acc_full(slot), 3);
        umma_commit_pair_mcast(empty_bar(s), 3);
      }
    }
  } else if (warp >= 4) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
    const int quad = warp & 3, side = (warp - 4) >> 2;
    const uint32_t taddr = tmem + ((uint32_t)(quad * 32) << 16) + side * 128;
    const uint32_t leader_empty0 = ptx::mapa_u32(acc_empty(0), 0);
    const int w_blocks = (a.N + kFp8Block - 1) / kFp8Block;
    const uint32_t buf = base + cfg::kOffStaging + (warp - 4) * cfg::kBufs * 4096;
    uint32_t it = 0, filled = 0;
    for (int tile = cluster; tile < a.num_tiles; tile += clusters) {
      const int2 at = tile_at(tile, a);
      const int row0 = at.x * 2 * BM + h * BM + quad * 32, n0 = at.y * 256 + side * 128;
      float2 acc[64];
#pragma unroll
      for (int j = 0; j < 64; ++j) acc[j] = make_float2(0.f, 0.f);
      scaled_sums<128, 2, 256>(acc, a.a_scale + (int64_t)min(row0 + lane, a.M - 1) * a.lds, a.w_scale + (int64_t)min(n0 / kFp8Block, w_blocks - 1) * a.num_kb, a.num_kb, it,
                               taddr, [&](int i) { return acc_full(2 * i + side); }, [&](int i) {
                                 if (lane == 0) mbar_arrive_cluster_relaxed(leader_empty0 + 8u * (2 * i + side));
                               });
      store_sums<128, cfg::kBufs>(&tma_c, buf, filled, lane, a.out_f32, row0, a.M, n0, a.N, acc);
    }
    if (lane == 0) bulk_wait_all();
  }
  __syncwarp();
  ptx::tcgen05_fence_before();
  __syncthreads();
  ptx::cluster_sync_all();                       // nobody leaves while the other may still signal its barriers
  if (warp == 1) {
    ptx::tcgen05_fence_after();
    tmem_dealloc_pair(tmem, 512);
  }
}

int make_map(nvc_ctx* ctx, CUtensorMap* map, const void* base, CUtensorMapDataType type, uint64_t inner, uint64_t rows, uint64_t row_bytes, uint32_t box_inner,
             uint32_t box_rows) {
  cuuint64_t gdim[2] = {inner, rows}, gstr[1] = {row_bytes};
  cuuint32_t box[2] = {box_inner, box_rows}, estr[2] = {1, 1};
  const CUresult r = ctx->encode_tiled(map, type, 2, const_cast<void*>(base), gdim, gstr, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                       CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r == CUDA_SUCCESS) return NVC_OK;
  nvc_set_error(ctx, "cuTensorMapEncodeTiled failed with CUresult " + std::to_string((int)r));
  return NVC_EINVAL;
}

// One call's operands
struct Call {
  const nvc_fp8* A;
  int lda;
  const nvc_fp8* W;
  void* C;
  int ldc, K, groups;
  cudaStream_t stream;
};

// The three maps of a call: boxes of 128 rows of A and b_rows of W, a block of 128 wide; 32 rows of 128 bytes of C
int make_maps(nvc_ctx* ctx, const Call& c, const Args& a, uint32_t b_rows, CUtensorMap* ta, CUtensorMap* tb, CUtensorMap* tc) {
  int rc = make_map(ctx, ta, c.A, CU_TENSOR_MAP_DATA_TYPE_UINT8, (uint64_t)c.K, (uint64_t)a.M, (uint64_t)c.lda, BK, BM);
  if (!rc) rc = make_map(ctx, tb, c.W, CU_TENSOR_MAP_DATA_TYPE_UINT8, (uint64_t)c.K, (uint64_t)a.N * c.groups, (uint64_t)c.K, BK, b_rows);
  const int size = a.out_f32 ? 4 : 2;
  if (!rc)
    rc = make_map(ctx, tc, c.C, a.out_f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, (uint64_t)a.N, (uint64_t)a.M, (uint64_t)c.ldc * size,
                  128 / size, 32);
  return rc;
}

template <int BN, bool kGrouped>
int launch(nvc_ctx* ctx, const Call& c, Args a) {
  CUtensorMap ta, tb, tc;
  const int rc = make_maps(ctx, c, a, BN, &ta, &tb, &tc);
  if (rc) return rc;
  a.n_tiles = (a.N + BN - 1) / BN;
  a.m_tiles = (a.M + BM - 1) / BM;
  const int64_t tiles = (int64_t)a.m_tiles * a.n_tiles;
  NVC_REQUIRE(ctx, tiles <= 0x7fffffffLL - ctx->num_sms, NVC_ESHAPE, "too many tiles");
  a.num_tiles = (int)tiles;
  const int grid = (int)(tiles < ctx->num_sms ? tiles : ctx->num_sms);
  NVC_CUDA_CHECK(ctx, nvc_launch(ctx, gemm_fp8_kernel<BN, kGrouped>, dim3(grid), dim3(Cfg<BN>::kThreads), Cfg<BN>::kSmemBytes, c.stream, ta, tb, tc, a));
  NVC_CUDA_CHECK(ctx, cudaGetLastError());
  ctx->launches++;
  return NVC_OK;
}

int launch_pair(nvc_ctx* ctx, const Call& c, Args a) {
  CUtensorMap ta, tb, tc;
  const int rc = make_maps(ctx, c, a, 64, &ta, &tb, &tc);
  if (rc) return rc;
  a.n_tiles = (a.N + 255) / 256;
  a.m_tiles = (a.M + 2 * BM - 1) / (2 * BM);
  const int64_t tiles = (int64_t)a.m_tiles * a.n_tiles;
  NVC_REQUIRE(ctx, tiles <= 0x7fffffffLL - ctx->num_sms, NVC_ESHAPE, "too many tiles");
  a.num_tiles = (int)tiles;
  const int avail = ctx->pair_clusters[1] > 0 ? ctx->pair_clusters[1] : ctx->num_sms / 2;
  const int waves = (int)((tiles + avail - 1) / avail), clusters = (int)((tiles + waves - 1) / waves);
  // column tiles fastest, every row of tiles streams all weights: weights that leave L2 no room are walked in bands of row tiles (gemm_pair.cu)
  if ((int64_t)a.N * c.K > (32 << 20)) {
    const int64_t most = (48 << 20) / ((int64_t)2 * BM * c.K);
    a.band = (int)(most < 1 ? 1 : (most > 16 ? 16 : most));
    a.band = (a.m_tiles + (a.m_tiles + a.band - 1) / a.band - 1) / ((a.m_tiles + a.band - 1) / a.band);
  }
  NVC_CUDA_CHECK(ctx, nvc_launch_cluster(ctx, gemm_fp8_pair_kernel, dim3(2 * clusters), dim3(PairCfg::kThreads), PairCfg::kSmemBytes, c.stream, 2, ta, tb, tc, a));
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
  X(256, false) X(128, false) X(256, true) X(128, true)
#undef X
  NVC_CUDA_CHECK(ctx, cudaFuncSetAttribute(gemm_fp8_pair_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, PairCfg::kSmemBytes));
  return NVC_OK;
}

extern "C" int nvc_gemm_fp8_ex(nvc_ctx* ctx, const nvc_fp8* A, int lda, const float* a_scale, int lds, const nvc_fp8* W, const float* w_scale, void* C, int ldc, int out_dtype,
                               int M, int Nout, int K, int force, void* stream) {
  int rc = nvc_gemm_fp8_check(ctx, A, lda, a_scale, lds, W, w_scale, C, ldc, out_dtype, M, Nout, K, 1);
  if (rc || M == 0) return rc;
  DeviceGuard guard(ctx->device);
  const Args a = {a_scale, w_scale, nullptr, lds, out_dtype == NVC_DT_F32, M, Nout, (K + BK - 1) / BK, 0, 0, 0, 1, 0};
  const Call c = {A, lda, W, C, ldc, K, 1, nvc_stream(stream)};
  const int64_t m_tiles = (M + BM - 1) / BM;
  if (force == 0) force = m_tiles * ((Nout + 255) / 256) <= ctx->num_sms ? 2 : 5;
  if (force == 2) return launch<128, false>(ctx, c, a);
  if (force == 3) return launch<256, false>(ctx, c, a);
  return launch_pair(ctx, c, a);
}

extern "C" int nvc_gemm_fp8(nvc_ctx* ctx, const nvc_fp8* A, int lda, const float* a_scale, int lds, const nvc_fp8* W, const float* w_scale, void* C, int ldc, int out_dtype,
                            int M, int Nout, int K, void* stream) {
  return nvc_gemm_fp8_ex(ctx, A, lda, a_scale, lds, W, w_scale, C, ldc, out_dtype, M, Nout, K, 0, stream);
}

extern "C" int nvc_gemm_fp8_grouped(nvc_ctx* ctx, const nvc_fp8* A, int lda, const float* a_scale, int lds, const nvc_fp8* W, const float* w_scale, void* C, int ldc,
                                    int out_dtype, int M_cap, int Nout, int K, const int32_t* tile_group, int groups, int zero, void* stream) {
  int rc = nvc_gemm_fp8_check(ctx, A, lda, a_scale, lds, W, w_scale, C, ldc, out_dtype, M_cap, Nout, K, groups);
  if (rc) return rc;
  NVC_REQUIRE(ctx, tile_group, NVC_EINVAL, "null pointer");
  NVC_REQUIRE(ctx, M_cap % BM == 0, NVC_EINVAL, "M_cap must be a multiple of 128");
  if (M_cap == 0) return NVC_OK;
  DeviceGuard guard(ctx->device);
  const Args a = {a_scale, w_scale, tile_group, lds, out_dtype == NVC_DT_F32, M_cap, Nout, (K + BK - 1) / BK, 0, 0, 0, 1, zero != 0};
  const Call c = {A, lda, W, C, ldc, K, groups, nvc_stream(stream)};
  const int64_t m_tiles = M_cap / BM;
  if (m_tiles * ((Nout + 255) / 256) <= ctx->num_sms) return launch<128, true>(ctx, c, a);
  return launch<256, true>(ctx, c, a);
}
