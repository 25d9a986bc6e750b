// Products of 8-bit rows and weights (fp8.cuh), dense and grouped by expert:
//   C[m, n] = sum over k-blocks b of a_scale[m, b] * w_scale[n / 128, b] * (sum over the block's k of A[m, k] * W[n, k]),  bf16 or fp32
// The inner sums run on the tensor cores (e4m3 products are exact in fp32) in an accumulator of their own per k-block; the outer sums, whose factors differ
// from block to block, in fp32 registers.
//
// What bounds them: the tensor pipe takes 512 cycles for a k-block of 128 x 256, the epilogue has to read and scale every k-block's sums in the same time, and the operands have to come
// from L2.  On CTA pairs (32 KB per k-block and SM) the epilogue holds them; tiles of one CTA are held by the operands' way (48 KB, and 32 for 128 x 128).  Numbers of zero, us, whole /
// nothing read and summed / a quarter of the tensor instructions besides: 4 096 x 4 096 x 4 096 on pairs 55.5 / 46.8 / 42.7, tiles of 256 columns 61.0 / 57.7 / 48.1, of 128 64.5 / 57.8 /
// 50.3; 72 blocks of rows by expert, 4 096 x 2 048, 75.2 / 69.6 / 60.5; 333 x 4 096 x 2 560 on tiles of 128 9.9 / 9.4 / 8.5.
// 8 192 x 24 576 x 4 096 bf16: 660 to 680 us in short runs (2.4 PFLOP/s), 792 after seconds of them, which the power cap holds at 1.35 GHz; numbers of zero, which need
// less power, 535 (3.1) and 595 at 1.77 GHz.  That is 790 to 805 cycles per k-block of a pair's 256 x 256.
//
// Three kernels, chosen by choose_route: gemm_fp8_kernel, gemm_fp8_pair_kernel for many tiles, gemm_fp8_split_kernel for few.  The first one, also that of the
// experts' products, walks tiles of 128 x BN with a persistent grid, one CTA per SM:
//   warp 0       TMA producer: 128 x 128 bytes of A and BN x 128 of W per k-block into a ring that runs on into the next tile
//   warps 1, 2   tcgen05.mma M 128, N BN, K 32, four per k-block, every other k-block each, into one of two (BN 256) or four accumulators in tensor memory
//   warps 4-11   two per quadrant of tensor memory, one for either half of the columns: accumulator times scales onto registers, rows through shared memory and TMA
#include "fp8.cuh"
#include "ptx_pair.cuh"
#include "internal.h"

#include <algorithm>
#include <cmath>

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

// (a0, a1) += (d0, d1) * (s0, s1), both in one instruction
__device__ __forceinline__ void fma2(float2& a, uint32_t d0, uint32_t d1, float s0, float s1) {
  asm volatile("{\n\t.reg .b64 x, y, z;\n\t"        // volatile: not in front of the wait for d0, d1
      "mov.b64 x, {%0, %1};\n\tmov.b64 y, {%2, %3};\n\tmov.b64 z, {%4, %5};\n\t"
      "fma.rn.f32x2 x, y, z, x;\n\t"
      "mov.b64 {%0, %1}, x;\n\t}"
      : "+f"(a.x), "+f"(a.y) : "r"(d0), "r"(d1), "f"(s0), "f"(s1));
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

// ptx::mbar_wait without its message: a call in the loop takes registers that hold sums otherwise (8 192 x 24 576 x 4 096 572 us with the message, 535 without)
__device__ __forceinline__ void wait_quietly(uint32_t bar, uint32_t parity) {
  uint32_t spins = 0;
  while (!ptx::mbar_try_wait(bar, parity))
    if (++spins > NVC_MBAR_SPIN_LIMIT) __trap();
}

// The epilogue's walk over k-blocks: accumulator it % kAcc of tensor memory (kStride columns each), kCols columns of it in reads of kRead.
// Two warps of a quarter of the SM share its 512 cycles per k-block of 128 x 256, of which the sums take 330 and the reads 256; one after the other in a warp they take longer
// than that.  So reads are under way two at a time, the next k-block's first ones between the sums of this one's last, and whether it is there is asked for ahead of time (a
// barrier's answer takes 100 to 200 cycles beside the tensor core's own reads of shared memory).  8 192 x 24 576 x 4 096, us, numbers of zero, which leave the power cap
// out: 640 with wait, reads and sums in order, 597 with the reads ahead, 555 with the question ahead, 535 without a call in the loop; without scales to fetch 487 (from a table that
// another warp fills they take 607), the tensor pipe alone, without sums, 383.
// step(kb): before the sums of a k-block; sum(c, v): adds read c; release(i): the accumulator has been read out.
template <int kCols, int kRead, int kAcc, int kStride, typename Full, typename Release, typename Step, typename Sum>
__device__ __forceinline__ void walk_sums(int num_kb, uint32_t& it, uint32_t taddr, Full full, Release release, Step step, Sum sum) {
  constexpr int kReads = kCols / kRead;
  static_assert(kReads == 1 || kReads == 2 || kReads == 4, "one, two or four reads");
  uint32_t v[2][kRead];
  uint32_t t = taddr + it % kAcc * kStride;
  auto read = [&](int c) {
    if constexpr (kRead == 16) ptx::tmem_ld_32x32b_x16(t + c * kRead, v[c & 1]);
    else ptx::tmem_ld_32x32b_x32(t + c * kRead, v[c & 1]);
  };
  wait_quietly(full(it % kAcc), (it / kAcc) & 1);
  ptx::tcgen05_fence_after();
  read(0);
  if (kReads > 1) read(1);
  for (int kb = 0; kb < num_kb; ++kb) {
    step(kb);
    const bool more = kb + 1 < num_kb;
    const uint32_t next_bar = full((it + 1) % kAcc), next_parity = ((it + 1) / kAcc) & 1;
    bool ready = false;
    if (kReads < 4) ready = mbar_test(next_bar, next_parity);
    ptx::tmem_ld_wait();
    if (kReads == 4) {
      sum(0, v[0]);
      read(2);
      sum(1, v[1]);
      read(3);
      ready = mbar_test(next_bar, next_parity);
      ptx::tmem_ld_wait();
    }
    ptx::tcgen05_fence_before();
    release(it % kAcc);
    ++it;
    if (kReads > 1) sum(kReads - 2, v[0]);
    else sum(0, v[0]);
    if (more) {
      if (!ready) wait_quietly(next_bar, next_parity);
      ptx::tcgen05_fence_after();
      t = taddr + it % kAcc * kStride;
      read(0);
    }
    if (kReads > 1) {
      sum(kReads - 1, v[1]);
      if (more) read(1);
    }
  }
}

// The sums of a thread that has one row of A: its scale times the weight block's
template <int kCols, int kAcc, int kStride, typename Full, typename Release>
__device__ __forceinline__ void scaled_sums(float2* acc, const float* sa, const float* sw, int num_kb, uint32_t& it, uint32_t taddr, Full full, Release release) {
  float next_a = sa[0], next_w = sw[0], s;
  walk_sums<kCols, 32, kAcc, kStride>(num_kb, it, taddr, full, release,
                                      [&](int kb) {
                                        s = next_a * next_w;
                                        if (kb + 1 < num_kb) {
                                          next_a = sa[kb + 1];
                                          next_w = sw[kb + 1];
                                        }
                                      },
                                      [&](int c, const uint32_t* v) {
#pragma unroll
                                        for (int j = 0; j < 16; ++j) fma2(acc[c * 16 + j], v[2 * j], v[2 * j + 1], s, s);
                                      });
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
    const int n = n0 + (out_f32 ? c : c & ~1) * 32;
    if (n >= N || row0 >= M) continue;           // not written to a buffer either: the wait counts copies, and there is none for these
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
      if (lane == 0) tma_store_2d(tma_c, b, n, row0);
      ++filled;
    }
  }
}

// In front of the launch wait: the ring's first lap of weights into L2, where a later write still finds them.  They are read behind the wait, whoever wrote them: a kernel that does
// not signal its dependents early lets them start when its last CTA has ended, which orders nothing that it wrote.  Behind a norm, read ahead / asked for ahead / neither, us:
// 64 x 24 576 x 4 096 25.2 / 25.5 / 26.7, 200 x 12 288 x 1 024 10.9 / 11.1 / 11.7, 8 x 4 096 x 4 096 8.3 / 9.0; two laps and more 0.1 to 2 us longer.
__device__ __forceinline__ void ask_for_weights(const CUtensorMap* w, int kb0, int n, int row) {
  for (int kb = kb0; kb < kb0 + n; ++kb) ptx::tma_prefetch_l2_2d(w, kb * BK, row);
}

template <int BN>
struct Cfg {
  static constexpr int kBytesA = BM * BK, kBytesB = BN * BK, kStageBytes = kBytesA + kBytesB;
  static constexpr int kStages = BN == 256 ? 4 : 6;                          // 192 KB
  static constexpr int kAcc = BN == 256 ? 2 : 4;                             // accumulators
  static constexpr int kTmemCols = kAcc * BN;
  static constexpr int kThreads = 384;
  // a k-block's operands are asked for ahead by the warp that issues it: an answer is only unmistakable where it is the same warp that waited for the stage's last use
  static_assert(kStages % 2 == 0 && kAcc % 2 == 0, "two issuing warps");
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
  int out_f32, M, N, num_kb, num_tiles, n_tiles, m_tiles, band, zero, groups, a_box;       // a_box: rows of A that a copy brings, 128 or, of fewer, those that exist
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
      if (!kGrouped) ask_for_weights(&tma_b, 0, min(a.num_kb, cfg::kStages), tile_at(blockIdx.x, a).y * BN);
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
  auto group_of = [&](int tile) {
    if (!kGrouped) return 0;
    const int grp = tile < a.num_tiles ? __ldcg(a.tile_group + tile / a.n_tiles) : -1;
    return grp < a.groups ? grp : -1;
  };
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
        const uint32_t dst = base + s * cfg::kStageBytes;
        wait_quietly(empty_bar(s), ((it / cfg::kStages) & 1) ^ 1u);        // first lap: falls through
        ptx::mbar_arrive_expect_tx(full_bar(s), cfg::kBytesB + a.a_box * BK);          // rows of A behind the box hold what they held: their sums are never stored
        ptx::tma_load_2d(dst + cfg::kBytesA, &tma_b, full_bar(s), kb * BK, grp * a.N + at.y * BN);
        ptx::tma_load_2d(dst, &tma_a, full_bar(s), kb * BK, at.x * BM);
      }
    }
  } else if ((warp == 1 || warp == 2) && ptx::elect_one()) {
    constexpr uint32_t idesc = idesc_fp8(BM, BN), desc_hi = ptx::umma_desc_hi_sw128(1024);
    const uint32_t a_lo0 = ptx::umma_desc_lo(base, 16);
    uint32_t it = 0;
    bool here = false, free = false;             // what was asked ahead: the operands, the accumulator of this thread's next k-block
    for (int tile = blockIdx.x; tile < a.num_tiles; tile += gridDim.x) {
      const int grp = next;
      next = group_of(tile + gridDim.x);
      if (kGrouped && grp < 0) continue;
      for (int kb = 0; kb < a.num_kb; ++kb, ++it) {
        if ((it & 1) != (uint32_t)(warp - 1)) continue;
        const uint32_t s = it % cfg::kStages, acc = it % cfg::kAcc;
        if (!here) wait_quietly(full_bar(s), (it / cfg::kStages) & 1);
        if (!free) wait_quietly(acc_empty(acc), ((it / cfg::kAcc) & 1) ^ 1u);      // its last k-block has been read out
        here = mbar_test(full_bar((it + 2) % cfg::kStages), ((it + 2) / cfg::kStages) & 1);
        free = mbar_test(acc_empty((it + 2) % cfg::kAcc), (((it + 2) / cfg::kAcc) & 1) ^ 1u);
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
  const uint32_t leader_full0 = ptx::mapa_u32(full_bar(0), 0);
  if (warp == 0 && ptx::elect_one()) {
    const int n0 = tile_at(cluster, a).y * 256 + h * 64, n = min(a.num_kb, cfg::kStages);
    ask_for_weights(&tma_b, 0, n, n0);
    ask_for_weights(&tma_b, 0, n, n0 + 128);
  }
  __syncwarp();
  pdl_wait();
  if (warp < 4) asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
  if (warp == 0 && ptx::elect_one()) {
    uint32_t it = 0;
    for (int tile = cluster; tile < a.num_tiles; tile += clusters) {
      const int2 at = tile_at(tile, a);
      for (int kb = 0; kb < a.num_kb; ++kb, ++it) {
        const int s = it % cfg::kStages;
        const uint32_t dst = base + s * cfg::kStageBytes;
        wait_quietly(empty_bar(s), ((it / cfg::kStages) & 1) ^ 1u);
        if (h == 0) ptx::mbar_arrive_expect_tx(full_bar(s), 2 * cfg::kStageBytes);
        tma_load_2d_pair(dst + cfg::kBytesA, &tma_b, leader_full0 + 8u * s, kb * BK, at.y * 256 + h * 64);
        tma_load_2d_pair(dst + cfg::kBytesA + 64 * BK, &tma_b, leader_full0 + 8u * s, kb * BK, at.y * 256 + 128 + h * 64);
        tma_load_2d_pair(dst, &tma_a, leader_full0 + 8u * s, kb * BK, at.x * 2 * BM + h * BM);
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
        wait_quietly(full_bar(s), (it / cfg::kStages) & 1);
        wait_quietly(acc_empty(slot), ((it >> 1) & 1) ^ 1u);
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

// Few tiles: a cluster of S CTAs shares the k-blocks of one.  Every CTA parks its sums in its idle ring, row by row of A, 128 columns each, and adds up its share of the
// rows over the cluster, in the order of the ranks.
//   warp 0         TMA: 128 rows of W and up to NT of A per k-block
//   warp 1 (and 2) tcgen05.mma; the other warps sums
// NT 16, 32 (few rows): the operands change places - 128 rows of W are the rows of the product, the rows of A its columns, so that no part of the tensor pipe's and the
// epilogue's work is done for rows that do not exist.  A thread has a row of W and every row of A; the scales' products lie in a table, filled 32 k-blocks at a time.  The ring
// is half an SM's shared memory: two CTAs share an SM, and the next product starts while this one ends.
// NT 128: 128 rows of A and 128 columns; a thread has one row, and one scale for all its columns (with the operands changed, reading 64 scales per k-block from
// shared memory took 1 200 cycles, this 600).
template <int NT>
struct SplitCfg {
  static constexpr bool kSwap = NT < 128;
  static constexpr int kBytesW = 128 * BK, kBytesA = NT * BK, kStageBytes = kBytesW + kBytesA;
  static constexpr int kStages = kSwap ? 5 : 6;                              // 90 to 100 KB, or 192
  static constexpr int kAcc = 4;
  static constexpr int kTmemCols = kAcc * NT;
  static constexpr int kIssuers = kSwap ? 1 : 2, kFirst = kSwap ? 2 : 4;     // warps that issue products, the first one that sums
  static_assert(kStages % kIssuers == 0 && kAcc % kIssuers == 0, "as in Cfg");
  static constexpr int kSides = kSwap ? 1 : 2, kCols = NT / kSides, kRead = NT == 32 ? 32 : 16;
  static constexpr int kSumThreads = 128 * kSides, kThreads = 32 * kFirst + kSumThreads;
  static constexpr int kTableKb = 32, kPitch = NT + 4;                       // the table: k-blocks, floats per k-block
  static constexpr int kOffTable = kStages * kStageBytes;
  static constexpr int kOffBar = kOffTable + (kSwap ? kTableKb * kPitch * 4 : 0);
  static constexpr int kNumBars = 2 * kStages + 2 * kAcc;
  static constexpr int kSmemBytes = kOffBar + kNumBars * 8 + 16 + 1024;
  static_assert((kSwap ? 2 : 1) * (kSmemBytes + 1024) <= 233472, "CTAs per SM");
  static_assert(NT * 512 <= kStages * kStageBytes, "the sums fit the ring");
  // where row j of A has columns 4 c .. 4 c + 3: neighbouring threads write neighbouring columns of a row, or the same columns of neighbouring rows
  __device__ static uint32_t parked(int j, int c) { return (uint32_t)(j * 512 + ((kSwap ? c : c ^ (j & 31)) << 4)); }
};

template <int NT>
__global__ void __launch_bounds__(SplitCfg<NT>::kThreads, SplitCfg<NT>::kSwap ? 2 : 1)
gemm_fp8_split_kernel(const __grid_constant__ CUtensorMap tma_a, const __grid_constant__ CUtensorMap tma_w, void* __restrict__ C, int64_t ldc, int kb_per_split,
                      const Args a) {
  using cfg = SplitCfg<NT>;
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
  const int n0 = blockIdx.x * 128, m0 = blockIdx.y * NT, rank = blockIdx.z, S = gridDim.z;
  const int kb0 = rank * kb_per_split, num_kb = min(kb_per_split, a.num_kb - kb0);
  const uint32_t stage_tx = cfg::kBytesW + a.a_box * BK;                  // rows of A behind the box hold what they held: their sums are never stored
  if (warp == 0) {
    if (lane == 0) {
      ptx::tma_prefetch_desc(&tma_a);
      ptx::tma_prefetch_desc(&tma_w);
      for (int s = 0; s < cfg::kStages; ++s) {
        ptx::mbar_init(full_bar(s), 1);
        ptx::mbar_init(empty_bar(s), 1);
      }
      for (int i = 0; i < cfg::kAcc; ++i) {
        ptx::mbar_init(acc_full(i), 1);
        ptx::mbar_init(acc_empty(i), 4 * cfg::kSides);
      }
      ptx::fence_barrier_init();
      ask_for_weights(&tma_w, kb0, min(num_kb, cfg::kStages), n0);
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
  if (warp == 0 && ptx::elect_one()) {
    for (int kb = 0; kb < num_kb; ++kb) {
      const int s = kb % cfg::kStages;
      const uint32_t dst = base + s * cfg::kStageBytes;
      wait_quietly(empty_bar(s), ((kb / cfg::kStages) & 1) ^ 1u);
      ptx::mbar_arrive_expect_tx(full_bar(s), stage_tx);
      ptx::tma_load_2d(dst, &tma_w, full_bar(s), (kb0 + kb) * BK, n0);
      ptx::tma_load_2d(dst + cfg::kBytesW, &tma_a, full_bar(s), (kb0 + kb) * BK, m0);
    }
  } else if (warp >= 1 && warp <= cfg::kIssuers && ptx::elect_one()) {
    constexpr uint32_t idesc = idesc_fp8(128, NT), desc_hi = ptx::umma_desc_hi_sw128(1024);
    const uint32_t w_lo0 = ptx::umma_desc_lo(base, 16);
    bool here = false, free = false;             // what was asked ahead: the operands, the accumulator of this thread's next k-block
    for (uint32_t kb = warp - 1; kb < (uint32_t)num_kb; kb += cfg::kIssuers) {
      const uint32_t s = kb % cfg::kStages, i = kb % cfg::kAcc, next = kb + cfg::kIssuers;
      if (!here) wait_quietly(full_bar(s), (kb / cfg::kStages) & 1);
      if (!free) wait_quietly(acc_empty(i), ((kb / cfg::kAcc) & 1) ^ 1u);
      here = mbar_test(full_bar(next % cfg::kStages), (next / cfg::kStages) & 1);
      free = mbar_test(acc_empty(next % cfg::kAcc), ((next / cfg::kAcc) & 1) ^ 1u);
      ptx::tcgen05_fence_after();
      const uint32_t w_lo = w_lo0 + ((s * cfg::kStageBytes) >> 4), a_lo = w_lo + (cfg::kBytesW >> 4);
      const uint32_t rows_lo = cfg::kSwap ? w_lo : a_lo, cols_lo = cfg::kSwap ? a_lo : w_lo;
#pragma unroll
      for (int k = 0; k < BK / 32; ++k)
        umma_fp8_ss(tmem + i * NT, ptx::umma_desc(rows_lo + 2 * k, desc_hi), ptx::umma_desc(cols_lo + 2 * k, desc_hi), idesc, k != 0 ? 1u : 0u);
      ptx::umma_commit(empty_bar(s));
      ptx::umma_commit(acc_full(i));
    }
  }
  __syncwarp();
  if (warp >= cfg::kFirst) {
    const int quad = warp & 3, side = (warp - cfg::kFirst) >> 2, et = threadIdx.x - 32 * cfg::kFirst;
    const uint32_t taddr = tmem + ((uint32_t)(quad * 32) << 16) + side * cfg::kCols;
    const float* sw = a.w_scale + (int64_t)blockIdx.x * a.num_kb + kb0;
    auto release = [&](int i) {
      if (lane == 0) ptx::mbar_arrive(acc_empty(i));
    };
    float2 acc[cfg::kCols / 2];
#pragma unroll
    for (int j = 0; j < cfg::kCols / 2; ++j) acc[j] = make_float2(0.f, 0.f);
    uint32_t it = 0;
    if constexpr (cfg::kSwap) {
      float* table = reinterpret_cast<float*>(gen + cfg::kOffTable);
      for (int kt = 0; kt < num_kb; kt += cfg::kTableKb) {
        // neighbouring threads take neighbouring k-blocks of a row; rows behind the last count for nothing
        if (kt) ptx::named_bar_sync(1, cfg::kSumThreads);
        constexpr int kRowsPerPass = cfg::kSumThreads / cfg::kTableKb, kPasses = NT / kRowsPerPass;
        const int tb = et % cfg::kTableKb, tj = et / cfg::kTableKb;
        if (kt + tb < num_kb) {
          const float w = sw[kt + tb];
          const float* src = a.a_scale + (int64_t)m0 * a.lds + kb0 + kt + tb;
          float t[kPasses];
#pragma unroll
          for (int i = 0; i < kPasses; ++i) {
            const int j = tj + i * kRowsPerPass;
            t[i] = m0 + j < a.M ? src[(int64_t)j * a.lds] : 0.f;
          }
#pragma unroll
          for (int i = 0; i < kPasses; ++i) table[tb * cfg::kPitch + tj + i * kRowsPerPass] = t[i] * w;
        }
        ptx::named_bar_sync(1, cfg::kSumThreads);
        // a read's scales are fetched ahead of the sums of the read in front
        constexpr int kReads = cfg::kCols / cfg::kRead;
        float4 f[2][cfg::kRead / 4];
        const float4* p = nullptr;
        auto fetch = [&](int c) {
#pragma unroll
          for (int j = 0; j < cfg::kRead / 4; ++j) f[c & 1][j] = p[c * (cfg::kRead / 4) + j];
        };
        walk_sums<cfg::kCols, cfg::kRead, cfg::kAcc, NT>(min(cfg::kTableKb, num_kb - kt), it, taddr, acc_full, release,
                                                         [&](int b) {
                                                           p = reinterpret_cast<const float4*>(table + b * cfg::kPitch);
                                                           fetch(0);
                                                         },
                                                         [&](int c, const uint32_t* v) {
                                                           if (c + 1 < kReads) fetch(c + 1);
#pragma unroll
                                                           for (int j = 0; j < cfg::kRead / 4; ++j) {
                                                             const float4 g = f[c & 1][j];
                                                             fma2(acc[c * (cfg::kRead / 2) + 2 * j], v[4 * j], v[4 * j + 1], g.x, g.y);
                                                             fma2(acc[c * (cfg::kRead / 2) + 2 * j + 1], v[4 * j + 2], v[4 * j + 3], g.z, g.w);
                                                           }
                                                         });
      }
    } else {
      scaled_sums<cfg::kCols, cfg::kAcc, NT>(acc, a.a_scale + (int64_t)min(m0 + quad * 32 + lane, a.M - 1) * a.lds + kb0, sw, num_kb, it, taddr, acc_full, release);
    }
    // all products of this CTA are done: nothing reads or fills the ring any more
    ptx::fence_proxy_async_smem();
    if constexpr (cfg::kSwap) {
      float* park = reinterpret_cast<float*>(gen) + quad * 32 + lane;
#pragma unroll
      for (int j = 0; j < cfg::kCols / 2; ++j) {
        park[(2 * j) * 128] = acc[j].x;
        park[(2 * j + 1) * 128] = acc[j].y;
      }
    } else {
#pragma unroll
      for (int c = 0; c < cfg::kCols / 4; ++c)
        ptx::st_shared_f4(base + cfg::parked(quad * 32 + lane, side * (cfg::kCols / 4) + c), acc[2 * c].x, acc[2 * c].y, acc[2 * c + 1].x, acc[2 * c + 1].y);
    }
  }
  if (S > 1) ptx::cluster_sync_all();
  else __syncthreads();
  if (warp >= cfg::kFirst) {
    constexpr int kR = 2, kWarps = 4 * cfg::kSides;          // rows under way at a time: a read of another CTA's shared memory takes a while
    const int rows = min(NT, a.M - m0), n = n0 + lane * 4;
    for (int j0 = rank + S * (warp - cfg::kFirst); j0 < rows; j0 += kWarps * kR * S) {
      float4 t[kR][8];
#pragma unroll
      for (int r = 0; r < kR; ++r) {
        const int j = j0 + kWarps * r * S;
        const uint32_t mine = base + cfg::parked(j, lane);
#pragma unroll
        for (int z = 0; z < 8; ++z)
          if (z < S && j < rows) t[r][z] = ptx::ld_cluster_f4(S == 1 ? mine : ptx::mapa_u32(mine, (uint32_t)z));
      }
#pragma unroll
      for (int r = 0; r < kR; ++r) {
        const int j = j0 + kWarps * r * S;
        float4 sum = t[r][0];
#pragma unroll
        for (int z = 1; z < 8; ++z)
          if (z < S) { sum.x += t[r][z].x; sum.y += t[r][z].y; sum.z += t[r][z].z; sum.w += t[r][z].w; }
        if (j < rows && n < a.N) {
          const int64_t at = (int64_t)(m0 + j) * ldc + n;
          if (a.out_f32) *reinterpret_cast<float4*>(static_cast<float*>(C) + at) = sum;
          else *reinterpret_cast<uint2*>(static_cast<nvc_bf16*>(C) + at) = make_uint2(pack_bf16(sum.x, sum.y), pack_bf16(sum.z, sum.w));
        }
      }
    }
  }
  __syncwarp();
  ptx::tcgen05_fence_before();
  __syncthreads();
  if (S > 1) ptx::cluster_sync_all();            // nobody leaves while another may still read its sums
  if (warp == 1) {
    ptx::tcgen05_fence_after();
    ptx::tmem_dealloc(tmem, cfg::kTmemCols);
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

// The three maps of a call: boxes of a_box rows of A and b_rows of W, a block of 128 wide; 32 rows of 128 bytes of C
int make_maps(nvc_ctx* ctx, const Call& c, const Args& a, uint32_t b_rows, CUtensorMap* ta, CUtensorMap* tb, CUtensorMap* tc) {
  int rc = make_map(ctx, ta, c.A, CU_TENSOR_MAP_DATA_TYPE_UINT8, (uint64_t)c.K, (uint64_t)a.M, (uint64_t)c.lda, BK, a.a_box);
  if (!rc) rc = make_map(ctx, tb, c.W, CU_TENSOR_MAP_DATA_TYPE_UINT8, (uint64_t)c.K, (uint64_t)a.N * c.groups, (uint64_t)c.K, BK, b_rows);
  const int size = a.out_f32 ? 4 : 2;
  if (!rc)
    rc = make_map(ctx, tc, c.C, a.out_f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, (uint64_t)a.N, (uint64_t)a.M, (uint64_t)c.ldc * size,
                  128 / size, 32);
  return rc;
}

// The rows of A that a copy brings: as many as there are, in whole atoms of eight, and no more than `most`
int box_rows(int M, int most) { return M >= most ? most : (M + 7) / 8 * 8; }

template <int BN, bool kGrouped>
int launch(nvc_ctx* ctx, const Call& c, Args a) {
  CUtensorMap ta, tb, tc;
  a.a_box = box_rows(a.M, BM);
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
  a.a_box = BM;
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

template <int NT>
int launch_split(nvc_ctx* ctx, const Call& c, Args a, int S) {
  CUtensorMap ta, tw;
  a.a_box = box_rows(a.M, NT);
  int rc = make_map(ctx, &ta, c.A, CU_TENSOR_MAP_DATA_TYPE_UINT8, (uint64_t)c.K, (uint64_t)a.M, (uint64_t)c.lda, BK, a.a_box);
  if (!rc) rc = make_map(ctx, &tw, c.W, CU_TENSOR_MAP_DATA_TYPE_UINT8, (uint64_t)c.K, (uint64_t)a.N, (uint64_t)c.K, BK, 128);
  if (rc) return rc;
  const int m_tiles = (a.M + NT - 1) / NT, kb_per = (a.num_kb + S - 1) / S;
  NVC_REQUIRE(ctx, m_tiles <= 65535, NVC_ESHAPE, "too many tiles");
  S = (a.num_kb + kb_per - 1) / kb_per;          // no empty shares
  NVC_CUDA_CHECK(ctx, nvc_launch_cluster3(ctx, gemm_fp8_split_kernel<NT>, dim3((a.N + 127) / 128, m_tiles, S), dim3(SplitCfg<NT>::kThreads), SplitCfg<NT>::kSmemBytes, c.stream,
                                          dim3(1, 1, S), ta, tw, c.C, (int64_t)c.ldc, kb_per, a));
  NVC_CUDA_CHECK(ctx, cudaGetLastError());
  ctx->launches++;
  return NVC_OK;
}

// What both products ask of their arguments.
int nvc_gemm_fp8_check(nvc_ctx* ctx, const nvc_fp8* A, int lda, const float* a_scale, int lds, const nvc_fp8* W, const float* w_scale, void* C, int ldc, int out_dtype, int M, int Nout,
          int K, int groups) {
  NVC_REQUIRE(ctx, ctx && A && a_scale && W && w_scale && C, NVC_EINVAL, "null pointer");
  NVC_REQUIRE(ctx, M >= 0 && Nout > 0 && K > 0 && groups > 0, NVC_EINVAL, "bad sizes");
  // row and column numbers of the last tiles
  NVC_REQUIRE(ctx, (int64_t)Nout * groups <= 0x7fffffff - 2 * BM && M <= 0x7fffffff - 2 * BM && K <= 0x7fffffff - BK, NVC_ESHAPE, "too many rows or too wide");
  NVC_REQUIRE(ctx, K % 16 == 0 && Nout % 16 == 0, NVC_ESHAPE, "K and Nout must be multiples of 16");
  NVC_REQUIRE(ctx, lda % 16 == 0 && lda >= K && ldc % 8 == 0 && ldc >= Nout && lds >= (K + BK - 1) / BK, NVC_ESHAPE,
              "row strides must cover the rows, A's be a multiple of 16 and C's of 8");
  NVC_REQUIRE(ctx, out_dtype == NVC_DT_BF16 || out_dtype == NVC_DT_F32, NVC_EINVAL, "bad out_dtype");
  NVC_REQUIRE(ctx, ((uintptr_t)A % 16) == 0 && ((uintptr_t)W % 16) == 0 && ((uintptr_t)C % 16) == 0, NVC_EINVAL, "pointers must be 16-byte aligned");
  NVC_REQUIRE(ctx, ctx->encode_tiled != nullptr, NVC_EDEVICE, "cuTensorMapEncodeTiled unavailable");
  return NVC_OK;
}

// The kernels of a dense product, and over how many CTAs a tile's k-blocks are shared.
enum { kFew16 = 1, kFew32, kShared, kRows128, kRows256, kPair };
struct Route {
  int tile, S;
};

// The kernel with the least time by a model of waves and k-blocks (us): a start, w waves, k-blocks per wave (those of a full chip take longer), the weights' way from
// memory where a wave does not show it, the sums' way over the cluster.  Fitted to 3 229 timings of 301 products (17 weights of 0.4 to 100 MB, 1 to 4 096 rows): 6 to 10 % off
// in the mean; its choice is 1.4 % above the best of all kernels and shares in the mean, at most 21 % (profiles/fp8_product_routes.txt).  No one kernel does it all: 64 x 1 024 x 2 048
// 4.4 us on kFew32 with five shares, 6.4 on kRows128, 9.0 on kPair; 256 x 4 096 x 4 096 11.1 on kShared with two, 12.4, 16.7; 512 x 24 576 x 4 096 49.6 on kPair, 69.7 on kRows128.
Route choose_route(const nvc_ctx* ctx, int M, int N, int num_kb) {
  const double mb = (double)N * num_kb * BK * 1e-6;
  auto tiles = [&](int rows, int cols) { return (double)((M + rows - 1) / rows) * ((N + cols - 1) / cols); };
  Route best = {kPair, 1};
  double least = 1e30;
  auto offer = [&](int tile, int S, double t) {
    if (t < least) { least = t; best = {tile, S}; }
  };
  auto walk = [&](int tile, double n, double places, double start, double wave, double kb, double full, double weights) {
    const double w = std::ceil(n / places);
    offer(tile, 1, start + w * (wave + num_kb * (kb + full * std::min(n / places, 1.0))) + weights * mb);
  };
  const double sms = ctx->num_sms, pairs = ctx->pair_clusters[1] > 0 ? ctx->pair_clusters[1] : ctx->num_sms / 2;
  walk(kPair, tiles(256, 256), pairs, 3.36, 0.95, 0.357, 0.110, 0.0);
  walk(kRows256, tiles(128, 256), sms, 2.71, 1.31, 0.372, 0.104, 0.0438);
  walk(kRows128, tiles(128, 128), sms, 2.48, 0.61, 0.240, 0.053, 0.0335);
  for (int S = 1; S <= 8 && S <= num_kb; ++S) {
    const int kbs = (num_kb + S - 1) / S;
    if ((num_kb + kbs - 1) / kbs != S) continue;                           // the same shares as with fewer
    const double one = ctx->fp8_clusters[S] > 0 ? ctx->fp8_clusters[S] : ctx->num_sms / S, two = 2 * one, many = S > 1;
    auto share = [&](int tile, int rows, double places, double start, double wave, double kb, double full, double weights, double join, double row) {
      const double n = tiles(rows, 128), w = std::ceil(n / places);
      if (w > 2 && S > 1) return;                                          // not measured
      offer(tile, S, start + w * (wave + kbs * (kb + full * std::min(n / places, 1.0)) + row * std::min(M, rows)) + weights * mb + join * many);
    };
    if (M <= 16) share(kFew16, 16, two, 1.45, 0.76, 0.184, 0.0, 0.119, 0.57, 0.0105);
    if (M > 16 && M <= 96) share(kFew32, 32, two, 2.38, 0.0, 0.201, 0.116, 0.096, 0.0, 0.036);
    if (M <= 1100) share(kShared, 128, one, 2.57, 0.07, 0.197, 0.166, 0.0535, 0.37, 0.0166);
  }
  return best;
}

}  // namespace

extern "C" int nvc_gemm_fp8_init(nvc_ctx* ctx) {
#define X(BN, G) NVC_CUDA_CHECK(ctx, (cudaFuncSetAttribute(gemm_fp8_kernel<BN, G>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<BN>::kSmemBytes)));
  X(256, false) X(128, false) X(256, true) X(128, true)
#undef X
  // all of an SM's 228 KB to shared memory: two CTAs of half of it fit
#define X(NT) \
  NVC_CUDA_CHECK(ctx, cudaFuncSetAttribute(gemm_fp8_split_kernel<NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, SplitCfg<NT>::kSmemBytes)); \
  NVC_CUDA_CHECK(ctx, cudaFuncSetAttribute(gemm_fp8_split_kernel<NT>, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared));
  X(16) X(32) X(128)
#undef X
  for (int S = 1; S <= 8; ++S) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(64, 1, S);
    cfg.blockDim = dim3(SplitCfg<128>::kThreads);
    cfg.dynamicSmemBytes = SplitCfg<128>::kSmemBytes;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = S;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, gemm_fp8_split_kernel<128>, &cfg) != cudaSuccess || n <= 0) {
      (void)cudaGetLastError();
      n = ctx->num_sms / S;
    }
    ctx->fp8_clusters[S] = n;
  }
  NVC_CUDA_CHECK(ctx, cudaFuncSetAttribute(gemm_fp8_pair_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, PairCfg::kSmemBytes));
  return NVC_OK;
}

extern "C" int nvc_gemm_fp8_ex(nvc_ctx* ctx, const nvc_fp8* A, int lda, const float* a_scale, int lds, const nvc_fp8* W, const float* w_scale, void* C, int ldc, int out_dtype,
                               int M, int Nout, int K, int force, void* stream) {
  int rc = nvc_gemm_fp8_check(ctx, A, lda, a_scale, lds, W, w_scale, C, ldc, out_dtype, M, Nout, K, 1);
  if (rc || M == 0) return rc;
  NVC_REQUIRE(ctx, force == 0 || (force / 10 >= kFew16 && force / 10 <= kPair && force % 10 >= 1 && force % 10 <= 8), NVC_EINVAL, "bad route");
  DeviceGuard guard(ctx->device);
  const Args a = {a_scale, w_scale, nullptr, lds, out_dtype == NVC_DT_F32, M, Nout, (K + BK - 1) / BK, 0, 0, 0, 1, 0, 1, BM};
  const Call c = {A, lda, W, C, ldc, K, 1, nvc_stream(stream)};
  const Route r = force ? Route{force / 10, force % 10} : choose_route(ctx, M, Nout, a.num_kb);
  switch (r.tile) {
    case kFew16: return launch_split<16>(ctx, c, a, r.S);
    case kFew32: return launch_split<32>(ctx, c, a, r.S);
    case kShared: return launch_split<128>(ctx, c, a, r.S);
    case kRows128: return launch<128, false>(ctx, c, a);
    case kRows256: return launch<256, false>(ctx, c, a);
    default: return launch_pair(ctx, c, a);
  }
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
  const Args a = {a_scale, w_scale, tile_group, lds, out_dtype == NVC_DT_F32, M_cap, Nout, (K + BK - 1) / BK, 0, 0, 0, 1, zero != 0, groups, BM};
  const Call c = {A, lda, W, C, ldc, K, groups, nvc_stream(stream)};
  // The times of choose_route over the tiles that there may be: M_cap holds the rows, groups x 127 of padding and up to 127 of rounding; a group of up to 112 rows fills one
  // tile, a larger one half a tile more than its rows.  128 columns where they promise no more than 6 % above 256, since routers leave some groups empty, and fewer wide tiles
  // leave SMs idle (us, 128 / 256: 64 tokens, 24 groups, 10 of them used, 1 536 x 2 048 12.8 / 15.1; 600, 8 groups, 4 096 x 1 024 15.2 / 16.3; 2 500, 16 groups, 2 048 x 2 048
  // 21.8 / 23.6; 8 000, 16 groups, 4 096 x 2 048 89.7 / 83.5)
  const double rows = std::max((double)M_cap - 127.0 * groups - 64.0, 1.0), per = rows / groups;
  const double m_tiles = groups * (per <= 112.0 ? std::min(per, 1.0) : per / BM + 0.5), mb = std::min(rows, (double)groups) * Nout * K * 1e-6;
  auto time = [&](int cols, double start, double wave, double kb, double full, double weights) {
    const double n = m_tiles * ((Nout + cols - 1) / cols) / ctx->num_sms;
    return start + std::ceil(n) * (wave + a.num_kb * (kb + full * std::min(n, 1.0))) + weights * mb;
  };
  if (time(128, 2.48, 0.61, 0.240, 0.053, 0.0335) <= 1.06 * time(256, 2.71, 1.31, 0.372, 0.104, 0.0438)) return launch<128, true>(ctx, c, a);
  return launch<256, true>(ctx, c, a);
}
