// Causal attention of prompt portions over the 4-bit paged cache on tcgen05 (fp16 operands, fp32 sums in tensor memory).
//
// One CTA per SM, 256 query rows - the rows of all the query heads of a key head, head by head within a token - as two tiles of 128 against key tiles of 128 tokens:
//   * 4 warps decode the cache's rows into fp16 tiles in shared memory (K and V, two of each), once for 256 rows: half a percent of what decoding for each head would cost.  A thread
//     has a token's row: 64 bytes of codes and 8 of scales, requested two tiles ahead;
//   * a warp for each tile w issues its products, S_w = Q_w K^T and O_w += P_w V, so that the tensor cores work on one while the other's softmax runs.  There is room for one S: the tiles take
//     it in turn, 128 columns of tensor memory that s_read of the other tile's rows lets go.  P_w (64 columns, fp16 pairs, the A operand) and O_w (128) have their own;
//   * 4 warps for each tile: a thread owns a row, takes its S into registers at once, and writes P_w.  The reference of the exponentials
//     follows the row's maximum when that grew by more than 2^8, shifted by 2^7, as in the kernel for few rows; only then O is rescaled.
// Queries are brought to fp16 behind a power of two of their own row, that the score's factor takes back.  The sign of the scale goes with them, so that a row's maximum may be taken in front of
// the factor.
//
// A cached value that is no number counts for the rows that see it, and for no other.  A weight of 0 would not keep it from them, so it goes in as 0, and the first token with a NaN in each
// block of 16 dims is remembered: a row that sees it has NaN there.
//
// What bounds it: where contexts are long, the tensor cores' waits for softmax and for units' ends (their pipe is busy 62 and 57 % of the cycles) - 2 048 behind 13 952, 32 heads to 8: 360 us, 1 390
// TFLOP/s of 1 675 that a call alone with cold caches may have, and 1 130 to 1 160 of the 1 410 that the power cap leaves calls behind one another; a prompt of 8 191: 435 us, 1 260 of 1 675 -, a unit's
// queries and result where they are short (16 prompts of 1 024: 233 us, 590 TFLOP/s).
//
// Work is cut as in the kernel for few rows: the key tiles of all (sequence, 256 rows, key head) units in one list, an equal stretch for each CTA; units that lie in several CTAs are joined by
// combine_kernel from records in the workspace.
#pragma once
#include "fp4.cuh"
#include "ptx.cuh"

namespace fp4p {

constexpr int kKT = 128, kRows = 256, kThreads = 512;
constexpr int kTileBytes = 128 * 128 * 2;                  // fp16, two halves of 64 dims: [128 rows][128 bytes], 16-byte chunks permuted by the row
constexpr int kHalf = kTileBytes / 2;
constexpr int kOffQ = 0, kOffK = 2 * kTileBytes, kOffV = kOffK + 2 * kTileBytes, kOffFactor = kOffV + 2 * kTileBytes, kOffNan = kOffFactor + kRows * 4, kOffPark = kOffNan + 4 * 48;
constexpr int kOffBar = kOffPark + 8 * 96 + 16;
constexpr int kNumBars = 18;
constexpr int kSmemBytes = kOffBar + kNumBars * 8 + 16 + 1024;          // and room to begin at a multiple of 1024
constexpr int kUnitCost = 5;                               // a unit's queries and result, in tiles (a prompt of 8 191 in us: 4 470, 5 438, 6 439, 9 451; 3 / 5 / 8 for 16 of 1 024 253 / 241 / 251, 64 x 128 behind 400
// 84 / 78 / 83, 8 x 300 behind 1 000 to 8 000 338 / 321 / 324, 2 048 behind 13 952 364 / 362 / 367)
// Where the tables have room for no more, and all units run at once, each has a CTA (in us, stretches and joining / a CTA for each, caches cold, 16 heads to 8: 1 x 100 tokens 22.4 / 12.2, 333 24.6 / 16.3,
// 1 024 30.7 / 25.0, 64 behind 1 000 27.1 / 24.9, behind 2 000 28.9 / 38.9; 32 to 2, 64 behind 1 000 25.9 / 26.6)
constexpr int kAloneTiles = 9;
constexpr float kFloor = -1.0e30f, kShift = 7.0f, kGrow = 8.0f;
constexpr int kRecord = kRows * 130;                       // floats: O [32 groups of 4 dims][256 rows][4], reference [256], sum [256]
constexpr int kChunk = 2048;                               // sequences whose weights are looked at together (in shared memory)

struct Args {
  const nvc_bf16* q;
  nvc_bf16* out;
  int64_t ldq, ldo;
  const uint8_t *kc, *ks, *vc, *vs;
  const int32_t *block_tables, *context_lens, *cu_seqlens;
  int bt_stride, num_blocks, kv, block_size, B, group, rows;
  Fp4Div by_group, by_block;
  float q_sign, factor;                                    // -1, 0 or 1; what scores are multiplied with (positive)
  int4* notes;                                             // of each CTA, the unit that begins there and ends in another: sequence (-1: none), 256 rows' number, key head, last CTA
  float* parts;                                            // two records of each CTA
  bool alone;                                              // a unit for each CTA (no joining kernel)
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t halves(float lo, float hi) {
  uint32_t d;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}
__device__ __forceinline__ uint32_t mul2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
// two fp32 numbers in a register pair, and operations on both at once
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(lo), "f"(hi));
  return d;
}
__device__ __forceinline__ float lo_of(uint64_t x) { return __uint_as_float((uint32_t)x); }
__device__ __forceinline__ float hi_of(uint64_t x) { return __uint_as_float((uint32_t)(x >> 32)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ float max3(float a, uint32_t b, uint32_t c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(__uint_as_float(b)), "f"(__uint_as_float(c)));
  return d;
}
__device__ __forceinline__ void tmem_st_x16(uint32_t at, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(at), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]),
               "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
// instruction descriptor: fp16 x fp16 -> fp32 (formats 0), M = N = 128
__host__ __device__ constexpr uint32_t idesc(int b_mn_major) { return (1u << 4) | ((uint32_t)b_mn_major << 16) | (128u >> 3 << 17) | (128u >> 4 << 24); }

// (without the message of ptx::mbar_wait: a call takes registers from the code around it)
__device__ __forceinline__ void wait_bar(uint32_t bar, uint32_t parity) {
  uint32_t spins = 0;
  while (!ptx::mbar_try_wait(bar, parity))
    if (++spins > NVC_MBAR_SPIN_LIMIT) __trap();
}

struct Seq { int len, qlen, begin, blocks; };              // begin: its first row; blocks: units of 256 rows
__device__ __forceinline__ Seq seq_of(const Args& p, int b) {
  Seq s;
  s.len = (int)min((int64_t)max(p.context_lens[b], 0), (int64_t)p.bt_stride * p.block_size);
  s.begin = p.cu_seqlens[b];
  s.qlen = min(max(p.cu_seqlens[b + 1] - s.begin, 0), p.rows);
  s.blocks = (int)(((int64_t)s.qlen * p.group + kRows - 1) / kRows);
  return s;
}
// key tiles of a unit: up to its last row's last key; one where there is none
__device__ __forceinline__ int tiles_of(const Args& p, const Seq& s, int j) {
  const int last = min(s.qlen - 1, p.by_group(kRows * j + kRows - 1));
  return max(1, (max(s.len - s.qlen + last + 1, 0) + kKT - 1) / kKT);
}

// A CTA's pieces: tiles [t, end) of unit (b, j, h)
struct Piece {
  int b, j, h, t, end, tiles, rest;                        // rest: what the stretch still has behind the unit's begin
  Seq s;
  __device__ __forceinline__ bool cut(int into) {
    t = max(0, into - kUnitCost);
    end = min(tiles, rest - kUnitCost);
    return end > t;
  }
  __device__ __forceinline__ void park(volatile int* to) const {
    to[0] = b; to[1] = j; to[2] = h; to[3] = t; to[4] = end; to[5] = tiles; to[6] = rest; to[7] = s.len; to[8] = s.qlen; to[9] = s.begin; to[10] = s.blocks;
  }
  __device__ __forceinline__ void take(const volatile int* from) {
    b = from[0]; j = from[1]; h = from[2]; t = from[3]; end = from[4]; tiles = from[5]; rest = from[6]; s.len = from[7]; s.qlen = from[8]; s.begin = from[9]; s.blocks = from[10];
  }
};
__device__ __forceinline__ bool next_piece(const Args& p, Piece& x) {
  x.rest -= x.tiles + kUnitCost;
  if (x.rest <= kUnitCost) return false;
  if (++x.h == p.kv) {
    x.h = 0;
    if (++x.j == x.s.blocks) {
      x.j = 0;
      do {
        if (++x.b >= p.B) return false;
        x.s = seq_of(p, x.b);
      } while (x.s.blocks == 0);
    }
    x.tiles = tiles_of(p, x.s, x.j);
  }
  return x.cut(0);
}
__device__ __forceinline__ int64_t sum64(int64_t x) {
#pragma unroll
  for (int w = 1; w < 32; w <<= 1) x += __shfl_xor_sync(0xffffffffu, x, w);
  return x;
}
// Where the CTA's stretch begins, found by all its warps (16) together.  weights: shared memory for kChunk numbers; every thread gets the result.  per: a stretch's length.
__device__ __forceinline__ bool plan(const Args& p, int64_t* weights, int warp, int lane, Piece& x, int& per, int64_t& total) {
  constexpr int kW = kThreads / 32;
  __shared__ int64_t sums[kW];
  auto cost_of = [&](int j, const Seq& s) { return p.alone ? 1 : tiles_of(p, s, j) + kUnitCost; };
  auto weigh = [&](int b) {                                // a sequence's weight, of a whole warp
    const Seq s = seq_of(p, b);
    int64_t mine = 0;
    for (int j = lane; j < s.blocks; j += 32) mine += cost_of(j, s);
    return sum64(mine) * p.kv;
  };
  int64_t mine = 0;
  for (int b = warp; b < p.B; b += kW) {
    const int64_t w = weigh(b);
    if (b < kChunk && lane == 0) weights[b] = w;           // the first of them stay for the second look
    mine += w;
  }
  if (lane == 0) sums[warp] = mine;
  __syncthreads();
  total = 0;
#pragma unroll
  for (int i = 0; i < kW; ++i) total += sums[i];
  per = p.alone ? 1 : max((int)((total + gridDim.x - 1) / gridDim.x), 2 + kUnitCost);
  int64_t at = (int64_t)per * blockIdx.x;
  if (at >= total) return false;
  int b0 = 0;
  for (;;) {                                               // by chunks of sequences
    const int n = min(kChunk, p.B - b0);
    // every warp alike: lanes take runs of m sequences
    const int m = (n + 31) / 32;
    int64_t upto = 0;
    for (int i = 0; i < m; ++i)
      if (lane * m + i < n) upto += weights[lane * m + i];
#pragma unroll
    for (int w = 1; w < 32; w <<= 1) {
      const int64_t up = __shfl_up_sync(0xffffffffu, upto, w);
      if (lane >= w) upto += up;
    }
    const unsigned behind = __ballot_sync(0xffffffffu, upto > at);
    if (behind) {
      const int f = __ffs(behind) - 1;
      const int64_t before = __shfl_sync(0xffffffffu, upto, max(f - 1, 0));
      at -= f ? before : 0;
      int i = f * m;
      while (at >= weights[i]) at -= weights[i++];
      x.b = b0 + i;
      break;
    }
    at -= __shfl_sync(0xffffffffu, upto, 31);
    b0 += kChunk;
    __syncthreads();
    for (int b = b0 + warp; b < min(p.B, b0 + kChunk); b += kW) {
      const int64_t w = weigh(b);
      if (lane == 0) weights[b - b0] = w;
    }
    __syncthreads();
  }
  x.s = seq_of(p, x.b);
  for (int j0 = 0;; j0 += 32) {                            // within the sequence: 256 rows after 256 rows
    const int64_t w = j0 + lane < x.s.blocks ? (int64_t)cost_of(j0 + lane, x.s) * p.kv : 0;
    int64_t upto = w;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t up = __shfl_up_sync(0xffffffffu, upto, d);
      if (lane >= d) upto += up;
    }
    const unsigned behind = __ballot_sync(0xffffffffu, upto > at);
    if (behind) {
      const int f = __ffs(behind) - 1;
      at -= __shfl_sync(0xffffffffu, upto - w, f);
      x.j = j0 + f;
      break;
    }
    at -= __shfl_sync(0xffffffffu, upto, 31);
  }
  x.tiles = tiles_of(p, x.s, x.j);
  if (p.alone) {
    x.h = (int)at;
    x.t = x.rest = 0;                                      // all of it, and nothing behind it
    x.end = x.tiles;
    return true;
  }
  const int unit = x.tiles + kUnitCost;
  x.h = (int)((uint32_t)at / (uint32_t)unit);              // a unit's heads: below 2^32 in all
  const int into = (int)at - x.h * unit;
  x.rest = into + per;
  return x.cut(into);
}

__global__ void __launch_bounds__(kThreads, 1) attn_kernel(const Args p) {
  pdl_trigger();
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* const gen = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t bar0 = base + kOffBar;
  auto q_full = [&](int w) { return bar0 + 8u * w; };
  auto k_full = [&](uint32_t s) { return bar0 + 8u * (2 + s); };
  auto k_empty = [&](uint32_t s) { return bar0 + 8u * (4 + s); };
  auto v_full = [&](uint32_t s) { return bar0 + 8u * (6 + s); };
  auto v_empty = [&](uint32_t s) { return bar0 + 8u * (8 + s); };
  auto s_full = [&](int w) { return bar0 + 8u * (10 + w); };
  auto p_full = [&](int w) { return bar0 + 8u * (12 + w); };
  auto o_done = [&](int w) { return bar0 + 8u * (14 + w); };
  auto s_read = [&](int w) { return bar0 + 8u * (16 + w); };
  const uint32_t tmem_slot = bar0 + 8u * kNumBars;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (warp == 0) {
    if (lane == 0) {
      for (int i = 0; i < 2; ++i) {
        ptx::mbar_init(q_full(i), 128);
        ptx::mbar_init(k_full(i), 128);
        ptx::mbar_init(k_empty(i), 2);
        ptx::mbar_init(v_full(i), 128);
        ptx::mbar_init(v_empty(i), 2);
        ptx::mbar_init(s_full(i), 1);
        ptx::mbar_init(p_full(i), 128);
        ptx::mbar_init(o_done(i), 1);
        ptx::mbar_init(s_read(i), 128);
      }
      ptx::fence_barrier_init();
    }
    __syncwarp();
  } else if (warp == 12) {
    ptx::tmem_alloc(tmem_slot, 512);
    ptx::tmem_relinquish();
  }
  Piece at;
  int per;
  int64_t total;
  const bool any = plan(p, reinterpret_cast<int64_t*>(gen + kOffK), warp, lane, at, per, total);
  ptx::tcgen05_fence_before();
  __syncthreads();
  ptx::tcgen05_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(gen + kOffBar + kNumBars * 8);
  // S of one tile at a time; its reader takes all of it into registers at once.  P of each tile, O of each tile
  const uint32_t tmem_s = tmem;
  auto tmem_p = [&](int w) { return tmem + 128u + 64u * w; };
  auto tmem_o = [&](int w) { return tmem + 256u + 128u * w; };
  pdl_wait();

  if (!any) {
    if (threadIdx.x == 0 && !p.alone) p.notes[blockIdx.x] = make_int4(-1, 0, 0, 0);
  } else if (warp >= 12) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    // ------------------------------------------------------------ the products: a warp for each tile (two of the four).  A product is taken in only when the ones before it are
    // nearly through, so that one warp's waits would leave the tensor cores without work
    if (warp < 14) {
      constexpr uint32_t hi = ptx::umma_desc_hi_sw128(1024);
      const int w = warp - 12;
      uint32_t g = 0, done = 0;
      bool more = true;
      while (more) {
        const int n = at.end - at.t;
        wait_bar(q_full(w), done & 1);
        // S_w(j), then P_w(j - 1) V: the tile's softmax finds its next S when it is through with one
        for (int j = 0; j <= n; ++j) {
          // (operands' addresses are hidden from the compiler: it would keep all of them for all stages)
          if (j < n) {
            const uint32_t k = g + j;
            uint32_t q_lo = ptx::umma_desc_lo(base + kOffQ + w * kTileBytes, 16), k_lo = ptx::umma_desc_lo(base + kOffK + (k & 1) * kTileBytes, 16);
            asm volatile("" : "+r"(q_lo), "+r"(k_lo));
            wait_bar(k_full(k & 1), (k >> 1) & 1);
            wait_bar(s_read(w ^ 1), (k & 1) ^ (w ^ 1));    // the S before this one, of the other tile, has been read: tile 0's waits for tile 1's of k - 1
            ptx::tcgen05_fence_after();
            if (ptx::elect_one()) {
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const uint32_t off = ((i >> 2) * kHalf + (i & 3) * 32) >> 4;
                ptx::umma_bf16_ss(tmem_s, ptx::umma_desc(q_lo + off, hi), ptx::umma_desc(k_lo + off, hi), idesc(0), i != 0);
              }
              ptx::umma_commit(s_full(w));
              ptx::umma_commit(k_empty(k & 1));
            }
            __syncwarp();
          }
          if (j > 0) {
            const uint32_t k = g + j - 1;
            uint32_t v_lo = ptx::umma_desc_lo(base + kOffV + (k & 1) * kTileBytes, (uint32_t)kHalf), from = tmem_p(w), to = tmem_o(w);       // dims are V's rows: 16 tokens a step
            asm volatile("" : "+r"(v_lo), "+r"(from), "+r"(to));
            wait_bar(v_full(k & 1), (k >> 1) & 1);
            wait_bar(p_full(w), k & 1);                    // P is there, O rescaled (or, in a piece's first tile, read out)
            ptx::tcgen05_fence_after();
            if (ptx::elect_one()) {
#pragma unroll
              for (int i = 0; i < 8; ++i) ptx::umma_bf16_ts(to, from + i * 8, ptx::umma_desc(v_lo + i * (2048 >> 4), hi), idesc(1), j > 1 || i != 0);
              ptx::umma_commit(o_done(w));
              ptx::umma_commit(v_empty(k & 1));
            }
            __syncwarp();
          }
        }
        g += n;
        ++done;
        more = next_piece(p, at);
      }
    }
  } else if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");
    // ------------------------------------------------------------ the cache's rows, decoded: a thread has a token of the tile
    const int r = threadIdx.x - 256;
    int* const nan_from = reinterpret_cast<int*>(gen + kOffNan);      // [piece % 4][block; 8: whether there is one; 3 more]
    struct Raw { uint4 c[4]; uint2 s; };
    const int last_page = p.bt_stride - 1;
    auto block_of = [&](const Piece& x, int tile) {        // of this thread's token; -1 where it has none
      const int tok = tile * kKT + r;
      if (tok >= x.s.len) return -1;
      return p.block_tables[(int64_t)x.b * p.bt_stride + min(p.by_block(tok), last_page)];
    };
    auto load = [&](const Piece& x, int tile, int blk, const uint8_t* codes, const uint8_t* scales) {
      Raw w;
      const int tok = tile * kKT + r;
      if (tok < x.s.len && (unsigned)blk < (unsigned)p.num_blocks) {
        const int64_t row = ((int64_t)blk * p.kv + x.h) * p.block_size + (tok - p.by_block(tok) * p.block_size);
        const uint4* c = reinterpret_cast<const uint4*>(codes + row * kFp4Codes);
#pragma unroll
        for (int i = 0; i < 4; ++i) w.c[i] = c[i];
        w.s = *reinterpret_cast<const uint2*>(scales + row * kFp4Scales);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) w.c[i] = make_uint4(0, 0, 0, 0);
        w.s = make_uint2(0, 0);
      }
      return w;
    };
    auto write = [&](const Raw& w, uint32_t tile_at, uint32_t bar) {
      const uint32_t row = tile_at + r * 128;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t c[4] = {w.c[i].x, w.c[i].y, w.c[i].z, w.c[i].w};
        const uint32_t two = (i < 2 ? w.s.x : w.s.y) >> (16 * (i & 1));
#pragma unroll
        for (int k = 0; k < 4; ++k) {                      // 8 dims: chunk 4i + k of 16 bytes
          const uint32_t f = (k < 2 ? two & 0xffu : (two >> 8) & 0xffu) * 0x00800080u;
          const uint4 x = fp4_halves8(c[k]);
          const uint32_t chunk = 4 * (i & 1) + k;
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(row + (i >> 1) * kHalf + ((chunk ^ (r & 7)) << 4)), "r"(mul2(x.x, f)), "r"(mul2(x.y, f)),
                       "r"(mul2(x.z, f)), "r"(mul2(x.w, f)) : "memory");
        }
      }
      ptx::fence_proxy_async_smem();
      ptx::mbar_arrive(bar);
    };
    uint32_t g = 0, done = 0;
    bool more = true;
    Raw rk, rv;
    int b1 = block_of(at, at.t), b2 = at.t + 1 < at.end ? block_of(at, at.t + 1) : -1, b3;
    rk = load(at, at.t, b1, p.kc, p.ks);
    rv = load(at, at.t, b1, p.vc, p.vs);
    while (more) {
      const Piece x = at;
      more = next_piece(p, at);
      const int nb = more ? block_of(at, at.t) : -1;
      wait_bar(k_empty(g & 1), ((g >> 1) & 1) ^ 1u);
      write(rk, base + kOffK + (g & 1) * kTileBytes, k_full(g & 1));
      if (x.t + 1 < x.end) rk = load(x, x.t + 1, b2, p.kc, p.ks);
      else if (more) rk = load(at, at.t, nb, p.kc, p.ks);
      // (the piece four before this one has been written out: the last V went in when a tile of the one three before, at the latest, was through its P V)
      if (r < 9) nan_from[12 * (done & 3) + r] = r < 8 ? 0x7fffffff : 0;
      ptx::named_bar_sync(1, 128);
      for (int j = x.t; j < x.end; ++j, ++g) {
        // b2: the next tile's block; K runs a tile ahead of V
        b3 = j + 2 < x.end ? block_of(x, j + 2) : -1;
        if (j + 1 < x.end) {
          wait_bar(k_empty((g + 1) & 1), (((g + 1) >> 1) & 1) ^ 1u);
          write(rk, base + kOffK + ((g + 1) & 1) * kTileBytes, k_full((g + 1) & 1));
          if (j + 2 < x.end) rk = load(x, j + 2, b3, p.kc, p.ks);
          else if (more) rk = load(at, at.t, nb, p.kc, p.ks);
        }
        wait_bar(v_empty(g & 1), ((g >> 1) & 1) ^ 1u);
        {
          uint32_t bad[2] = {__vcmpeq4(rv.s.x, 0xffffffffu), __vcmpeq4(rv.s.y, 0xffffffffu)};
          if (bad[0] | bad[1]) {
            for (int i = 0; i < 8; ++i)
              if (bad[i >> 2] >> (8 * (i & 3)) & 1) atomicMin(nan_from + 12 * (done & 3) + i, j * kKT + r);
            nan_from[12 * (done & 3) + 8] = 1;
            rv.s.x &= ~bad[0];
            rv.s.y &= ~bad[1];
          }
        }
        write(rv, base + kOffV + (g & 1) * kTileBytes, v_full(g & 1));
        if (j + 1 < x.end) rv = load(x, j + 1, b2, p.vc, p.vs);
        b2 = b3;
      }
      ++done;
      if (more) {
        rv = load(at, at.t, nb, p.vc, p.vs);
        b2 = at.t + 1 < at.end ? block_of(at, at.t + 1) : -1;
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 184;");
    // ------------------------------------------------------------ softmax, a thread for a row; queries in front of a piece, the result behind it
    const int w = warp >> 2, quad = warp & 3, r = quad * 32 + lane;
    const uint32_t lane_at = (uint32_t)(quad * 32) << 16;
    float* const factors = reinterpret_cast<float*>(gen + kOffFactor) + w * 128;
    uint8_t* const q_tile = gen + kOffQ + w * kTileBytes;
    const int* const nan_from = reinterpret_cast<const int*>(gen + kOffNan);
    // what a piece's tiles do not need lies in shared memory meanwhile (with it in registers some of a row's scores went to memory: a prompt of 8 191 in 537 us for 456)
    volatile int* const park = reinterpret_cast<volatile int*>(gen + kOffPark) + warp * 24;
    int4* const note = reinterpret_cast<int4*>(gen + kOffPark + 8 * 96);
    if (threadIdx.x == 0) *note = make_int4(-1, 0, 0, 0);
    uint32_t g = 0, done = 0;
    bool more = true;
    // This warp's 32 rows of a piece's Q, 4 lanes a row: all of it on its way, then to shared memory (that every product of the piece before has read: its last S has been seen).  With 16 lanes
    // a row there were 64 exchanges a thread for these 8: 16 prompts of 1 024 tokens in 249 us for 233
    uint4 y[4][4];
    const int rr = lane & 7, part_of = lane >> 3;           // row of eight, 16-byte chunks part_of, part_of + 4, ..
    auto fetch = [&](const Piece& x) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = kRows * x.j + 128 * w + quad * 32 + 8 * i + rr, tok = p.by_group(row), at_row = x.s.begin + tok;
        const bool there = row < x.s.qlen * p.group && (unsigned)at_row < (unsigned)p.rows;
        const uint4* src = reinterpret_cast<const uint4*>(p.q + (there ? at_row * p.ldq + (int64_t)(x.h * p.group + row - tok * p.group) * 128 : 0)) + part_of;
#pragma unroll
        for (int k = 0; k < 4; ++k) y[i][k] = there ? src[4 * k] : make_uint4(0, 0, 0, 0);
      }
    };
    auto place = [&] {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t top = max(max(fp4_amax8(y[i][0]), fp4_amax8(y[i][1])), max(fp4_amax8(y[i][2]), fp4_amax8(y[i][3])));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 8));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 16));
        int e = top >= 0x7f80u || top == 0 ? 0 : (int)(top >> 7) - 127;
        e = min(max(e, -126), 126);
        const float down = __uint_as_float((uint32_t)(127 - e) << 23) * p.q_sign;
        const int row = quad * 32 + 8 * i + rr;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint4 v = y[i][k];
          const int c = 4 * (k & 1) + part_of;
          *reinterpret_cast<uint4*>(q_tile + (k >> 1) * kHalf + row * 128 + ((c ^ rr) << 4)) =
              make_uint4(halves(bf16_lo(v.x) * down, bf16_hi(v.x) * down), halves(bf16_lo(v.y) * down, bf16_hi(v.y) * down), halves(bf16_lo(v.z) * down, bf16_hi(v.z) * down),
                         halves(bf16_lo(v.w) * down, bf16_hi(v.w) * down));
        }
        if (part_of == 0) factors[row] = fmaxf(__uint_as_float((uint32_t)(127 + e) << 23) * p.factor, 1.2e-38f);        // 0 would turn a masked score into a NaN
      }
      ptx::fence_proxy_async_smem();
      ptx::mbar_arrive(q_full(w));
    };
    auto ahead = [&](const Piece& x) {                      // to L2: 32 rows of two lines
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int row = kRows * x.j + 128 * w + quad * 32 + 16 * i + (lane >> 1), tok = p.by_group(row), at_row = x.s.begin + tok;
        if (row < x.s.qlen * p.group && (unsigned)at_row < (unsigned)p.rows)
          asm volatile("prefetch.global.L2 [%0];" ::"l"(p.q + at_row * p.ldq + (int64_t)(x.h * p.group + row - tok * p.group) * 128 + 64 * (lane & 1)));
      }
    };
    fetch(at);
    place();
    while (more) {
      int lim, least, n, t0;                               // the last key that the row sees, and the warp's first row; tiles; the next tile's first key
      {
        const Piece x = at;
        more = next_piece(p, at);                          // (its lengths are on their way meanwhile)
        if (lane == 0) {
          x.park(park);
          at.park(park + 11);
        }
        const int first = kRows * x.j + 128 * w;           // packed row of the tile's first
        lim = x.s.len - x.s.qlen + min(p.by_group(first + r), x.s.qlen - 1);
        least = x.s.len - x.s.qlen + p.by_group(first + quad * 32);
        n = x.end - x.t;
        t0 = x.t * kKT;
        if (x.s.qlen * p.group - first <= 32 * quad) n = -n;          // a warp without rows
        if (more) ahead(at);
      }
      __syncwarp();
      const float factor = factors[r];
      float ref = kFloor, sum = 0.f;
      if (n < 0) {                                         // its barriers go round alone, and it takes no issue slots from the others: 16 x 16 tokens behind 16 000 in 199 us for 214
        for (int j = 0; j > n; --j, ++g) {
          wait_bar(s_full(w), g & 1);
          ptx::mbar_arrive(s_read(w));
          if (j < 0) wait_bar(o_done(w), (g - 1) & 1);
          ptx::mbar_arrive(p_full(w));
        }
      }
      for (int j = 0; j < n; ++j, ++g, t0 += kKT) {
        wait_bar(s_full(w), g & 1);
        ptx::tcgen05_fence_after();
        const bool cut = t0 + kKT - 1 > least;
        const int l = lim - t0;
        uint32_t sv[128];
        float m0 = -INFINITY, m1 = -INFINITY, m2 = -INFINITY, m3 = -INFINITY;
        ptx::tmem_ld_32x32b_x32(tmem_s + lane_at, sv);
        ptx::tmem_ld_wait();
#pragma unroll
        for (int c = 0; c < 4; ++c) {                        // the next columns are on their way while these are looked at
          if (c < 3) ptx::tmem_ld_32x32b_x32(tmem_s + lane_at + 32 * (c + 1), sv + 32 * (c + 1));
          if (cut) {
#pragma unroll
            for (int i = 32 * c; i < 32 * c + 32; ++i)
              if (i > l) sv[i] = 0xff800000u;
          }
#pragma unroll
          for (int i = 32 * c; i < 32 * c + 32; i += 8) {
            m0 = max3(m0, sv[i], sv[i + 1]);
            m1 = max3(m1, sv[i + 2], sv[i + 3]);
            m2 = max3(m2, sv[i + 4], sv[i + 5]);
            m3 = max3(m3, sv[i + 6], sv[i + 7]);
          }
          if (c < 3) ptx::tmem_ld_wait();
        }
        ptx::tcgen05_fence_before();
        ptx::mbar_arrive(s_read(w));
        const float top = fmaxf(fmaxf(m0, m1), fmaxf(m2, m3)) * factor - kShift;
        const bool move = __any_sync(0xffffffffu, top > ref + kGrow);
        float alpha = 1.0f;
        if (move) {
          const float now = fmaxf(ref, top);
          alpha = ex2(ref - now);
          ref = now;
        }
        uint64_t s0 = 0, s1 = 0;                           // two sums each
        const uint64_t by = pair(factor, factor), less = pair(-ref, -ref);
        auto weights = [&](int from, uint32_t* to) {       // of 32 columns
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            const uint64_t y = fma2(pair(__uint_as_float(sv[from + i]), __uint_as_float(sv[from + i + 1])), by, less), z = fma2(pair(__uint_as_float(sv[from + i + 2]), __uint_as_float(sv[from + i + 3])), by, less);
            const float p0 = ex2(lo_of(y)), p1 = ex2(hi_of(y)), p2 = ex2(lo_of(z)), p3 = ex2(hi_of(z));
            s0 = add2(s0, pair(p0, p1));
            s1 = add2(s1, pair(p2, p3));
            to[i >> 1] = halves(p0, p1);
            to[(i >> 1) + 1] = halves(p2, p3);
          }
        };
        if (j > 0) {
          // the product of the tile before has been added to O, and has read its P.  Looked at in every tile, so that no phase of the barrier is missed
          wait_bar(o_done(w), (g - 1) & 1);
          if (move) {
            ptx::tcgen05_fence_after();
#pragma unroll 1
            for (int c = 0; c < 8; ++c) {
              uint32_t v[16];
              ptx::tmem_ld_32x32b_x16(tmem_o(w) + lane_at + 16 * c, v);
              ptx::tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * alpha);
              tmem_st_x16(tmem_o(w) + lane_at + 16 * c, v);
            }
          }
        }
        uint32_t pw[16];
        weights(0, pw);
        tmem_st_x16(tmem_p(w) + lane_at + 0, pw);
        weights(32, pw);
        tmem_st_x16(tmem_p(w) + lane_at + 16, pw);
        weights(64, pw);
        tmem_st_x16(tmem_p(w) + lane_at + 32, pw);
        weights(96, pw);
        tmem_st_x16(tmem_p(w) + lane_at + 48, pw);
        s0 = add2(s0, s1);
        sum = sum * alpha + (lo_of(s0) + hi_of(s0));
        ptx::tmem_st_wait();
        ptx::tcgen05_fence_before();
        ptx::mbar_arrive(p_full(w));
      }
      // ---- the result, or this CTA's part of it
      at.take(park + 11);
      if (more) {                                          // the next one's queries first: its S is made while this one's O is written
        fetch(at);
        place();
      }
      Piece x;
      x.take(park);
      const int first = kRows * x.j + 128 * w, real = x.s.qlen * p.group, tok = p.by_group(first + r);          // (below 2^31: the host's check)
      const bool rows = real - first > 32 * quad;
      wait_bar(o_done(w), (g - 1) & 1);
      ptx::tcgen05_fence_after();
      const bool begins = x.t == 0, ends = x.end == x.tiles;
      const int* const from = nan_from + 12 * (done++ & 3);
      if (rows && from[8]) {                               // (a NaN in the cache: into O where the row sees it, 16 columns at a time)
#pragma unroll 1
        for (int c = 0; c < 8; ++c) {
          uint32_t v[16];
          ptx::tmem_ld_32x32b_x16(tmem_o(w) + lane_at + 16 * c, v);
          ptx::tmem_ld_wait();
          const bool bad = from[c] <= lim;
#pragma unroll
          for (int i = 0; i < 16; ++i) v[i] = bad ? 0x7fffffffu : v[i];
          tmem_st_x16(tmem_o(w) + lane_at + 16 * c, v);
        }
        ptx::tmem_st_wait();
      }
      if (rows && begins && ends) {
        const float inv = sum == 0.f ? 0.f : 1.0f / sum;   // seen nothing: zeros
        const int at_row = x.s.begin + tok;
        const bool there = first + r < real && (unsigned)at_row < (unsigned)p.rows;
        uint4* dst = reinterpret_cast<uint4*>(p.out + at_row * p.ldo + (int64_t)(x.h * p.group + first + r - tok * p.group) * 128);
        uint32_t v[128];
#pragma unroll
        for (int c = 0; c < 4; ++c) ptx::tmem_ld_32x32b_x32(tmem_o(w) + lane_at + 32 * c, v + 32 * c);
        ptx::tmem_ld_wait();
        if (there) {
#pragma unroll
          for (int k = 0; k < 16; ++k)
            dst[k] = make_uint4(pack_bf16(__uint_as_float(v[8 * k]) * inv, __uint_as_float(v[8 * k + 1]) * inv), pack_bf16(__uint_as_float(v[8 * k + 2]) * inv, __uint_as_float(v[8 * k + 3]) * inv),
                                pack_bf16(__uint_as_float(v[8 * k + 4]) * inv, __uint_as_float(v[8 * k + 5]) * inv), pack_bf16(__uint_as_float(v[8 * k + 6]) * inv, __uint_as_float(v[8 * k + 7]) * inv));
        }
      } else if (rows) {
        if (begins && threadIdx.x == 0) *note = make_int4(x.b, x.j, x.h, (int)blockIdx.x + 1 + (x.tiles - 1 - x.end) / per);
        float* part = p.parts + ((int64_t)blockIdx.x * 2 + (begins ? 1 : 0)) * kRecord;
        const int row = 128 * w + r;
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          uint32_t v[32];
          ptx::tmem_ld_32x32b_x32(tmem_o(w) + lane_at + 32 * c, v);
          ptx::tmem_ld_wait();
#pragma unroll
          for (int k = 0; k < 8; ++k)
            __stcg(reinterpret_cast<float4*>(part) + (8 * c + k) * kRows + row, make_float4(__uint_as_float(v[4 * k]), __uint_as_float(v[4 * k + 1]), __uint_as_float(v[4 * k + 2]), __uint_as_float(v[4 * k + 3])));
        }
        __stcg(part + kRows * 128 + row, sum == 0.f ? kFloor : ref);
        __stcg(part + kRows * 129 + row, sum);
      }
      ptx::tcgen05_fence_before();                         // O has been read: the next P V may write it (p_full)
    }
    if (threadIdx.x == 0 && !p.alone) p.notes[blockIdx.x] = *note;
  }
  ptx::tcgen05_fence_before();
  __syncthreads();
  if (warp == 12) {
    ptx::tcgen05_fence_after();
    ptx::tmem_dealloc(tmem, 512);
  }
}

// Units that lie in several CTAs, by the CTA in which they begin: 32 rows of it a CTA (8 of them a unit), a thread for a row and four dims at a time.
__global__ void __launch_bounds__(256) combine_kernel(const Args p) {
  pdl_trigger();
  const int c0 = blockIdx.x >> 3, lane = threadIdx.x & 31, row = (blockIdx.x & 7) * 32 + lane, d0 = threadIdx.x >> 5;
  pdl_wait();
  const int4 note = __ldcg(p.notes + c0);
  if (note.x < 0) return;
  const Seq s = seq_of(p, note.x);
  const int packed = kRows * note.y + row, tok = p.by_group(packed), at_row = s.begin + tok;
  if (packed >= s.qlen * p.group || (unsigned)at_row >= (unsigned)p.rows) return;          // (no row: its record holds anything)
  const int c1 = note.w;
  auto record = [&](int i) { return p.parts + ((int64_t)i * 2 + (i == c0 ? 1 : 0)) * kRecord; };
  // two records (most units lie in two CTAs) on their way at once, the sums against the larger reference so far
  float top = kFloor, l = 0.f;
  float4 v[4] = {};
  for (int i = c0; i <= c1; i += 2) {
    const float *a = record(i), *b = record(min(i + 1, c1));
    float4 x[4], y[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {                          // dims 16 d0 + 4 k ..
      x[k] = __ldcg(reinterpret_cast<const float4*>(a) + (4 * d0 + k) * kRows + row);
      y[k] = __ldcg(reinterpret_cast<const float4*>(b) + (4 * d0 + k) * kRows + row);
    }
    const float ra = __ldcg(a + kRows * 128 + row), rb = i < c1 ? __ldcg(b + kRows * 128 + row) : kFloor;
    const float la = __ldcg(a + kRows * 129 + row), lb = i < c1 ? __ldcg(b + kRows * 129 + row) : 0.f;
    const float now = fmaxf(top, fmaxf(ra, rb)), f = ex2(top - now), fa = ex2(ra - now), fb = i < c1 ? ex2(rb - now) : 0.f;
    l = l * f + la * fa + lb * fb;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      v[k].x = v[k].x * f + x[k].x * fa + y[k].x * fb;
      v[k].y = v[k].y * f + x[k].y * fa + y[k].y * fb;
      v[k].z = v[k].z * f + x[k].z * fa + y[k].z * fb;
      v[k].w = v[k].w * f + x[k].w * fa + y[k].w * fb;
    }
    top = now;
  }
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  uint4* dst = reinterpret_cast<uint4*>(p.out + at_row * p.ldo + (int64_t)(note.z * p.group + packed - tok * p.group) * 128) + 2 * d0;
#pragma unroll
  for (int k = 0; k < 2; ++k)
    dst[k] = make_uint4(pack_bf16(v[2 * k].x * inv, v[2 * k].y * inv), pack_bf16(v[2 * k].z * inv, v[2 * k].w * inv), pack_bf16(v[2 * k + 1].x * inv, v[2 * k + 1].y * inv),
                        pack_bf16(v[2 * k + 1].z * inv, v[2 * k + 1].w * inv));
}

}  // namespace fp4p
