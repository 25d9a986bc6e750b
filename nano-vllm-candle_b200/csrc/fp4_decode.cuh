// Attention of few query rows over the 4-bit paged cache on mma.sync.m16n8k16 (fp16 operands, fp32 sums), for decode and for portions of few tokens.
//
// The cached tokens are the M side of both products, so that 8 columns - the query heads of a key head, or their rows for a few tokens - cost 16 matrix
// instructions for 16 tokens of 128 + 128 numbers, half of what a tile with the columns on the M side takes:
//   S^T [16 tokens, 8] = K [16, 128] . Q^T [128, 8];   O^T [128, 8] += V^T [128, 16] . P^T [16, 8]
// K's and V's fragments are made in registers: a thread's 16 bytes of a K row are its 32 dims (the order of the dims in the sum is free: Q's fragments have the same), and its 8
// bytes of a V row are 16 neighbouring dims of the result.  V's fragments pair two tokens in a register: their codes are put side by side before they are decoded (4 logical
// instructions for 16 numbers).  P goes from accumulator to operand through movmatrix.
//
// A warp is alone with a ring of two tiles of 32 tokens in shared memory, filled by bulk copies of a page's rows (4 608 bytes a tile).  The rows of a tile (of 16 tokens each time) are the
// products' rows in an order in which neither the reads of K nor those of V meet in a bank more than twice.
//
// Work is cut by what the device finds in the lengths: all tiles of all (sequence, key head, columns) units, one behind another, in equal stretches, one for each warp of a grid that fills the
// GPU once; a unit counts as kUnitCost tiles more than it has, for its queries and its result.  A unit inside a warp's stretch is written by it; the pieces of others are joined in shared memory
// where the warps are of one CTA, and by a second kernel (combine) where not.  Contexts of any mixture of lengths thus take the time of their sum.
//
// A cached value that is no number counts for the columns that see it, and for no other: where a tile is not seen whole by every column, such a value goes in as 0 (a weight of 0 would not keep
// it out), and the first token that has one in each block of 16 dims is remembered for the columns that do see it.
//
// What bounds it: a warp's instructions and their latency (2.5 of 4 an SM and cycle, the ALU at half its rate).  A tile takes 719 of them in pages of 16 and 629 in pages of 256, of which 288 are its
// arithmetic (128 conversions of two numbers, 128 products with their scales, 32 matrix instructions); the others are on the ALU (163, 134: bytes of words taken apart and put together, scales widened,
// masks, addresses) and the FMA pipe (106, 87: exponents, sums, references), and 55 to 75 loads, branches and barriers.  256 contexts of 1 to 4 000 tokens, 8 key heads of
// 4 query heads: 136 us for 596 MB, 4.4 TB/s; 4 of 30 000 to 131 000, 8 query heads: 80 us, 4.6 TB/s.
//
// The exponentials are taken against a reference that follows a column's maximum only when that grew by more than 2^8 (a vote; nothing is exchanged otherwise), shifted by 2^7: weights lie
// below 2^15, inside fp16, and those down to 2^-31 of the largest are kept.  Queries are brought to fp16 behind a power of two of their own, that the score's factor takes back.
#pragma once
#include "fp4.cuh"
#include "ptx.cuh"

namespace fp4d {

constexpr int kTile = 32, kHalf = 16, kWarps = 4;
constexpr int kAtV = kTile * kFp4Codes, kAtKs = 2 * kAtV, kAtVs = kAtKs + kTile * kFp4Scales;      // of a stage: K codes, V codes, K scales, V scales
constexpr int kStageBytes = kAtVs + kTile * kFp4Scales;
constexpr float kFloor = -3.0e38f;                                     // a piece's reference for a column that saw nothing in it
constexpr float kShift = 7.0f, kMost = 15.0f;
constexpr int kUnitCost = 2;

struct Args {
  const nvc_bf16* q;
  nvc_bf16* out;
  int64_t ldq, ldo;
  const uint8_t *kc, *ks, *vc, *vs;
  const int32_t *block_tables, *context_lens, *cu_seqlens;             // cu_seqlens null: one row of each sequence
  int bt_stride, num_blocks, kv, block_size, B, group, rows;
  float scale_log2e;
  int4* notes;                                                         // of each CTA, what begins there and ends in another: sequence (-1: nothing), unit, last CTA
  float* parts;                                                        // two records of each CTA
  int warps;                                                           // of the attention kernel's grid
  int alone;                                                           // > 0: each unit in a CTA of its own (no joining kernel); in decode, units of a sequence
};

// CTAs of an SM.  16 columns: 229 registers, of 168 (three CTAs) some go to memory: 256 contexts of 2 000, us: 186 / 172, 32 of 1 750 37 / 31.  8 columns: 4 and 3 CTAs alike
template <int NT> constexpr int kCtas = NT == 1 ? 4 : 2;
// Decode of short contexts: a CTA for each unit, which needs neither the list nor the joining kernel, where all units run at once and the longest that the tables have room for would not hold up the
// others for long.  In us, with the list / without (caches cold; 16 heads to 8): 1 x 128 10.3 / 6.2, 1 x 512 10.3 / 8.3, 1 x 1 024 11.1 / 12.3, 37 x 256 14.3 / 9.2, 37 x 1 024 22.5 / 16.4; of
// lengths from 1 on, a call behind the other, 74 x 1 024 18.9 / 18.2, 74 x 1 536 22.8 / 24.6; in more than one wave 112 x 1 024 40.6 / 43.0
template <int NT> bool alone(int sms, int64_t units, int64_t tiles) { return units <= (int64_t)sms * kCtas<NT> && tiles <= std::min<int64_t>(32, 24 + units / 12); }
constexpr int kRing = 2;                                               // tiles of a warp's ring (three and four: no difference)
constexpr int kRingBytes = kRing * kStageBytes;
template <int NT> constexpr int kCols = 8 * NT;
template <int NT> constexpr int kRecord = kCols<NT> * 130;             // floats: O [cols][128], reference [cols], sum [cols]
template <int NT> constexpr int kWarpBytes = kRingBytes + kRecord<NT> * 4;     // a stretch's last piece goes where the ring was
template <int NT> constexpr int kSmem = kWarps * kWarpBytes<NT>;
static_assert(kRecord<2> * 4 <= kRingBytes, "a record fits where the ring was");

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void mma(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t mul2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ uint32_t halves(float lo, float hi) {
  uint32_t d;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}
// (volatile, and of memory: held behind the wait for their stage and in front of the warp's barrier that lets it be filled again.  Without either: the same times within half a percent)
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t lds16(uint32_t a) {
  uint16_t v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t lds8(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.u8 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}
// The copies that the barrier counts are of memory of this GPU, so that it always completes
__device__ __forceinline__ void wait_bar(uint32_t bar, uint32_t parity) {
  uint32_t spins = 0;
  while (!ptx::mbar_try_wait(bar, parity))
    if (++spins > (1u << 23)) __trap();
}

// A sequence's share of the work: `units` (key head, columns) units of `tiles` tiles.
struct Seq { int len, qlen, tiles, units; };
template <int NT>
__device__ __forceinline__ Seq seq_of(const Args& p, int b) {
  Seq s;
  const int64_t room = (int64_t)p.bt_stride * p.block_size;
  s.len = (int)min((int64_t)max(p.context_lens[b], 0), room);
  s.qlen = p.cu_seqlens ? min(max(p.cu_seqlens[b + 1] - p.cu_seqlens[b], 0), p.rows) : 1;
  s.tiles = s.len / kTile + (s.len % kTile != 0);
  s.units = p.kv * ((s.qlen * p.group + kCols<NT> - 1) / kCols<NT>);
  return s;
}
__device__ __forceinline__ int64_t weight(const Seq& s, bool alone = false) { return s.tiles ? (int64_t)s.units * (alone ? 1 : s.tiles + kUnitCost) : 0; }
// n / d; the short division where the numbers allow it
__device__ __forceinline__ int64_t divide(int64_t n, int64_t d) {
  return (uint64_t)(n | d) >> 32 ? n / d : (int64_t)((uint32_t)n / (uint32_t)d);
}

// The list, summed: a lane has the sequences [lane * m, lane * m + m)
struct List { int m; int64_t upto, total; };            // upto: this lane's last sequence included
template <int NT>
__device__ __forceinline__ List list_of(const Args& p, int lane, bool alone = false) {
  List x;
  x.m = (p.B + 31) / 32;
  x.upto = 0;
#pragma unroll 4
  for (int i = 0; i < x.m; ++i) {
    const int b = lane * x.m + i;
    const Seq s = seq_of<NT>(p, min(b, p.B - 1));
    x.upto += b < p.B ? weight(s, alone) : 0;
  }
#pragma unroll
  for (int w = 1; w < 32; w <<= 1) {
    const int64_t up = __shfl_up_sync(0xffffffffu, x.upto, w);
    if (lane >= w) x.upto += up;
  }
  x.total = __shfl_sync(0xffffffffu, x.upto, 31);
  return x;
}

// A warp's pieces, one behind another: tiles [t, end) of unit u of sequence b.  `rest`: what the stretch still has behind the unit's begin.
struct Piece {
  int b, u, t, end, rest;
  Seq s;
  __device__ __forceinline__ bool cut(int into) {       // the unit's tiles from weight `into` of it on, as far as the stretch goes; false: none
    t = max(0, into - kUnitCost);
    end = min(s.tiles, rest - kUnitCost);
    return end > t;
  }
};
// place `at` of the list: its sequence, and what is left of `at` in it
template <int NT>
__device__ __forceinline__ void find(const Args& p, const List& list, int64_t& at, Piece& x, bool alone = false) {
  const int f = __ffs(__ballot_sync(0xffffffffu, list.upto > at)) - 1;
  const int64_t before = __shfl_sync(0xffffffffu, list.upto, max(f - 1, 0));
  at -= f ? before : 0;
  for (x.b = f * list.m;; ++x.b) {
    x.s = seq_of<NT>(p, x.b);
    const int64_t w = weight(x.s, alone);
    if (at < w) break;
    at -= w;
  }
}
template <int NT>
__device__ __forceinline__ bool first_piece(const Args& p, const List& list, int64_t at, int per, Piece& x) {
  if (at >= list.total) return false;
  find<NT>(p, list, at, x);
  const int unit = x.s.tiles + kUnitCost;
  x.u = (int)divide(at, unit);
  const int into = (int)(at - (int64_t)x.u * unit);
  x.rest = into + per;
  return x.cut(into);
}
template <int NT>
__device__ __forceinline__ bool next_piece(const Args& p, Piece& x) {
  x.rest -= x.s.tiles + kUnitCost;
  if (x.rest <= kUnitCost) return false;
  if (++x.u == x.s.units) {
    x.u = 0;
    do {
      if (++x.b >= p.B) return false;
      x.s = seq_of<NT>(p, x.b);
    } while (x.s.units == 0 || x.s.tiles == 0);
  }
  return x.cut(0);
}

// Column c of a unit: which row, which head, and how many keys it sees; false: none
template <int NT>
__device__ __forceinline__ bool column(const Args& p, const Seq& s, int b, int u, int c, int& row, int& head, int& seen) {
  const int chunks = p.kv == s.units ? 1 : s.units / p.kv, kvh = chunks == 1 ? u : u / chunks, r = (u - kvh * chunks) * kCols<NT> + c;
  int i = 0;
  row = b;
  if (p.cu_seqlens) {
    i = r / p.group;
    row = p.cu_seqlens[b] + i;
  }
  head = kvh * p.group + (r - i * p.group);
  seen = s.len - s.qlen + i + 1;
  return (p.cu_seqlens ? i < s.qlen : r < p.group) && (unsigned)row < (unsigned)p.rows;
}

// kPortions: rows of a sequence see more or fewer keys (with the look for numbers that are none, decode would take 3 % longer: 64 tokens behind 128 .. 4 000 in 28.3 us for 27.3)
template <int NT, bool kPortions>
__global__ void __launch_bounds__(32 * kWarps, kCtas<NT>) attn_kernel(const Args p) {
  pdl_trigger();
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(8) uint64_t bars[kWarps][kRing];
  __shared__ int4 pieces[kWarps][2];                  // sequence (-1: no piece), unit, first tile, tile behind the last
  __shared__ int tiles_of[kWarps][2];
  __shared__ int nan_from[kWarps][9];                 // by blocks; and whether there is one
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  if (lane < 2) pieces[warp][lane] = make_int4(-1, 0, 0, 0);
  const uint32_t bar = smem_u32(&bars[warp][0]);
  if (lane == 0) {
#pragma unroll
    for (int i = 0; i < kRing; ++i) ptx::mbar_init(bar + 8 * i, 1);
    ptx::fence_barrier_init();
  }
  __syncwarp();
  const bool alone = p.alone > 0;
  int per = 0;
  bool any, idle = false;                             // this warp has tiles; the CTA has none
  Piece at{};
  uint8_t* const mine = smem + warp * kWarpBytes<NT>;
  const uint32_t ring = smem_u32(mine);
  if (alone) {                                        // a unit's tiles, shared by the CTA's warps
    if constexpr (kPortions) {
      const List list = list_of<NT>(p, lane, true);
      int64_t place = blockIdx.x;
      idle = place >= list.total;
      if (!idle) find<NT>(p, list, place, at, true);
      at.u = (int)place;
    } else {
      at.b = blockIdx.x / p.alone;
      at.u = blockIdx.x - at.b * p.alone;
      at.s = seq_of<NT>(p, at.b);
      idle = at.s.tiles == 0;
    }
    const int share = (at.s.tiles + kWarps - 1) / kWarps;
    at.t = min(warp * share, at.s.tiles);
    at.end = min(at.t + share, at.s.tiles);
    at.rest = 0;                                      // no piece behind it
    any = !idle && at.t < at.end;
  } else {
    const List list = list_of<NT>(p, lane);
    per = max((int)divide(list.total + p.warps - 1, p.warps), 1 + kUnitCost);          // (a stretch of 2^31 tiles would be 10 TB of cache)
    any = first_piece<NT>(p, list, (int64_t)per * (blockIdx.x * kWarps + warp), per, at);
    idle = (int64_t)per * (blockIdx.x * kWarps) >= list.total;
  }

  // ---- the reading side: ahead by what the ring holds.  Lane 0 copies; the others know which rows are not there
  const int per_page = p.block_size / kHalf, last_page = p.bt_stride - 1;
  const bool whole = (per_page & 1) == 0;             // a tile lies in one page
  Piece rd = at;
  bool rd_any = any;
  int page = 0, page_left = 0, kvh = 0, next = 0;     // halves that the page still has; the next page's block
  uint32_t half_at = 0;                               // the place's half, counted through the cache
  bool there = false;                                 // the pool has the page
  auto turn = [&](int blk, int in_page) {
    there = (unsigned)blk < (unsigned)p.num_blocks;
    half_at = ((uint32_t)blk * p.kv + kvh) * per_page + in_page;
    page_left = per_page - in_page;
    next = p.block_tables[(int64_t)rd.b * p.bt_stride + min(page + 1, last_page)];
  };
  auto enter = [&] {                                  // to a piece's first tile
    const int chunks = p.kv == rd.s.units ? 1 : rd.s.units / p.kv;
    kvh = chunks == 1 ? rd.u : rd.u / chunks;
    page = 2 * rd.t / per_page;
    turn(p.block_tables[(int64_t)rd.b * p.bt_stride + page], 2 * rd.t - page * per_page);
  };
  if (rd_any) {
    enter();
    // the first rows on their way to L2, where whatever is still written finds them (they are read behind the wait).  With the store's weights alike a decode
    // step of the 0.6B model takes 0.956 ms for 0.967 (one sequence of 100), 1.048 for 1.058 (of 500)
    if (there) {
      const int tiles = whole ? min(min(kRing, rd.end - rd.t), page_left / 2) : 1, line = lane & 15;
      for (int i = 0; i < tiles; ++i) {
        const uint64_t half = half_at + 2 * i;
        if (whole || line < 8) fp4_prefetch((lane < 16 ? p.kc : p.vc) + half * (kHalf * kFp4Codes) + 128 * line);
        if (line < (whole ? 2 : 1)) fp4_prefetch((lane < 16 ? p.ks : p.vs) + half * (kHalf * kFp4Scales) + 128 * line);
      }
    }
  }
  pdl_wait();

  // sequences without a context: zeros
  for (int b = blockIdx.x * kWarps + warp; b < p.B; b += p.warps) {
    const Seq s = seq_of<NT>(p, b);
    if (s.tiles == 0)
      for (int i = 0; i < s.qlen; ++i) {
        const int row = p.cu_seqlens ? p.cu_seqlens[b] + i : b;
        if ((unsigned)row < (unsigned)p.rows)
          for (int c = lane; c < p.kv * p.group * 16; c += 32) reinterpret_cast<uint4*>(p.out + row * p.ldo)[c] = make_uint4(0, 0, 0, 0);
      }
  }
  if (idle) {
    if (threadIdx.x == 0 && !alone) p.notes[blockIdx.x] = make_int4(-1, 0, 0, 0);
    return;
  }

  // half a tile, or all of it (rows: 16 or 32)
  auto copy = [&](uint32_t to, uint32_t to_scales, uint32_t stage_bar, int rows) {
    ptx::bulk_load(to, p.kc + (uint64_t)half_at * (kHalf * kFp4Codes), rows * kFp4Codes, stage_bar);
    ptx::bulk_load(to + kAtV, p.vc + (uint64_t)half_at * (kHalf * kFp4Codes), rows * kFp4Codes, stage_bar);
    ptx::bulk_load(to_scales + kAtKs, p.ks + (uint64_t)half_at * (kHalf * kFp4Scales), rows * kFp4Scales, stage_bar);
    ptx::bulk_load(to_scales + kAtVs, p.vs + (uint64_t)half_at * (kHalf * kFp4Scales), rows * kFp4Scales, stage_bar);
  };
  uint32_t absent = 0;                                // bit 2 * stage + h: half h was not copied
  auto issue = [&](int stage) {
    if (!rd_any) return;
    const uint32_t st = ring + stage * kStageBytes, stage_bar = bar + 8 * stage;
    uint32_t gone = 0;
    if (whole) {
      if (page_left == 0) {
        ++page;
        turn(next, 0);
      }
      if (there) {
        if (ptx::elect_one()) {
          ptx::mbar_arrive_expect_tx(stage_bar, kStageBytes);
          copy(st, st, stage_bar, kTile);
        }
      } else {
        gone = 3;
        if (lane == 0) ptx::mbar_arrive(stage_bar);
      }
      page_left -= 2;
      half_at += 2;
    } else {                                          // a barrier phase takes one arrival: behind both halves, by the lane that told it their bytes
      const bool one = ptx::elect_one();
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (rd.t * kTile + h * kHalf < rd.s.len) {
          if (page_left == 0) {
            ++page;
            turn(next, 0);
          }
          if (there) {
            if (one) {
              asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(stage_bar), "r"(kStageBytes / 2) : "memory");
              copy(st + h * kHalf * kFp4Codes, st + h * kHalf * kFp4Scales, stage_bar, kHalf);
            }
          } else {
            gone |= 1u << h;
          }
          --page_left;
          ++half_at;
        } else {
          gone |= 1u << h;
        }
      }
      if (one) ptx::mbar_arrive(stage_bar);
    }
    absent = (absent & ~(3u << (2 * stage))) | gone << (2 * stage);
    if (++rd.t == rd.end) {
      rd_any = next_piece<NT>(p, rd);
      if (rd_any) {
        enter();
        int row, head, seen;                          // its queries, on their way to L2
        if (!(t & 1) && column<NT>(p, rd.s, rd.b, rd.u, g, row, head, seen)) fp4_prefetch(p.q + row * p.ldq + (int64_t)head * 128 + 32 * t);
      }
    }
  };

  if (any) {
    // ---- the computing side
    uint4 qw[NT][4];
    uint32_t qf[NT][16];
    float o[NT][8][4], ref[NT][2], sum[NT][2], factor[NT][2];
    int lim[NT][2], least = 0;                        // keys that this thread's columns see, and the unit's column that sees least
    int begun = 0;                                    // first tile of this piece
    bool head_piece = true;                           // the stretch's first
    bool fresh = true;                                // no tile of the piece has been looked at: the references are 0, and take the first maximum
    int limit[NT];                                    // of column g

    auto load_q = [&] {
#pragma unroll
      for (int x = 0; x < NT; ++x) {
        int row, head, seen;
        const bool real = column<NT>(p, at.s, at.b, at.u, 8 * x + g, row, head, seen);
        const uint4* src = reinterpret_cast<const uint4*>(p.q + (real ? row * p.ldq + (int64_t)head * 128 : 0)) + 4 * t;
#pragma unroll
        for (int i = 0; i < 4; ++i) qw[x][i] = real ? src[i] : make_uint4(0, 0, 0, 0);
        limit[x] = real ? seen : 0x7fffffff;
      }
    };
    auto begin = [&] {
      begun = at.t;
      fresh = true;
      if (kPortions) {
        __syncwarp();                                   // (the unit before has read it)
        if (lane < 9) nan_from[warp][lane] = lane < 8 ? 0x7fffffff : 0;
        __syncwarp();
      }
      least = at.s.len;
#pragma unroll
      for (int x = 0; x < NT; ++x) {
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) top = max(top, fp4_amax8(qw[x][i]));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // 2^-e brings the largest number to [1, 2); a row with an infinity or a NaN, or of zeros, stays as it is.  (2^-e and 2^e are floats for -126 <= e <= 126;
        // rows beyond are brought to [1, 4) or stay below 1.)
        int e = top >= 0x7f80u || top == 0 ? 0 : (int)(top >> 7) - 127;
        e = min(max(e, -126), 126);
        const float down = __uint_as_float((uint32_t)(127 - e) << 23), back = __uint_as_float((uint32_t)(127 + e) << 23);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t f[4] = {qw[x][i].x, qw[x][i].y, qw[x][i].z, qw[x][i].w};
#pragma unroll
          for (int j = 0; j < 4; ++j) qf[x][4 * i + j] = halves(bf16_lo(f[j]) * down, bf16_hi(f[j]) * down);
        }
        least = min(least, limit[x]);
#pragma unroll
        for (int c = 0; c < 2; ++c) {                 // columns 2t, 2t + 1 are lanes 8t, 8t + 4's
          factor[x][c] = __shfl_sync(0xffffffffu, back, 8 * t + 4 * c) * p.scale_log2e;
          lim[x][c] = min(__shfl_sync(0xffffffffu, limit[x], 8 * t + 4 * c), at.s.len);
          ref[x][c] = 0.f;
          sum[x][c] = 0.f;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) o[x][j][0] = o[x][j][1] = o[x][j][2] = o[x][j][3] = 0.f;
      }
      least = __reduce_min_sync(0xffffffffu, least);
    };

    // a unit, or this warp's piece of it, is complete
    auto end = [&] {
      const bool begins = begun == 0, ends = at.end == at.s.tiles;
#pragma unroll
      for (int x = 0; x < NT; ++x)
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int w = 4; w < 32; w <<= 1) sum[x][c] += __shfl_xor_sync(0xffffffffu, sum[x][c], w);
      if (kPortions && nan_from[warp][8]) {             // this thread's dims are block g
        const int from = nan_from[warp][g];
#pragma unroll
        for (int x = 0; x < NT; ++x)
#pragma unroll
          for (int c = 0; c < 2; ++c)
            if (from < lim[x][c]) {
#pragma unroll
              for (int j = 0; j < 8; ++j) o[x][j][c] = o[x][j][c + 2] = __uint_as_float(0x7fffffffu);
            }
      }
      if (begins && ends) {
#pragma unroll
        for (int x = 0; x < NT; ++x)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            int row, head, seen;
            if (!column<NT>(p, at.s, at.b, at.u, 8 * x + 2 * t + c, row, head, seen)) continue;
            const float inv = sum[x][c] == 0.f ? 0.f : 1.0f / sum[x][c];       // seen nothing: zeros
            uint4* dst = reinterpret_cast<uint4*>(p.out + row * p.ldo + (int64_t)head * 128) + 2 * g;
            uint32_t w[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) w[j] = pack_bf16(o[x][j][c] * inv, o[x][j][c + 2] * inv);
            dst[0] = make_uint4(w[0], w[1], w[2], w[3]);
            dst[1] = make_uint4(w[4], w[5], w[6], w[7]);
          }
      } else {
        // the stretch's first piece has a place of its own; its last, with nothing on its way any more, the ring's
        float* rec = reinterpret_cast<float*>(mine + (head_piece ? kRingBytes : 0));
        __syncwarp();
#pragma unroll
        for (int x = 0; x < NT; ++x)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float* to = rec + (8 * x + 2 * t + c) * 128 + 16 * g;
#pragma unroll
            for (int j = 0; j < 4; ++j)
              reinterpret_cast<float4*>(to)[j] = make_float4(o[x][2 * j][c], o[x][2 * j][c + 2], o[x][2 * j + 1][c], o[x][2 * j + 1][c + 2]);
            if (g == 0) {
              rec[kCols<NT> * 128 + 8 * x + 2 * t + c] = sum[x][c] == 0.f ? kFloor : ref[x][c];
              rec[kCols<NT> * 129 + 8 * x + 2 * t + c] = sum[x][c];
            }
          }
        if (lane == 0) {
          pieces[warp][head_piece ? 0 : 1] = make_int4(at.b, at.u, begun, at.end);
          tiles_of[warp][head_piece ? 0 : 1] = at.s.tiles;
        }
      }
      head_piece = false;
    };

    // row r of the products is token r, the two of every second pair exchanged: K's reads (rows g) take both 64-byte halves of 128 at once, and V's (rows 2t) two of each
    const int rk = g ^ ((g >> 1) & 1), rv = 2 * t + (t & 1);                 // tokens of rows g and 2t; of row 2t + 1: rv ^ 1
    const uint32_t at_k = (uint32_t)(rk * kFp4Codes + t * 16), at_ks = (uint32_t)(kAtKs + rk * kFp4Scales + 2 * t);
    const uint32_t at_v = (uint32_t)(kAtV + rv * kFp4Codes + g * 8), at_v1 = (uint32_t)(kAtV + (rv ^ 1) * kFp4Codes + g * 8);
    const uint32_t at_vs = (uint32_t)(kAtVs + rv * kFp4Scales + g), at_vs1 = (uint32_t)(kAtVs + (rv ^ 1) * kFp4Scales + g);
    load_q();
#pragma unroll
    for (int i = 0; i < kRing - 1; ++i) issue(i);
    begin();
#pragma unroll 1
    for (int i = 0;; ++i) {
      __syncwarp();                                   // everyone is done with the stage that is filled now
      issue((i + kRing - 1) % kRing);
      const int stage = i % kRing;
      uint32_t st = ring + stage * kStageBytes;
      wait_bar(bar + 8 * stage, (i / kRing) & 1);
      const uint32_t gone = (absent >> (2 * stage)) & 3u;
      if (gone || (at.t + 1) * kTile > at.s.len) {    // rows that are not there: scales of 0, whatever their codes are
        if ((gone >> (lane >> 4)) & 1 || at.t * kTile + lane >= at.s.len) {
          asm volatile("st.shared.v2.u32 [%0], {%1, %1};" ::"r"(st + kAtKs + lane * kFp4Scales), "r"(0) : "memory");
          asm volatile("st.shared.v2.u32 [%0], {%1, %1};" ::"r"(st + kAtVs + lane * kFp4Scales), "r"(0) : "memory");
        }
        ptx::fence_proxy_async_smem();
        __syncwarp();
      }
      if (kPortions && (at.t + 1) * kTile > least) {
        const uint2 scales = lds64(st + kAtVs + lane * kFp4Scales);
        const uint32_t lo = __vcmpeq4(scales.x, 0xffffffffu), hi = __vcmpeq4(scales.y, 0xffffffffu);
        if (__any_sync(0xffffffffu, lo | hi)) {
          if (lo | hi) {
            nan_from[warp][8] = 1;
            for (int i = 0; i < 8; ++i)
              if ((i < 4 ? lo : hi) >> (8 * (i & 3)) & 1) atomicMin(&nan_from[warp][i], at.t * kTile + lane);
            asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(st + kAtVs + lane * kFp4Scales), "r"(scales.x & ~lo), "r"(scales.y & ~hi) : "memory");
          }
          ptx::fence_proxy_async_smem();
          __syncwarp();
        }
      }
      asm volatile("" : "+r"(st)::"memory");
      // ---- S^T = K Q^T: of each half, rows g and g + 8
      float s[NT][2][4];
#pragma unroll
      for (int x = 0; x < NT; ++x)
#pragma unroll
        for (int h = 0; h < 2; ++h) s[x][h][0] = s[x][h][1] = s[x][h][2] = s[x][h][3] = 0.f;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t a = st + h * 1024 + at_k, b = st + h * 128 + at_ks;
        const uint4 lo = lds128(a), hi = lds128(a + 512);
        const uint32_t slo = lds16(b), shi = lds16(b + 64);
        const uint32_t wl[4] = {lo.x, lo.y, lo.z, lo.w}, wh[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const uint32_t fl = (w < 2 ? slo & 0xffu : slo >> 8) * 0x00800080u, fh = (w < 2 ? shi & 0xffu : shi >> 8) * 0x00800080u;
          const uint4 a4 = fp4_halves8(wl[w]), b4 = fp4_halves8(wh[w]);
          const uint32_t a0 = mul2(a4.x, fl), a2 = mul2(a4.y, fl), c0 = mul2(a4.z, fl), c2 = mul2(a4.w, fl);
          const uint32_t a1 = mul2(b4.x, fh), a3 = mul2(b4.y, fh), c1 = mul2(b4.z, fh), c3 = mul2(b4.w, fh);
#pragma unroll
          for (int x = 0; x < NT; ++x) {
            mma(s[x][h], a0, a1, a2, a3, qf[x][4 * w], qf[x][4 * w + 1]);
            mma(s[x][h], c0, c1, c2, c3, qf[x][4 * w + 2], qf[x][4 * w + 3]);
          }
        }
      }
      // ---- exponents: of half h, rows g (0, 1) and g + 8 (2, 3), columns 2t and 2t + 1
#pragma unroll
      for (int x = 0; x < NT; ++x)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int c = 0; c < 4; ++c) s[x][h][c] = fmaf(s[x][h][c], factor[x][c & 1], -ref[x][c & 1]);
      if ((at.t + 1) * kTile > least) {               // some column does not see the whole tile
        const int tok = at.t * kTile + rk;
#pragma unroll
        for (int x = 0; x < NT; ++x)
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int c = 0; c < 4; ++c) s[x][h][c] = tok + 16 * h + 4 * (c & 2) < lim[x][c & 1] ? s[x][h][c] : -INFINITY;
      }
      float top[NT][2], most = -INFINITY;
#pragma unroll
      for (int x = 0; x < NT; ++x)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          top[x][c] = fmaxf(fmaxf(s[x][0][c], s[x][0][c + 2]), fmaxf(s[x][1][c], s[x][1][c + 2]));
          most = fmaxf(most, top[x][c]);
        }
      if (fresh || __any_sync(0xffffffffu, most > kMost)) {
#pragma unroll
        for (int x = 0; x < NT; ++x)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
#pragma unroll
            for (int w = 4; w < 32; w <<= 1) top[x][c] = fmaxf(top[x][c], __shfl_xor_sync(0xffffffffu, top[x][c], w));
            const float over = top[x][c] - kShift;
            const float up = fresh ? (over == -INFINITY ? 0.f : over) : fmaxf(0.f, over), a = fresh ? 0.f : ex2(-up);
            ref[x][c] += up;
            sum[x][c] *= a;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              s[x][h][c] -= up;
              s[x][h][c + 2] -= up;
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              o[x][j][c] *= a;
              o[x][j][c + 2] *= a;
            }
          }
        fresh = false;
      }
      uint32_t pb[NT][2][2];
#pragma unroll
      for (int x = 0; x < NT; ++x)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float p0 = ex2(s[x][h][0]), p1 = ex2(s[x][h][1]), p2 = ex2(s[x][h][2]), p3 = ex2(s[x][h][3]);
          sum[x][0] += p0 + p2;
          sum[x][1] += p1 + p3;
          pb[x][h][0] = transpose8(halves(p0, p1));
          pb[x][h][1] = transpose8(halves(p2, p3));
        }
      // ---- O^T += V^T P^T: dims 16g + 2j (row g) and 16g + 2j + 1 (row g + 8); of each half the tokens of rows 2t, 2t + 1, 2t + 8, 2t + 9
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t vb = st + h * 1024, sb = st + h * 128;
        const uint2 ra = lds64(vb + at_v), rb = lds64(vb + at_v1), rc = lds64(vb + at_v + 512), re = lds64(vb + at_v1 + 512);
        const uint32_t f0 = (lds8(sb + at_vs) << 7) | (lds8(sb + at_vs1) << 23), f1 = (lds8(sb + at_vs + 64) << 7) | (lds8(sb + at_vs1 + 64) << 23);
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          const uint32_t xa = w ? ra.y : ra.x, xb = w ? rb.y : rb.x, xc = w ? rc.y : rc.x, xd = w ? re.y : re.x;
          const uint4 a0 = fp4_halves8((xa & 0x0f0f0f0fu) | ((xb << 4) & 0xf0f0f0f0u)), a1 = fp4_halves8(((xa >> 4) & 0x0f0f0f0fu) | (xb & 0xf0f0f0f0u));
          const uint4 a2 = fp4_halves8((xc & 0x0f0f0f0fu) | ((xd << 4) & 0xf0f0f0f0u)), a3 = fp4_halves8(((xc >> 4) & 0x0f0f0f0fu) | (xd & 0xf0f0f0f0u));
          const uint32_t v0[4] = {a0.x, a0.y, a0.z, a0.w}, v1[4] = {a1.x, a1.y, a1.z, a1.w}, v2[4] = {a2.x, a2.y, a2.z, a2.w}, v3[4] = {a3.x, a3.y, a3.z, a3.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t m0 = mul2(v0[j], f0), m1 = mul2(v1[j], f0), m2 = mul2(v2[j], f1), m3 = mul2(v3[j], f1);
#pragma unroll
            for (int x = 0; x < NT; ++x) mma(o[x][4 * w + j], m0, m1, m2, m3, pb[x][h][0], pb[x][h][1]);
          }
        }
      }
      if (++at.t == at.end) {
        Piece now = at;
        const bool more = next_piece<NT>(p, now);
        end();
        if (!more) break;
        at = now;
        load_q();
        begin();
      }
    }
  }
  __syncthreads();

  // ---- pieces of one unit, in the CTA's order of tiles: to the result where that is all of it, else to one of the CTA's two records.  16 threads a column, 8 numbers each
  auto record = [&](int i) { return reinterpret_cast<const float*>(smem + (i >> 1) * kWarpBytes<NT> + (i & 1 ? 0 : kRingBytes)); };
  const int4* piece = &pieces[0][0];
  int4 note = make_int4(-1, 0, 0, 0);
#pragma unroll 1
  for (int i = 0; i < 2 * kWarps;) {
    const int4 head_of = piece[i];
    if (head_of.x < 0) {
      ++i;
      continue;
    }
    int last = i, behind = head_of.w;
    uint32_t in = 1u << i;
    for (int j = i + 1; j < 2 * kWarps; ++j) {
      const int4 x = piece[j];
      if (x.x >= 0) {
        if (x.x != head_of.x || x.y != head_of.y) break;
        last = j;
        behind = x.w;
        in |= 1u << j;
      }
    }
    const int tiles = (&tiles_of[0][0])[i];
    const bool begins = head_of.z == 0, ends = behind == tiles;
    if (begins && !ends)                              // it ends in a later CTA: that many stretches of four warps behind this one's end
      note = make_int4(head_of.x, head_of.y, (int)blockIdx.x + 1 + (int)((tiles - 1 - behind) / ((int64_t)per * kWarps)), 0);
    float* part = p.parts + ((int64_t)blockIdx.x * 2 + (begins ? 1 : 0)) * kRecord<NT>;
    const int d = (threadIdx.x & 15) * 8;
#pragma unroll
    for (int x = 0; x < NT; ++x) {
      const int c = 8 * x + (threadIdx.x >> 4);
      float top = kFloor;
#pragma unroll
      for (int j = 0; j < 2 * kWarps; ++j)
        if (in >> j & 1) top = fmaxf(top, record(j)[kCols<NT> * 128 + c]);
      float l = 0.f;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f), w = v;
#pragma unroll
      for (int j = 0; j < 2 * kWarps; ++j)
        if (in >> j & 1) {
          const float* r = record(j);
          const float f = ex2(r[kCols<NT> * 128 + c] - top);
          const float4 y = *reinterpret_cast<const float4*>(r + c * 128 + d), z = *reinterpret_cast<const float4*>(r + c * 128 + d + 4);
          l += r[kCols<NT> * 129 + c] * f;
          v.x += y.x * f; v.y += y.y * f; v.z += y.z * f; v.w += y.w * f;
          w.x += z.x * f; w.y += z.y * f; w.z += z.z * f; w.w += z.w * f;
        }
      if (begins && ends) {
        int row, head, seen;
        if (column<NT>(p, seq_of<NT>(p, head_of.x), head_of.x, head_of.y, c, row, head, seen)) {
          const float inv = l == 0.f ? 0.f : 1.0f / l;
          *reinterpret_cast<uint4*>(p.out + row * p.ldo + (int64_t)head * 128 + d) =
              make_uint4(pack_bf16(v.x * inv, v.y * inv), pack_bf16(v.z * inv, v.w * inv), pack_bf16(w.x * inv, w.y * inv), pack_bf16(w.z * inv, w.w * inv));
        }
      } else {
        __stcg(reinterpret_cast<float4*>(part + c * 128 + d), v);
        __stcg(reinterpret_cast<float4*>(part + c * 128 + d + 4), w);
        if (d == 0) {
          __stcg(part + kCols<NT> * 128 + c, top);
          __stcg(part + kCols<NT> * 129 + c, l);
        }
      }
    }
    i = last + 1;
  }
  if (threadIdx.x == 0 && !alone) p.notes[blockIdx.x] = note;
}

// Units that lie in several CTAs, by the CTA in which they begin; a warp per column.
template <int NT>
__global__ void __launch_bounds__(32 * kCols<NT>) combine_kernel(const Args p) {
  pdl_trigger();
  const int c0 = blockIdx.x, c = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_wait();
  const int4 note = __ldcg(p.notes + c0);
  if (note.x < 0) return;
  const int c1 = note.z;
  const float* parts = p.parts;
  auto record = [&](int i) { return parts + ((int64_t)i * 2 + (i == c0 ? 1 : 0)) * kRecord<NT>; };
  // weights of the first 32 pieces and numbers of the first 8 on their way together
  constexpr int kAhead = 8;
  float4 x[kAhead];
  auto load = [&](int i0) {
#pragma unroll
    for (int j = 0; j < kAhead; ++j) x[j] = __ldcg(reinterpret_cast<const float4*>(record(min(i0 + j, c1)) + c * 128) + lane);
  };
  load(c0);
  float top = kFloor;
  for (int i = c0 + lane; i <= c1; i += 32) top = fmaxf(top, __ldcg(record(i) + kCols<NT> * 128 + c));
  top = warp_max(top);
  float l = 0.f, w = 0.f;
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i = 0; i <= c1 - c0; i += kAhead) {
    if ((i & 31) == 0) {
      w = 0.f;
      if (c0 + i + lane <= c1) {
        w = ex2(__ldcg(record(c0 + i + lane) + kCols<NT> * 128 + c) - top);
        l += w * __ldcg(record(c0 + i + lane) + kCols<NT> * 129 + c);
      }
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const float f = __shfl_sync(0xffffffffu, w, (i + j) & 31);
      if (c0 + i + j <= c1) { v.x += x[j].x * f; v.y += x[j].y * f; v.z += x[j].z * f; v.w += x[j].w * f; }
    }
    if (i + kAhead <= c1 - c0) load(c0 + i + kAhead);
  }
  l = warp_sum(l);
  int row, head, seen;
  if (!column<NT>(p, seq_of<NT>(p, note.x), note.x, note.y, c, row, head, seen)) return;
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  reinterpret_cast<uint2*>(p.out + row * p.ldo + (int64_t)head * 128)[lane] = make_uint2(pack_bf16(v.x * inv, v.y * inv), pack_bf16(v.z * inv, v.w * inv));
}

}  // namespace fp4d
