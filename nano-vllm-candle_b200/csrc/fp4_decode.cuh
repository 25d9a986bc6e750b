// Attention of few query rows over the 4-bit paged cache on mma.sync.m16n8k16 (fp16 operands, fp32 sums), for decode and for portions of few tokens.
//
// The cached tokens are the M side of both products, so that 8 columns - the query heads of a key head, or their rows for a few tokens - cost 16 matrix
// instructions for 16 tokens of 128 + 128 numbers, half of what a tile with the columns on the M side takes:
//   S^T [16 tokens, 8] = K [16, 128] . Q^T [128, 8];   O^T [128, 8] += V^T [128, 16] . P^T [16, 8]
// K's and V's fragments are made in registers: a thread's 16 bytes of a K row are its 32 dims (the order of the dims in the sum is free: Q's fragments have the same), and its 8
// bytes of a V row are 16 neighbouring dims of the result.  V's fragments pair two tokens in a register: their codes are put side by side before they are decoded (4 logical
// instructions for 16 numbers).  P goes from accumulator to operand through movmatrix.
//
// A warp is alone with a ring of four tiles of 16 tokens in shared memory (cp.async, 2 304 bytes a tile).  The scales of rows behind the context, and of pages outside the pool, arrive as
// zeros, so that whatever their codes are counts for nothing.
//
// Work is cut by what the device finds in the lengths: all tiles of all (sequence, key head, columns) units, one behind another, in equal stretches, one for each warp of a grid that fills the
// GPU once.  A unit inside a warp's stretch is written by it; the pieces of others are joined in shared memory where the warps are of one CTA, and by a second kernel (combine) where not.
// Contexts of any mixture of lengths thus take the time of their sum.
//
// The exponentials are taken against a reference that follows a column's maximum only when that grew by more than 2^8 (a vote; nothing is exchanged otherwise), shifted by 2^7: weights lie
// below 2^15, inside fp16, and those down to 2^-31 of the largest are kept.  Queries are brought to fp16 behind a power of two of their own, that the score's factor takes back.
#pragma once
#include "fp4.cuh"

namespace fp4d {

constexpr int kTile = 16, kStages = 4, kWarps = 4;
constexpr int kStageBytes = 2 * kTile * (kFp4Codes + kFp4Scales);      // K codes, V codes, K scales, V scales
constexpr int kRingBytes = kStages * kStageBytes;
constexpr float kFloor = -3.0e38f;                                     // reference of a column that has seen nothing
constexpr float kShift = 7.0f, kMost = 15.0f;
constexpr int kMinTiles = 2;                                           // of a warp's stretch

struct Args {
  const nvc_bf16* q;
  nvc_bf16* out;
  int64_t ldq, ldo;
  const uint8_t *kc, *ks, *vc, *vs;
  const int32_t *tables, *lens, *cu;                                   // cu null: one row of each sequence
  int bt_stride, num_blocks, kv, block_size, B, group, rows;
  float scale_log2e;
  float* parts;                                                        // two records of each CTA
  int warps;                                                           // of the attention kernel's grid
};

template <int NT> constexpr int kCols = 8 * NT;
template <int NT> constexpr int kRecord = kCols<NT> * 130;             // floats: O [cols][128], reference [cols], sum [cols]
template <int NT> constexpr int kWarpBytes = kRingBytes + kRecord<NT> * 4;     // the last piece goes where the ring was
template <int NT> constexpr int kSmem = kWarps * kWarpBytes<NT>;
static_assert(kRecord<2> * 4 <= kRingBytes, "a record fits where the ring was");

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mma(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
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
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
  return v;
}
__device__ __forceinline__ uint32_t lds16(uint32_t a) {
  uint16_t v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(a));
  return v;
}
__device__ __forceinline__ uint32_t lds8(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.u8 %0, [%1];" : "=r"(v) : "r"(a));
  return v;
}

// A sequence's share of the work: `units` (key head, columns) units of `tiles` tiles.
struct Seq { int len, qlen, tiles, units; };
template <int NT>
__device__ __forceinline__ Seq seq_of(const Args& p, int b) {
  Seq s;
  const int64_t room = (int64_t)p.bt_stride * p.block_size;
  s.len = (int)min((int64_t)max(p.lens[b], 0), room);
  s.qlen = p.cu ? max(p.cu[b + 1] - p.cu[b], 0) : 1;
  s.tiles = s.len / kTile + (s.len % kTile != 0);
  s.units = p.kv * ((s.qlen * p.group + kCols<NT> - 1) / kCols<NT>);
  return s;
}
// All tiles, the same in every lane
template <int NT>
__device__ __forceinline__ int64_t total_tiles(const Args& p, int lane) {
  int64_t sum = 0;
  for (int b = lane; b < p.B; b += 32) {
    const Seq s = seq_of<NT>(p, b);
    sum += (int64_t)s.units * s.tiles;
  }
#pragma unroll
  for (int w = 1; w < 32; w <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
  return sum;
}
__device__ __forceinline__ int64_t stretch(const Args& p, int64_t total) {
  const int64_t per = (total + p.warps - 1) / p.warps;
  return per < kMinTiles ? kMinTiles : per;
}

// A place in the list of tiles: tile t of unit u of sequence b
struct Place {
  int b, u, t;
  Seq s;
};
template <int NT>
__device__ __forceinline__ Place find(const Args& p, int64_t at, int lane) {      // at < all tiles
  int64_t before = 0;
  for (int b0 = 0;; b0 += 32) {
    int64_t mine = 0;
    if (b0 + lane < p.B) {
      const Seq s = seq_of<NT>(p, b0 + lane);
      mine = (int64_t)s.units * s.tiles;
    }
    int64_t up = mine;
#pragma unroll
    for (int w = 1; w < 32; w <<= 1) {
      const int64_t x = __shfl_up_sync(0xffffffffu, up, w);
      if (lane >= w) up += x;
    }
    const unsigned behind = __ballot_sync(0xffffffffu, before + up > at);
    if (behind) {
      const int f = __ffs(behind) - 1;
      const int64_t start = before + __shfl_sync(0xffffffffu, up - mine, f);
      Place x;
      x.b = b0 + f;
      x.s = seq_of<NT>(p, x.b);
      x.u = (int)((at - start) / x.s.tiles);
      x.t = (int)(at - start - (int64_t)x.u * x.s.tiles);
      return x;
    }
    before += __shfl_sync(0xffffffffu, up, 31);
  }
}
template <int NT>
__device__ __forceinline__ void next_unit(const Args& p, Place& x) {
  x.t = 0;
  if (++x.u < x.s.units) return;
  x.u = 0;
  do {
    if (++x.b >= p.B) return;
    x.s = seq_of<NT>(p, x.b);
  } while (x.s.units == 0 || x.s.tiles == 0);
}

// Column c of a unit: which row, which head, and how many keys it sees; false: none
template <int NT>
__device__ __forceinline__ bool column(const Args& p, const Seq& s, int b, int u, int c, int& row, int& head, int& seen) {
  const int chunks = s.units / p.kv, kvh = u / chunks, r = (u - kvh * chunks) * kCols<NT> + c;
  const int i = r / p.group;
  head = kvh * p.group + (r - i * p.group);
  row = p.cu ? p.cu[b] + i : b;
  seen = s.len - s.qlen + i + 1;
  return i < s.qlen && (unsigned)row < (unsigned)p.rows;
}

template <int NT>
__global__ void __launch_bounds__(32 * kWarps, NT == 1 ? 4 : 3) attn_kernel(const Args p) {
  pdl_trigger();
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int4 notes[kWarps][2];                   // of a piece: sequence (-1: no piece), unit, whether it begins and ends its unit
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  if (lane < 2) notes[warp][lane] = make_int4(-1, 0, 0, 0);
  pdl_wait();
  const int64_t total = total_tiles<NT>(p, lane), per = stretch(p, total);
  const int64_t first = per * (blockIdx.x * kWarps + warp);
  if (per * blockIdx.x * kWarps >= total) return;                             // the whole CTA
  const int n = (int)max((int64_t)0, min(per, total - first));
  uint8_t* const mine = smem + warp * kWarpBytes<NT>;
  const uint32_t ring = smem_u32(mine);

  if (n > 0) {
    Place at = find<NT>(p, first, lane);

    // ---- the reading side: a place of its own, kStages - 1 tiles ahead
    Place rd = at;
    int rd_left = n, page = -1, blk = -1;              // page: number whose block `blk` is
    const int per_page = p.block_size / kTile;
    int kvh, in_page;
    auto enter = [&] {                                  // a unit's first tile of this stretch
      const int chunks = rd.s.units / p.kv;
      kvh = rd.u / chunks;
      page = rd.t / per_page;
      in_page = rd.t - page * per_page;
      blk = p.tables[(int64_t)rd.b * p.bt_stride + page];
    };
    enter();
    // lane c copies 16-byte chunks c and c + 32 of the 64 of a tile's codes: row c / 4; two rows share 128 bytes, whose eight chunks are permuted so that neither the
    // reads of K (two rows at once) nor those of V (four rows, 32 bytes of each) meet in a bank
    const uint32_t to = (uint32_t)((lane >> 3) * 128 + ((((lane >> 2) & 1) * 4 + (lane & 3)) ^ (2 * ((lane >> 3) & 3))) * 16);
    auto issue = [&](int stage) {
      if (rd_left > 0) {
        const bool there = (unsigned)blk < (unsigned)p.num_blocks;
        const int64_t row = ((int64_t)(there ? blk : 0) * p.kv + kvh) * p.block_size + in_page * kTile;
        const uint32_t st = ring + stage * kStageBytes;
        const uint8_t *k = p.kc + row * kFp4Codes + lane * 16, *v = p.vc + row * kFp4Codes + lane * 16;
        copy16(st + to, k, 16);
        copy16(st + to + 512, k + 512, 16);
        copy16(st + 1024 + to, v, 16);
        copy16(st + 1024 + to + 512, v + 512, 16);
        if (lane < 16) {                                // two rows' scales; zeros for the ones that are not there
          const int live = there ? (rd.s.len - rd.t * kTile - 2 * (lane & 7)) * kFp4Scales : 0;
          copy16(st + 2048 + lane * 16, (lane < 8 ? p.ks : p.vs) + row * kFp4Scales + (lane & 7) * 16, (uint32_t)min(max(live, 0), 16));
        }
        --rd_left;
        if (rd_left > 0) {
          if (++rd.t == rd.s.tiles) {
            next_unit<NT>(p, rd);
            enter();
          } else if (++in_page == per_page) {
            in_page = 0;
            blk = p.tables[(int64_t)rd.b * p.bt_stride + ++page];
          }
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) issue(i);

    // ---- the computing side
    uint32_t qf[NT][16];
    float o[NT][8][4], ref[NT][2], sum[NT][2], factor[NT][2];
    int lim[NT][2], least = 0;                          // keys that this thread's columns see, and the unit's column that sees least
    int begun = 0;                                      // first tile of this piece
    bool head_piece = true;                             // the stretch's first

    auto begin = [&] {
      begun = at.t;
      least = 0x7fffffff;
#pragma unroll
      for (int x = 0; x < NT; ++x) {
        int row, head, seen;
        const bool real = column<NT>(p, at.s, at.b, at.u, 8 * x + g, row, head, seen);
        uint4 w[4] = {};
        if (real) {
          const uint4* src = reinterpret_cast<const uint4*>(p.q + row * p.ldq + (int64_t)head * 128) + 4 * t;
#pragma unroll
          for (int i = 0; i < 4; ++i) w[i] = src[i];
        }
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) top = max(top, fp4_amax8(w[i]));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // 2^-e brings the largest number to [1, 2); a row with an infinity or a NaN, or of zeros, stays as it is.  (2^-e and 2^e are floats for -126 <= e <= 126;
        // rows beyond are brought to [1, 4) or stay below 1.)
        int e = top >= 0x7f80u || top == 0 ? 0 : (int)(top >> 7) - 127;
        e = min(max(e, -126), 126);
        const float down = __uint_as_float((uint32_t)(127 - e) << 23), back = __uint_as_float((uint32_t)(127 + e) << 23);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t f[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
          for (int j = 0; j < 4; ++j) qf[x][4 * i + j] = halves(bf16_lo(f[j]) * down, bf16_hi(f[j]) * down);
        }
        const int limit = real ? seen : 0x7fffffff;
#pragma unroll
        for (int c = 0; c < 2; ++c) {                   // columns 2t, 2t + 1 are lanes 8t, 8t + 4's
          factor[x][c] = __shfl_sync(0xffffffffu, back, 8 * t + 4 * c) * p.scale_log2e;
          lim[x][c] = __shfl_sync(0xffffffffu, limit, 8 * t + 4 * c);
          least = min(least, lim[x][c]);
          ref[x][c] = kFloor;
          sum[x][c] = 0.f;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) o[x][j][0] = o[x][j][1] = o[x][j][2] = o[x][j][3] = 0.f;
      }
      least = __reduce_min_sync(0xffffffffu, min(least, at.s.len));
    };

    // a unit, or this warp's piece of it, is complete
    auto end = [&](int ends_at) {
      const bool begins = begun == 0, ends = ends_at == at.s.tiles;
#pragma unroll
      for (int x = 0; x < NT; ++x)
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int w = 4; w < 32; w <<= 1) sum[x][c] += __shfl_xor_sync(0xffffffffu, sum[x][c], w);
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
        // the stretch's first piece has a place of its own; its last, with nothing left to read, the ring's
        if (!head_piece) {
          asm volatile("cp.async.wait_group 0;" ::: "memory");
          __syncwarp();
        }
        float* rec = reinterpret_cast<float*>(mine + (head_piece ? kRingBytes : 0));
#pragma unroll
        for (int x = 0; x < NT; ++x)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float* to = rec + (8 * x + 2 * t + c) * 128 + 16 * g;
#pragma unroll
            for (int j = 0; j < 4; ++j)
              reinterpret_cast<float4*>(to)[j] = make_float4(o[x][2 * j][c], o[x][2 * j][c + 2], o[x][2 * j + 1][c], o[x][2 * j + 1][c + 2]);
            if (g == 0) {
              rec[kCols<NT> * 128 + 8 * x + 2 * t + c] = ref[x][c];
              rec[kCols<NT> * 129 + 8 * x + 2 * t + c] = sum[x][c];
            }
          }
        if (lane == 0) notes[warp][head_piece ? 0 : 1] = make_int4(at.b, at.u, begins, ends);
      }
      head_piece = false;
    };

    begin();
    for (int i = 0; i < n; ++i) {
      __syncwarp();                                     // everyone is done with the stage that is filled now
      issue((i + kStages - 1) % kStages);
      asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
      __syncwarp();
      const uint32_t st = ring + (i % kStages) * kStageBytes;
      // ---- S^T = K Q^T: rows g and g + 8
      float s[NT][4];
#pragma unroll
      for (int x = 0; x < NT; ++x) s[x][0] = s[x][1] = s[x][2] = s[x][3] = 0.f;
      {
        const uint32_t a = st + (g >> 1) * 128 + ((((g & 1) * 4 + t) ^ (2 * ((g >> 1) & 3))) << 4);
        const uint4 lo = lds128(a), hi = lds128(a + 512);
        const uint32_t slo = lds16(st + 2048 + g * 8 + 2 * t), shi = lds16(st + 2048 + 64 + g * 8 + 2 * t);
        const uint32_t wl[4] = {lo.x, lo.y, lo.z, lo.w}, wh[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const uint32_t fl = (w < 2 ? slo & 0xffu : slo >> 8) * 0x00800080u, fh = (w < 2 ? shi & 0xffu : shi >> 8) * 0x00800080u;
          const uint4 a4 = fp4_halves8(wl[w]), b4 = fp4_halves8(wh[w]);
          const uint32_t a0 = mul2(a4.x, fl), a2 = mul2(a4.y, fl), c0 = mul2(a4.z, fl), c2 = mul2(a4.w, fl);
          const uint32_t a1 = mul2(b4.x, fh), a3 = mul2(b4.y, fh), c1 = mul2(b4.z, fh), c3 = mul2(b4.w, fh);
#pragma unroll
          for (int x = 0; x < NT; ++x) {
            mma(s[x], a0, a1, a2, a3, qf[x][4 * w], qf[x][4 * w + 1]);
            mma(s[x], c0, c1, c2, c3, qf[x][4 * w + 2], qf[x][4 * w + 3]);
          }
        }
      }
      // ---- weights: token g (0, 1) and g + 8 (2, 3), columns 2t and 2t + 1
      const int tok = at.t * kTile + g;
      if ((at.t + 1) * kTile > least) {                 // some column does not see the whole tile
#pragma unroll
        for (int x = 0; x < NT; ++x)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const int l = min(lim[x][c], at.s.len);
            // a factor that turns a masked score's sign, or is 0, leaves it masked: the masked score is what comes out of it
            s[x][c] = tok < l ? s[x][c] * factor[x][c] : -INFINITY;
            s[x][c + 2] = tok + 8 < l ? s[x][c + 2] * factor[x][c] : -INFINITY;
          }
      } else {
#pragma unroll
        for (int x = 0; x < NT; ++x)
#pragma unroll
          for (int c = 0; c < 4; ++c) s[x][c] *= factor[x][c & 1];
      }
      bool grew = false;
#pragma unroll
      for (int x = 0; x < NT; ++x)
#pragma unroll
        for (int c = 0; c < 4; ++c) grew |= s[x][c] - ref[x][c & 1] > kMost;
      if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
        for (int x = 0; x < NT; ++x)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float top = fmaxf(s[x][c], s[x][c + 2]);
#pragma unroll
            for (int w = 4; w < 32; w <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
            const float now = fmaxf(ref[x][c], top - kShift), a = ex2(ref[x][c] - now);
            ref[x][c] = now;
            sum[x][c] *= a;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              o[x][j][c] *= a;
              o[x][j][c + 2] *= a;
            }
          }
      }
      uint32_t pb[NT][2];
#pragma unroll
      for (int x = 0; x < NT; ++x) {
        const float p0 = ex2(s[x][0] - ref[x][0]), p1 = ex2(s[x][1] - ref[x][1]), p2 = ex2(s[x][2] - ref[x][0]), p3 = ex2(s[x][3] - ref[x][1]);
        sum[x][0] += p0 + p2;
        sum[x][1] += p1 + p3;
        pb[x][0] = transpose8(halves(p0, p1));
        pb[x][1] = transpose8(halves(p2, p3));
      }
      // ---- O^T += V^T P^T: dims 16g + 2j (row g) and 16g + 2j + 1 (row g + 8), tokens 2t, 2t + 1, 2t + 8, 2t + 9
      {
        const uint32_t base = st + 1024 + t * 128 + (g & 1) * 8, sw = 2 * t;
        const uint2 ra = lds64(base + (((g >> 1) ^ sw) << 4)), rb = lds64(base + (((4 + (g >> 1)) ^ sw) << 4));
        const uint2 rc = lds64(base + 512 + (((g >> 1) ^ sw) << 4)), re = lds64(base + 512 + (((4 + (g >> 1)) ^ sw) << 4));
        const uint32_t sc = st + 2048 + 128 + t * 16 + g;
        const uint32_t f0 = (lds8(sc) << 7) | (lds8(sc + 8) << 23), f1 = (lds8(sc + 64) << 7) | (lds8(sc + 72) << 23);
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
            for (int x = 0; x < NT; ++x) mma(o[x][4 * w + j], m0, m1, m2, m3, pb[x][0], pb[x][1]);
          }
        }
      }
      ++at.t;
      if (at.t == at.s.tiles || i + 1 == n) {
        end(at.t);
        if (i + 1 < n) {
          next_unit<NT>(p, at);
          begin();
        }
      }
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();

  // ---- pieces of one unit, in the CTA's order of tiles: to the result where that is all of it, else to one of the CTA's two records
  auto record = [&](int i) { return reinterpret_cast<const float*>(smem + (i >> 1) * kWarpBytes<NT> + (i & 1 ? 0 : kRingBytes)); };
  const int4* note = &notes[0][0];
  for (int i = 0; i < 2 * kWarps;) {
    if (note[i].x < 0) {
      ++i;
      continue;
    }
    int last = i;
    for (int j = i + 1; j < 2 * kWarps; ++j)
      if (note[j].x >= 0) {
        if (note[j].x != note[i].x || note[j].y != note[i].y) break;
        last = j;
      }
    const bool begins = note[i].z, ends = note[last].w;
    const int b = note[i].x, u = note[i].y;
    float* part = p.parts + ((int64_t)blockIdx.x * 2 + (begins ? 1 : 0)) * kRecord<NT>;
    const Seq s = seq_of<NT>(p, b);
    for (int c = warp; c < kCols<NT>; c += kWarps) {
      int row, head, seen;
      const bool real = column<NT>(p, s, b, u, c, row, head, seen);
      float top = kFloor;
      for (int j = i; j <= last; ++j)
        if (note[j].x >= 0) top = fmaxf(top, record(j)[kCols<NT> * 128 + c]);
      float l = 0.f;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int j = i; j <= last; ++j)
        if (note[j].x >= 0) {
          const float w = ex2(record(j)[kCols<NT> * 128 + c] - top);
          const float4 x = *reinterpret_cast<const float4*>(record(j) + c * 128 + 4 * lane);
          l += record(j)[kCols<NT> * 129 + c] * w;
          v.x += x.x * w; v.y += x.y * w; v.z += x.z * w; v.w += x.w * w;
        }
      if (begins && ends) {
        const float inv = l == 0.f ? 0.f : 1.0f / l;
        if (real) reinterpret_cast<uint2*>(p.out + row * p.ldo + (int64_t)head * 128)[lane] = make_uint2(pack_bf16(v.x * inv, v.y * inv), pack_bf16(v.z * inv, v.w * inv));
      } else {
        __stcg(reinterpret_cast<float4*>(part + c * 128) + lane, v);
        if (lane == 0) {
          __stcg(part + kCols<NT> * 128 + c, top);
          __stcg(part + kCols<NT> * 129 + c, l);
        }
      }
    }
    i = last + 1;
  }
}

// Units that lie in several CTAs, and those without a tile (zeros).  One CTA per (unit of a sequence, sequence), a warp per column.
template <int NT>
__global__ void __launch_bounds__(32 * kCols<NT>) combine_kernel(const Args p, int most_units) {
  pdl_trigger();
  const int b = blockIdx.x / most_units, u = blockIdx.x - b * most_units, c = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_wait();
  const Seq s = seq_of<NT>(p, b);
  if (u >= s.units) return;
  int row, head, seen;
  if (!column<NT>(p, s, b, u, c, row, head, seen)) return;
  uint2* dst = reinterpret_cast<uint2*>(p.out + row * p.ldo + (int64_t)head * 128) + lane;
  if (s.tiles == 0) {
    *dst = make_uint2(0, 0);
    return;
  }
  int64_t before = 0, total = 0;
  for (int i = lane; i < p.B; i += 32) {
    const Seq x = seq_of<NT>(p, i);
    const int64_t w = (int64_t)x.units * x.tiles;
    total += w;
    if (i < b) before += w;
  }
#pragma unroll
  for (int w = 1; w < 32; w <<= 1) {
    before += __shfl_xor_sync(0xffffffffu, before, w);
    total += __shfl_xor_sync(0xffffffffu, total, w);
  }
  const int64_t per = stretch(p, total) * kWarps, start = before + (int64_t)u * s.tiles;
  const int c0 = (int)(start / per), c1 = (int)((start + s.tiles - 1) / per);
  if (c0 == c1) return;
  const float* parts = p.parts;
  auto record = [&](int i) { return parts + ((int64_t)i * 2 + (i == c0 ? 1 : 0)) * kRecord<NT>; };
  float top = kFloor;
  for (int i = c0 + lane; i <= c1; i += 32) top = fmaxf(top, __ldcg(record(i) + kCols<NT> * 128 + c));
  top = warp_max(top);
  float l = 0.f;
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i0 = c0; i0 <= c1; i0 += 32) {
    float w = 0.f;
    if (i0 + lane <= c1) {
      w = ex2(__ldcg(record(i0 + lane) + kCols<NT> * 128 + c) - top);
      l += w * __ldcg(record(i0 + lane) + kCols<NT> * 129 + c);
    }
    const int m = min(32, c1 - i0 + 1);
#pragma unroll 4
    for (int j = 0; j < m; ++j) {
      const float f = __shfl_sync(0xffffffffu, w, j);
      const float4 x = __ldcg(reinterpret_cast<const float4*>(record(i0 + j) + c * 128) + lane);
      v.x += x.x * f; v.y += x.y * f; v.z += x.z * f; v.w += x.w * f;
    }
  }
  l = warp_sum(l);
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  *dst = make_uint2(pack_bf16(v.x * inv, v.y * inv), pack_bf16(v.z * inv, v.w * inv));
}

}  // namespace fp4d
