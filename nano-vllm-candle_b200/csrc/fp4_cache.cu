// Rows into the 4-bit cache, and back.  nvc_qk_norm_rope_store_fp4 is nvc_qk_norm_rope_store with a cache in 4 bits: q / k RMSNorm, RoPE and the scatter in
// one pass over the QKV rows (src/models/qwen3.rs:206-234); nvc_store_kvcache_fp4 scatters rows that are ready; nvc_read_kvcache_fp4 gives rows back.
#include "fp4.cuh"
#include "internal.h"

#include <algorithm>
#include <type_traits>

namespace {

struct StoreArgs {
  const nvc_bf16 *q, *k, *v;            // heads' rows: q may be absent (nh = 0)
  int64_t ldq, ldk, ldv;
  nvc_bf16 *q_out, *k_out;              // k_out may be null
  int64_t ldqo, ldko;
  uint8_t *kc, *ks, *vc, *vs;
  int kv, block_size, slots;            // slots: of the cache
  const float4* table;                  // null: rows are stored as they are
  int max_pos;
  const uint4 *qw, *kw;                 // null: no norm
  const int32_t *positions, *slot_mapping;
  float eps;
  int N, nh;
};

// 8 lanes per (token, head): lane l owns the numbers [8l, 8l + 8) and [64 + 8l, 64 + 8l + 8), so that a rotation's pairs are one lane's and a block of 16 is two
// neighbouring lanes'.  A warp takes `span` fours of one token's heads (fours of q heads, then of k, then of v heads), so that the token's angles and slot and the norms' weights are read once for
// them.  Per token (nh + 2 kv) * 256 bytes in, nh * 256 (and kv * 256 in place) + kv * 144 out.  Kinds of heads in loops of their own: with one loop for all, the instructions were what bound it (370 a
// four, 95 us for 16 000 tokens of 32 + 16 heads).  Now 275: 80 us, 4.1 TB/s: loads' latency, with a row ahead of 20 warps in flight, 20 KB an SM (2.3 instructions of 4 a
// cycle).
// kTurned: heads are normed and turned.  CTAs of an SM: rows as they are take 58 registers for 96 (in one kernel with the others 16 000 of 8 heads took 30.8 us for 22.6)
template <bool kTurned> constexpr int kStoreCtas = kTurned ? 5 : 8;
template <bool kTurned>
__global__ void __launch_bounds__(128, kStoreCtas<kTurned>) store_fp4_kernel(const StoreArgs p, int span, int warps_per_token) {
  pdl_trigger();
  const int64_t warp = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31, l = lane & 7, sub = lane >> 3;
  const unsigned mask = 0xffu << (lane & ~7);
  const int n = warps_per_token == 1 ? (int)min(warp, (int64_t)p.N) : (int)((uint32_t)warp / (uint32_t)warps_per_token);      // several warps a token: below 2^32 in all
  const int first = warps_per_token == 1 ? 0 : (int)((uint32_t)warp - (uint32_t)n * warps_per_token) * span;
  if (n >= p.N) return;
  // what no kernel of a step writes - slot, position, angles - in front of the wait for the one that writes the rows
  const int slot = p.slot_mapping[n];
  float4 c0, c1, s0, s1;
  c0 = c1 = s0 = s1 = make_float4(0.f, 0.f, 0.f, 0.f);
  const int q_fours = (p.nh + 3) >> 2, kv_fours = (p.kv + 3) >> 2;
  if (kTurned && first < q_fours + kv_fours) {
    const int pos = p.positions[n];
    if ((unsigned)pos < (unsigned)p.max_pos) {
      const float4* cs = p.table + (int64_t)pos * 32;                        // cos[64], sin[64]
      c0 = cs[2 * l]; c1 = cs[2 * l + 1]; s0 = cs[16 + 2 * l]; s1 = cs[16 + 2 * l + 1];
    } else {                                                                  // a position that the table does not have: rows of NaN
      const float bad = __uint_as_float(0x7fffffffu);
      c0 = c1 = s0 = s1 = make_float4(bad, bad, bad, bad);
    }
  }
  const bool stored = (unsigned)slot < (unsigned)p.slots;
  const int block = stored ? slot / p.block_size : 0;
  const int64_t page_row = (int64_t)block * p.kv * p.block_size + (stored ? slot - block * p.block_size : 0);
  // (read behind the wait.  By one CTA: asked for by all, they cost 512 tokens 8.4 us for 7.0)
  if (kTurned && p.qw && blockIdx.x == 0 && threadIdx.x < 4) fp4_prefetch((lane < 2 ? p.qw : p.kw) + 8 * (lane & 1));
  pdl_wait();

  // heads 4 * i + sub of one kind, i from `from` to `to`; the next row on its way while one is worked on
  auto heads = [&](auto kind, const nvc_bf16* src, nvc_bf16* dst, const uint4* w, uint8_t* codes_to, uint8_t* scales_to, int count, int from, int to) {
    constexpr bool kTurn = kTurned && decltype(kind)::value != 2, kStore = decltype(kind)::value != 0;
    if (from >= to) return;
    uint4 w0 = make_uint4(0, 0, 0, 0), w1 = w0;
    if (kTurn && w) { w0 = w[l]; w1 = w[l + 8]; }
    const uint4* row = reinterpret_cast<const uint4*>(src) + (int64_t)(4 * from + sub) * 16 + l;
    uint4* out = reinterpret_cast<uint4*>(dst) + (int64_t)(4 * from + sub) * 16 + l;
    uint4 a = make_uint4(0, 0, 0, 0), b = a;
    if (4 * from + sub < count) { a = ld_once_u4(row); b = ld_once_u4(row + 8); }
#pragma unroll 2
    for (int i = from; i < to; ++i, out += 64) {
      uint4 x = a, y = b;
      row += 64;
      if (i + 1 < to && 4 * i + 4 + sub < count) { a = ld_once_u4(row); b = ld_once_u4(row + 8); }
      if (4 * i + sub >= count) break;                                       // (a head's eight lanes alike)
      if constexpr (kTurn) {
        uint4 o1, o2;
        qk_norm_rope8(x, y, mask, w != nullptr, w0, w1, p.eps, c0, c1, s0, s1, o1, o2);
        x = o1;
        y = o2;
        if (dst) {
          out[0] = x;
          out[8] = y;
        }
      }
      if (kStore) {
        uint32_t ma = fp4_amax8(x), mb = fp4_amax8(y);
        ma = max(ma, __shfl_xor_sync(mask, ma, 1));
        mb = max(mb, __shfl_xor_sync(mask, mb, 1));
        const uint32_t sa = fp4_scale_byte(ma), sb = fp4_scale_byte(mb);
        if (stored) {
          const int64_t at = page_row + (int64_t)(4 * i + sub) * p.block_size;
          uint32_t* codes = reinterpret_cast<uint32_t*>(codes_to + at * kFp4Codes);
          uint8_t* scales = scales_to + at * kFp4Scales;
          codes[l] = sa == 255u ? 0u : fp4_codes8(x, fp4_inverse(sa));
          codes[l + 8] = sb == 255u ? 0u : fp4_codes8(y, fp4_inverse(sb));
          if (!(l & 1)) {
            scales[l >> 1] = (uint8_t)sa;
            scales[4 + (l >> 1)] = (uint8_t)sb;
          }
        }
      }
    }
  };
  const int last = first + span;
  const nvc_bf16* none = nullptr;
  if (kTurned) heads(std::integral_constant<int, 0>(), p.nh ? p.q + n * p.ldq : none, p.nh ? p.q_out + n * p.ldqo : nullptr, p.qw, nullptr, nullptr, p.nh, first, min(last, q_fours));
  heads(std::integral_constant<int, 1>(), p.k + n * p.ldk, p.k_out ? p.k_out + n * p.ldko : nullptr, p.kw, p.kc, p.ks, p.kv, max(first - q_fours, 0), min(last - q_fours, kv_fours));
  heads(std::integral_constant<int, 2>(), p.v + n * p.ldv, nullptr, nullptr, p.vc, p.vs, p.kv, max(first - q_fours - kv_fours, 0), min(last - q_fours - kv_fours, kv_fours));
}

__device__ __forceinline__ uint32_t prmt_signs(uint32_t x, uint32_t selector) {
  uint32_t d;
  asm("prmt.b32 %0, %1, %1, %2;" : "=r"(d) : "r"(x), "r"(selector));
  return d;
}
// 8 lanes per (row, head), 16 numbers of K and of V a lane.  288 bytes out for 144 in.  16 000 tokens of 8 heads: 12.5 us for 8.6 of bytes, a lane's one slot, row and store behind one another (1.45
// instructions of 4 a cycle, memory at 18 %); a side for 8 lanes, with divisions in 64 bits: 19 us
__global__ void __launch_bounds__(256)
read_fp4_kernel(const uint8_t* kc, const uint8_t* ks, const uint8_t* vc, const uint8_t* vs, int kv, int block_size, Fp4Div by_heads, Fp4Div by_block, int slots, const int32_t* slot_list,
                uint4* k, nvc_bf16* k_scale, uint4* v, nvc_bf16* v_scale, int units) {
  pdl_trigger();
  const int unit = (int)(blockIdx.x * 32 + (threadIdx.x >> 3)), l = threadIdx.x & 7;          // (below 2^31 + 32)
  pdl_wait();
  if ((unsigned)unit >= (unsigned)units) return;
  const int n = by_heads(unit), h = unit - n * kv;
  const int slot = slot_list[n];
  uint2 a = make_uint2(0, 0), b = a;
  uint32_t sa = 0, sb = 0;
  if ((unsigned)slot < (unsigned)slots) {
    const int block = by_block(slot);
    const int64_t at = (((int64_t)block * kv + h) * block_size + (slot - block * block_size)) * 8 + l;
    a = reinterpret_cast<const uint2*>(kc)[at];
    b = reinterpret_cast<const uint2*>(vc)[at];
    sa = ks[at];
    sb = vs[at];
  }
  // four codes -> four e4m3 bytes: the magnitudes 0, 0.5, 1, 1.5 and 2, 3, 4, 6 by their place; of a byte 0x80, a code with its sign takes 0xff (the sign eight times)
  auto e4m3 = [](uint32_t c) { return __byte_perm(0x3c383000u, 0x4c484440u, c & 0x7777u) | (prmt_signs(0x80808080u, c) << 1 & 0x80808080u); };
  auto four = [&](uint2 c) { return make_uint4(e4m3(c.x), e4m3(c.x >> 16), e4m3(c.y), e4m3(c.y >> 16)); };
  const int64_t to = (int64_t)unit * 8 + l;
  k[to] = four(a);
  v[to] = four(b);
  k_scale[to] = __bfloat16_as_ushort(__float2bfloat16_rn(fp4_scale(sa)));
  v_scale[to] = __bfloat16_as_ushort(__float2bfloat16_rn(fp4_scale(sb)));
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

int launch_store(nvc_ctx* ctx, const StoreArgs& p, void* stream) {
  // few tokens: their heads over many warps, as long as all run at once; many: all heads of a token in one (2 048 tokens of 32 + 16 heads, us: 12 fours a warp 14.5, 6 16.4, 4 18.4; 1 024: 12.3, 10.2,
  // 12.2; 512: 12.3, 8.3, 8.1, and 3 6.8)
  const int fours = (p.nh + 3) / 4 + 2 * ((p.kv + 3) / 4);
  const int64_t room = (int64_t)ctx->num_sms * 4 * (p.table ? kStoreCtas<true> : kStoreCtas<false>);
  const int most = (int)std::max<int64_t>(1, std::min<int64_t>(fours, room / p.N)), span = (fours + most - 1) / most, per_token = (fours + span - 1) / span;
  const int64_t blocks = ((int64_t)p.N * per_token + 3) / 4;
  NVC_REQUIRE(ctx, blocks <= 0x7fffffffLL, NVC_ESHAPE, "too many rows");
  DeviceGuard guard(ctx->device);
  NVC_CUDA_CHECK(ctx, nvc_launch(ctx, p.table ? store_fp4_kernel<true> : store_fp4_kernel<false>, dim3((unsigned)blocks), dim3(128), 0, nvc_stream(stream), p, span, per_token));
  NVC_CUDA_CHECK(ctx, cudaGetLastError());
  ctx->launches++;
  return NVC_OK;
}

}  // namespace

int nvc_fp4_cache_check(nvc_ctx* ctx, const nvc_fp4_cache* c) {
  NVC_REQUIRE(ctx, ctx && c && c->k && c->k_scale && c->v && c->v_scale, NVC_EINVAL, "null pointer");
  NVC_REQUIRE(ctx, c->num_blocks > 0 && c->kv > 0 && c->block_size > 0, NVC_EINVAL, "bad sizes of the cache");
  NVC_REQUIRE(ctx, c->block_size % 16 == 0, NVC_ESHAPE, "block_size must be a multiple of 16");
  NVC_REQUIRE(ctx, (int64_t)c->num_blocks * c->block_size <= 0x7fffffffLL, NVC_ESHAPE, "a cache has at most 2^31 - 1 slots");
  NVC_REQUIRE(ctx, (int64_t)c->num_blocks * (c->block_size / 16) * c->kv <= 0xffffffffLL, NVC_ESHAPE, "a cache has at most 2^36 rows");
  NVC_REQUIRE(ctx, aligned16(c->k) && aligned16(c->k_scale) && aligned16(c->v) && aligned16(c->v_scale), NVC_EINVAL, "the cache's parts must be 16-byte aligned");
  return NVC_OK;
}

extern "C" int nvc_qk_norm_rope_store_fp4(nvc_ctx* ctx, nvc_bf16* qkv, int ld, const nvc_bf16* qw, const nvc_bf16* kw, float eps, const float* cos_sin, int max_pos,
                                          const int32_t* positions, const int32_t* slot_mapping, const nvc_fp4_cache* cache, nvc_bf16* q_out, int ldqo, int N, int nh, void* stream) {
  if (const int rc = nvc_fp4_cache_check(ctx, cache)) return rc;
  const int kv = cache->kv;
  NVC_REQUIRE(ctx, qkv && cos_sin && positions && slot_mapping, NVC_EINVAL, "null pointer");
  NVC_REQUIRE(ctx, (qw == nullptr) == (kw == nullptr), NVC_EINVAL, "q/k norm weights must both be given or both be NULL");
  NVC_REQUIRE(ctx, N >= 0 && nh > 0 && max_pos > 0 && nh <= 0xffffff && kv <= 0xffffff, NVC_EINVAL, "bad sizes");
  NVC_REQUIRE(ctx, ld >= ((int64_t)nh + 2 * kv) * 128 && ld % 8 == 0 && (!q_out || (ldqo >= (int64_t)nh * 128 && ldqo % 8 == 0)), NVC_ESHAPE,
              "row strides must cover the heads and be multiples of 8");
  NVC_REQUIRE(ctx, aligned16(qkv) && aligned16(qw) && aligned16(kw) && aligned16(cos_sin) && aligned16(q_out), NVC_EINVAL, "pointers must be 16-byte aligned");
  if (N == 0) return NVC_OK;
  StoreArgs p{};
  p.q = qkv; p.k = qkv + (int64_t)nh * 128; p.v = qkv + ((int64_t)nh + kv) * 128;
  p.ldq = p.ldk = p.ldv = ld;
  p.q_out = q_out ? q_out : qkv;
  p.ldqo = q_out ? ldqo : ld;
  p.k_out = q_out ? nullptr : qkv + (int64_t)nh * 128;
  p.ldko = ld;
  p.kc = cache->k; p.ks = cache->k_scale; p.vc = cache->v; p.vs = cache->v_scale;
  p.kv = kv; p.block_size = cache->block_size; p.slots = cache->num_blocks * cache->block_size;
  p.table = reinterpret_cast<const float4*>(cos_sin); p.max_pos = max_pos;
  p.qw = reinterpret_cast<const uint4*>(qw); p.kw = reinterpret_cast<const uint4*>(kw);
  p.positions = positions; p.slot_mapping = slot_mapping; p.eps = eps; p.N = N; p.nh = nh;
  return launch_store(ctx, p, stream);
}

extern "C" int nvc_store_kvcache_fp4(nvc_ctx* ctx, const nvc_bf16* k, int ldk, const nvc_bf16* v, int ldv, const nvc_fp4_cache* cache, const int32_t* slot_mapping, int N,
                                     void* stream) {
  if (const int rc = nvc_fp4_cache_check(ctx, cache)) return rc;
  NVC_REQUIRE(ctx, k && v && slot_mapping, NVC_EINVAL, "null pointer");
  NVC_REQUIRE(ctx, N >= 0 && cache->kv <= 0xffffff, NVC_EINVAL, "bad sizes");
  NVC_REQUIRE(ctx, ldk >= (int64_t)cache->kv * 128 && ldv >= (int64_t)cache->kv * 128 && ldk % 8 == 0 && ldv % 8 == 0, NVC_ESHAPE,
              "row strides must cover the heads and be multiples of 8");
  NVC_REQUIRE(ctx, aligned16(k) && aligned16(v), NVC_EINVAL, "pointers must be 16-byte aligned");
  if (N == 0) return NVC_OK;
  StoreArgs p{};
  p.k = k; p.v = v; p.ldk = ldk; p.ldv = ldv;
  p.kc = cache->k; p.ks = cache->k_scale; p.vc = cache->v; p.vs = cache->v_scale;
  p.kv = cache->kv; p.block_size = cache->block_size; p.slots = cache->num_blocks * cache->block_size;
  p.slot_mapping = slot_mapping; p.N = N;
  return launch_store(ctx, p, stream);
}

extern "C" int nvc_read_kvcache_fp4(nvc_ctx* ctx, const nvc_fp4_cache* cache, const int32_t* slots, nvc_fp8* k, nvc_bf16* k_scale, nvc_fp8* v, nvc_bf16* v_scale, int N,
                                    void* stream) {
  if (const int rc = nvc_fp4_cache_check(ctx, cache)) return rc;
  NVC_REQUIRE(ctx, slots && k && k_scale && v && v_scale, NVC_EINVAL, "null pointer");
  NVC_REQUIRE(ctx, N >= 0 && cache->kv <= 0xffffff, NVC_EINVAL, "bad sizes");
  NVC_REQUIRE(ctx, aligned16(k) && aligned16(v), NVC_EINVAL, "pointers must be 16-byte aligned");
  if (N == 0) return NVC_OK;
  const int64_t units = (int64_t)N * cache->kv, blocks = (units + 31) / 32;
  NVC_REQUIRE(ctx, units <= 0x7fffffffLL, NVC_ESHAPE, "too many rows");
  DeviceGuard guard(ctx->device);
  NVC_CUDA_CHECK(ctx, nvc_launch(ctx, read_fp4_kernel, dim3((unsigned)blocks), dim3(256), 0, nvc_stream(stream), cache->k, cache->k_scale, cache->v, cache->v_scale, cache->kv,
                                 cache->block_size, fp4_div(cache->kv), fp4_div(cache->block_size), cache->num_blocks * cache->block_size, slots, reinterpret_cast<uint4*>(k), k_scale,
                                 reinterpret_cast<uint4*>(v), v_scale, (int)units));
  NVC_CUDA_CHECK(ctx, cudaGetLastError());
  ctx->launches++;
  return NVC_OK;
}
