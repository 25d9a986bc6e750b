// Attention over the 4-bit paged cache: decode (one new row of each sequence) and prompt portions (the last rows of each context, causal).
// FLOPs: 4 * 128 for every (query head, visible key); bytes: 144 for every (key head, cached token), 512 for every query head's row and its result.
#include "fp4_decode.cuh"
#include "fp4_prefill.cuh"
#include "internal.h"

#include <algorithm>

#include <cmath>

namespace {

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

template <int NT> int64_t parts_bytes(const nvc_ctx* ctx) { return (int64_t)ctx->num_sms * fp4d::kCtas<NT> * (16 + 2 * fp4d::kRecord<NT> * 4); }

constexpr int kMostAlone = 65535;          // CTAs

template <int NT>
int launch_few(nvc_ctx* ctx, fp4d::Args& p, int64_t most_rows, int blocks, cudaStream_t stream, size_t workspace_bytes) {
  const int64_t units = p.kv * ((most_rows + fp4d::kCols<NT> - 1) / fp4d::kCols<NT>);          // of a sequence, at most
  const int64_t tiles = ((int64_t)blocks * p.block_size + fp4d::kTile - 1) / fp4d::kTile;        // of a sequence, at most (a hint that is too low costs time alone)
  // units at most by max_seqlen_q, and whatever cu_seqlens say
  const int64_t room = p.cu_seqlens ? p.kv * ((int64_t)p.rows * p.group / fp4d::kCols<NT> + p.B) : units * p.B;
  const bool alone = fp4d::alone<NT>(ctx->num_sms, std::min(units * p.B, room), tiles) && room <= kMostAlone;
  const int64_t most = units * p.B * (tiles + fp4d::kUnitCost);      // the list's length, at most
  const int64_t a_cta = (1 + fp4d::kUnitCost) * fp4d::kWarps;
  const int grid = alone ? (int)room : (int)std::min<int64_t>((int64_t)ctx->num_sms * fp4d::kCtas<NT>, (most + a_cta - 1) / a_cta);
  NVC_REQUIRE(ctx, p.notes && ((uintptr_t)p.notes & 15) == 0 && workspace_bytes >= (size_t)parts_bytes<NT>(ctx), NVC_ENOMEM, "workspace too small");
  p.parts = reinterpret_cast<float*>(p.notes + grid);
  p.warps = grid * fp4d::kWarps;
  p.alone = alone ? (int)units : 0;
  NVC_CUDA_CHECK(ctx, nvc_launch(ctx, p.cu_seqlens ? fp4d::attn_kernel<NT, true> : fp4d::attn_kernel<NT, false>, dim3(grid), dim3(32 * fp4d::kWarps), (size_t)fp4d::kSmem<NT>, stream, p));
  if (!alone) NVC_CUDA_CHECK(ctx, nvc_launch(ctx, fp4d::combine_kernel<NT>, dim3(grid), dim3(32 * fp4d::kCols<NT>), 0, stream, p));
  NVC_CUDA_CHECK(ctx, cudaGetLastError());
  ctx->launches += alone ? 1 : 2;
  return NVC_OK;
}

// Rows of a sequence and key head up to which the kernel for few rows takes them, in passes of 16: 32, and 64 where the portions' kernel would have few CTAs with work (us, few / portions; 32 rows: 32
// sequences behind 1 750 50 / 62, 64 of 300 35 / 42; 48: 70 / 63, 42 / 43, 8 behind 16 000 123 / 110; 64: 88 / 65, 49 / 44, 160 / 111, 4 behind 2 000 25 / 27, one behind 16 000 33 / 39)
constexpr int kFewRows = 32, kFewRowsOfFew = 64;
int64_t most_rows_of(int rows, int max_qlen, int group) { return std::min(rows, max_qlen) * (int64_t)group; }
size_t many_bytes(const nvc_ctx* ctx) { return (size_t)ctx->num_sms * (16 + 2 * fp4p::kRecord * 4); }

int launch_many(nvc_ctx* ctx, const fp4d::Args& f, int64_t most_rows, float scale, cudaStream_t stream, size_t workspace_bytes) {
  NVC_REQUIRE(ctx, f.notes && ((uintptr_t)f.notes & 15) == 0 && workspace_bytes >= many_bytes(ctx), NVC_ENOMEM, "workspace too small");
  // A unit for each CTA where all of them run at once, by max_seqlen_q; the grid has room for whatever cu_seqlens say
  const int64_t room = f.kv * ((int64_t)f.rows * f.group / fp4p::kRows + f.B), tiles = ((int64_t)f.bt_stride * f.block_size + fp4p::kKT - 1) / fp4p::kKT;          // units at most; tiles of one
  const int64_t units = std::min(room, f.kv * (int64_t)f.B * ((most_rows + fp4p::kRows - 1) / fp4p::kRows));
  const bool alone = units <= ctx->num_sms && room <= kMostAlone && tiles <= fp4p::kAloneTiles;
  const int grid = alone ? (int)room : ctx->num_sms;
  const fp4p::Args p{f.q, f.out, f.ldq, f.ldo, f.kc, f.ks, f.vc, f.vs, f.block_tables, f.context_lens, f.cu_seqlens, f.bt_stride, f.num_blocks, f.kv, f.block_size, f.B, f.group,
                     f.rows, fp4_div(f.group), fp4_div(f.block_size), scale > 0.f ? 1.f : scale < 0.f ? -1.f : 0.f,
                     scale == 0.f ? 1.f : std::fabs(scale) * 1.4426950408889634f, f.notes, reinterpret_cast<float*>(f.notes + grid), alone};
  NVC_CUDA_CHECK(ctx, nvc_launch(ctx, fp4p::attn_kernel, dim3(grid), dim3(fp4p::kThreads), (size_t)fp4p::kSmemBytes, stream, p));
  if (!alone) NVC_CUDA_CHECK(ctx, nvc_launch(ctx, fp4p::combine_kernel, dim3(grid * 8), dim3(256), 0, stream, p));
  NVC_CUDA_CHECK(ctx, cudaGetLastError());
  ctx->launches += alone ? 1 : 2;
  return NVC_OK;
}

int attn_fp4(nvc_ctx* ctx, const nvc_bf16* q, int ldq, const nvc_fp4_cache* cache, const int32_t* block_tables, int bt_stride, int blocks, const int32_t* context_lens,
             const int32_t* cu_seqlens_q, int B, int rows, int max_qlen, int nh, float scale, nvc_bf16* out, int ldo, void* workspace, size_t workspace_bytes, void* stream) {
  if (const int rc = nvc_fp4_cache_check(ctx, cache)) return rc;
  NVC_REQUIRE(ctx, q && block_tables && context_lens && out, NVC_EINVAL, "null pointer");
  NVC_REQUIRE(ctx, B >= 0 && rows >= 0 && max_qlen >= 0 && nh > 0 && bt_stride > 0, NVC_EINVAL, "bad sizes");
  NVC_REQUIRE(ctx, nh % cache->kv == 0, NVC_ESHAPE, "nh must be a multiple of kv");
  NVC_REQUIRE(ctx, ldq % 8 == 0 && ldq >= (int64_t)nh * 128 && ldo % 8 == 0 && ldo >= (int64_t)nh * 128, NVC_ESHAPE, "row strides must cover the heads and be multiples of 8");
  NVC_REQUIRE(ctx, aligned16(q) && aligned16(out), NVC_EINVAL, "pointers must be 16-byte aligned");
  NVC_REQUIRE(ctx, std::isfinite(scale), NVC_EINVAL, "the scale must be finite");
  if (B == 0 || rows == 0 || max_qlen == 0) return NVC_OK;
  const int group = nh / cache->kv;
  const int64_t most_rows = most_rows_of(rows, max_qlen, group);             // of a sequence and key head
  NVC_REQUIRE(ctx, (int64_t)rows * group <= 0x7fffffffLL, NVC_ESHAPE, "too many rows");
  fp4d::Args p{q, out, ldq, ldo, cache->k, cache->k_scale, cache->v, cache->v_scale, block_tables, context_lens, cu_seqlens_q, bt_stride, cache->num_blocks, cache->kv,
               cache->block_size, B, group, rows, scale * 1.4426950408889634f, static_cast<int4*>(workspace), nullptr, 0, 0};
  DeviceGuard guard(ctx->device);
  const int few = (int64_t)B * cache->kv <= ctx->num_sms / 4 ? kFewRowsOfFew : kFewRows;
  if (cu_seqlens_q && most_rows > few) return launch_many(ctx, p, most_rows, scale, nvc_stream(stream), workspace_bytes);
  return most_rows <= 8 ? launch_few<1>(ctx, p, most_rows, blocks, nvc_stream(stream), workspace_bytes) : launch_few<2>(ctx, p, most_rows, blocks, nvc_stream(stream), workspace_bytes);
}

}  // namespace

extern "C" int nvc_fp4_attn_init(nvc_ctx* ctx) {
  for (auto kernel : {fp4d::attn_kernel<1, false>, fp4d::attn_kernel<1, true>}) NVC_CUDA_CHECK(ctx, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, fp4d::kSmem<1>));
  for (auto kernel : {fp4d::attn_kernel<2, false>, fp4d::attn_kernel<2, true>}) NVC_CUDA_CHECK(ctx, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, fp4d::kSmem<2>));
  NVC_CUDA_CHECK(ctx, cudaFuncSetAttribute(fp4p::attn_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, fp4p::kSmemBytes));
  return NVC_OK;
}

extern "C" size_t nvc_attn_fp4_workspace_bytes(const nvc_ctx* ctx, int nh, int kv, int max_seqlen_q) {
  if (!ctx || nh <= 0 || kv <= 0 || max_seqlen_q <= 0) return 0;
  const int64_t rows = most_rows_of(max_seqlen_q, max_seqlen_q, (nh + kv - 1) / kv);
  const size_t few = (size_t)std::max(parts_bytes<1>(ctx), parts_bytes<2>(ctx));          // of either, so that a longer call's serves a shorter one
  return rows > kFewRows ? std::max(few, many_bytes(ctx)) : few;
}

extern "C" int nvc_paged_decode_attn_fp4(nvc_ctx* ctx, const nvc_bf16* q, int ldq, const nvc_fp4_cache* cache, const int32_t* block_tables, int bt_stride,
                                         const int32_t* context_lens, int B, int nh, float scale, nvc_bf16* out, int ldo, void* workspace, size_t workspace_bytes, void* stream) {
  return attn_fp4(ctx, q, ldq, cache, block_tables, bt_stride, bt_stride, context_lens, nullptr, B, B, 1, nh, scale, out, ldo, workspace, workspace_bytes, stream);
}

extern "C" int nvc_paged_decode_attn_fp4_ex(nvc_ctx* ctx, const nvc_bf16* q, int ldq, const nvc_fp4_cache* cache, const int32_t* block_tables, int bt_stride, int max_blocks_hint,
                                            const int32_t* context_lens, int B, int nh, float scale, nvc_bf16* out, int ldo, void* workspace, size_t workspace_bytes, void* stream) {
  const int blocks = max_blocks_hint > 0 ? std::min(max_blocks_hint, bt_stride) : bt_stride;
  return attn_fp4(ctx, q, ldq, cache, block_tables, bt_stride, blocks, context_lens, nullptr, B, B, 1, nh, scale, out, ldo, workspace, workspace_bytes, stream);
}

extern "C" int nvc_prefill_attn_paged_fp4(nvc_ctx* ctx, const nvc_bf16* q, int ldq, const nvc_fp4_cache* cache, const int32_t* block_tables, int bt_stride,
                                          const int32_t* context_lens, const int32_t* cu_seqlens_q, int B, int total_q_tokens, int max_seqlen_q, int nh, float scale, nvc_bf16* out,
                                          int ldo, void* workspace, size_t workspace_bytes, void* stream) {
  NVC_REQUIRE(ctx, ctx && cu_seqlens_q, NVC_EINVAL, "null pointer");
  return attn_fp4(ctx, q, ldq, cache, block_tables, bt_stride, bt_stride, context_lens, cu_seqlens_q, B, total_q_tokens, max_seqlen_q, nh, scale, out, ldo, workspace, workspace_bytes, stream);
}
