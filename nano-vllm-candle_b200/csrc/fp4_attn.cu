// Attention over the 4-bit paged cache: decode (one new row of each sequence) and prompt portions (the last rows of each context, causal).
// FLOPs: 4 * 128 for every (query head, visible key); bytes: 144 for every (key head, cached token), 512 for every query head's row and its result.
#include "fp4.cuh"
#include "internal.h"

#include <cmath>

namespace {

struct AttnArgs {
  const nvc_bf16* q;
  int64_t ldq, ldo;
  nvc_bf16* out;
  const uint8_t *kc, *ks, *vc, *vs;
  int num_blocks, kv, block_size;
  const int32_t *block_tables, *context_lens, *cu_seqlens;      // cu_seqlens null: one row of each sequence
  int bt_stride, B, rows, max_qlen, group;
  float scale_log2e;
};

// One CTA per (row, key head, 8 query heads): 16 cached tokens at a time, decoded into shared memory as fp32.
__global__ void __launch_bounds__(128) attn_fp4_plain_kernel(const AttnArgs p) {
  pdl_trigger();
  __shared__ float qs[8][128], ksm[16][129], vsm[16][128], ps[8][16], al[8];
  const int row = blockIdx.x, kvh = blockIdx.y, h0 = blockIdx.z * 8, tid = threadIdx.x;
  const int G = min(8, p.group - h0);
  pdl_wait();
  int b = row, qlen = 1, i = 0;
  if (p.cu_seqlens) {
    int lo = 0, hi = p.B;                                        // the last sequence that begins at or in front of the row and has rows
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (p.cu_seqlens[mid + 1] <= row) lo = mid + 1;
      else hi = mid;
    }
    if (lo >= p.B) return;                                       // behind the last sequence: left as it is
    b = lo;
    i = row - p.cu_seqlens[b];
    qlen = p.cu_seqlens[b + 1] - p.cu_seqlens[b];
    if (i < 0) return;
  }
  const int len = min(max(p.context_lens[b], 0), (int)min((int64_t)0x7fffffff, (int64_t)p.bt_stride * p.block_size));
  const int seen = max(0, len - qlen + i + 1);
  const int head = kvh * p.group + h0;
  for (int h = 0; h < G; ++h) qs[h][tid] = __uint_as_float((uint32_t)p.q[row * p.ldq + (int64_t)(head + h) * 128 + tid] << 16);
  float o[8] = {}, m = -INFINITY, l = 0.f;                       // m, l: of head tid / 16
  for (int t0 = 0; t0 < seen; t0 += 16) {
    const int blk = p.block_tables[(int64_t)b * p.bt_stride + t0 / p.block_size];
    const bool there = (unsigned)blk < (unsigned)p.num_blocks;
    const int64_t at = ((int64_t)(there ? blk : 0) * p.kv + kvh) * p.block_size + t0 % p.block_size;
    __syncthreads();
    {
      const int t = tid >> 3, c = tid & 7;                       // token, block of 16 numbers
      const bool live = there && t0 + t < seen;
      for (int side = 0; side < 2; ++side) {
        const uint2 w = live ? reinterpret_cast<const uint2*>((side ? p.vc : p.kc) + (at + t) * kFp4Codes)[c] : make_uint2(0, 0);
        const float s = fp4_scale(live ? ((side ? p.vs : p.ks) + (at + t) * kFp4Scales)[c] : 0);
        float* to = side ? &vsm[t][16 * c] : &ksm[t][16 * c];
        const uint4 x = fp4_halves8(w.x), y = fp4_halves8(w.y);
        const uint32_t f[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
        for (int j = 0; j < 8; ++j) {
          const float2 two = __half22float2(*reinterpret_cast<const __half2*>(&f[j]));
          to[2 * j] = two.x * s;
          to[2 * j + 1] = two.y * s;
        }
      }
    }
    __syncthreads();
    const int h = tid >> 4, t = tid & 15;
    float x = 0.f;
    if (h < G)
      for (int d = 0; d < 128; ++d) x += qs[h][d] * ksm[t][d];
    x = t0 + t < seen ? x * p.scale_log2e : -INFINITY;
    float top = x;
    for (int w = 1; w < 16; w <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
    const float mn = fmaxf(m, top), ref = mn == -INFINITY ? 0.f : mn;
    const float a = exp2f(m - ref), e = x == -INFINITY ? 0.f : exp2f(x - ref);
    float sum = e;
    for (int w = 1; w < 16; w <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
    l = l * a + sum;
    m = mn;
    ps[h][t] = e;
    if (t == 0) al[h] = a;
    __syncthreads();
    for (int g = 0; g < G; ++g) {
      o[g] *= al[g];
      for (int j = 0; j < 16; ++j) o[g] += ps[g][j] * vsm[j][tid];
    }
  }
  __syncthreads();
  if ((tid & 15) == 0) al[tid >> 4] = l;
  __syncthreads();
  for (int g = 0; g < G; ++g)
    p.out[row * p.ldo + (int64_t)(head + g) * 128 + tid] = __bfloat16_as_ushort(__float2bfloat16_rn(seen ? o[g] / al[g] : 0.f));
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

int attn_fp4(nvc_ctx* ctx, const nvc_bf16* q, int ldq, const nvc_fp4_cache* cache, const int32_t* block_tables, int bt_stride, const int32_t* context_lens,
             const int32_t* cu_seqlens_q, int B, int rows, int max_qlen, int nh, float scale, nvc_bf16* out, int ldo, void* workspace, size_t workspace_bytes, void* stream) {
  if (const int rc = nvc_fp4_cache_check(ctx, cache)) return rc;
  NVC_REQUIRE(ctx, q && block_tables && context_lens && out, NVC_EINVAL, "null pointer");
  NVC_REQUIRE(ctx, B >= 0 && rows >= 0 && max_qlen >= 0 && nh > 0 && bt_stride > 0, NVC_EINVAL, "bad sizes");
  NVC_REQUIRE(ctx, nh % cache->kv == 0, NVC_ESHAPE, "nh must be a multiple of kv");
  NVC_REQUIRE(ctx, ldq % 8 == 0 && ldq >= (int64_t)nh * 128 && ldo % 8 == 0 && ldo >= (int64_t)nh * 128, NVC_ESHAPE, "row strides must cover the heads and be multiples of 8");
  NVC_REQUIRE(ctx, aligned16(q) && aligned16(out), NVC_EINVAL, "pointers must be 16-byte aligned");
  NVC_REQUIRE(ctx, std::isfinite(scale), NVC_EINVAL, "the scale must be finite");
  if (B == 0 || rows == 0 || max_qlen == 0) return NVC_OK;
  const int group = nh / cache->kv, chunks = (group + 7) / 8;
  NVC_REQUIRE(ctx, cache->kv <= 65535 && chunks <= 65535, NVC_ESHAPE, "too many heads");
  AttnArgs p{q, ldq, ldo, out, cache->k, cache->k_scale, cache->v, cache->v_scale, cache->num_blocks, cache->kv, cache->block_size, block_tables, context_lens, cu_seqlens_q,
             bt_stride, B, rows, max_qlen, group, scale * 1.4426950408889634f};
  DeviceGuard guard(ctx->device);
  NVC_CUDA_CHECK(ctx, nvc_launch(ctx, attn_fp4_plain_kernel, dim3(rows, cache->kv, chunks), dim3(128), 0, nvc_stream(stream), p));
  NVC_CUDA_CHECK(ctx, cudaGetLastError());
  ctx->launches++;
  return NVC_OK;
}

}  // namespace

extern "C" size_t nvc_attn_fp4_workspace_bytes(const nvc_ctx* ctx, int nh, int kv) { return 0; }

extern "C" int nvc_paged_decode_attn_fp4(nvc_ctx* ctx, const nvc_bf16* q, int ldq, const nvc_fp4_cache* cache, const int32_t* block_tables, int bt_stride,
                                         const int32_t* context_lens, int B, int nh, float scale, nvc_bf16* out, int ldo, void* workspace, size_t workspace_bytes, void* stream) {
  return attn_fp4(ctx, q, ldq, cache, block_tables, bt_stride, context_lens, nullptr, B, B, 1, nh, scale, out, ldo, workspace, workspace_bytes, stream);
}

extern "C" int nvc_prefill_attn_paged_fp4(nvc_ctx* ctx, const nvc_bf16* q, int ldq, const nvc_fp4_cache* cache, const int32_t* block_tables, int bt_stride,
                                          const int32_t* context_lens, const int32_t* cu_seqlens_q, int B, int total_q_tokens, int max_seqlen_q, int nh, float scale, nvc_bf16* out,
                                          int ldo, void* workspace, size_t workspace_bytes, void* stream) {
  NVC_REQUIRE(ctx, ctx && cu_seqlens_q, NVC_EINVAL, "null pointer");
  return attn_fp4(ctx, q, ldq, cache, block_tables, bt_stride, context_lens, cu_seqlens_q, B, total_q_tokens, max_seqlen_q, nh, scale, out, ldo, workspace, workspace_bytes, stream);
}
