"""A workspace of the 4-bit attention that a caller keeps: one for its longest call serves the shorter ones."""
import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu
ops = importlib.import_module("nano-vllm-candle_b200.ops")
BF16, I32, U8 = torch.bfloat16, torch.int32, torch.uint8


@pytest.mark.parametrize("nh,kv", [(8, 8), (16, 8), (12, 4), (32, 8), (40, 5), (64, 4), (65, 1)])
def test_size_does_not_fall(ctx, nh, kv):
    sizes = [ctx.l.nvc_attn_fp4_workspace_bytes(ctx.h, nh, kv, n) for n in (1, 2, 3, 4, 5, 7, 8, 9, 16, 17, 31, 32, 33, 64, 65, 1000, 1 << 20)]
    assert sizes[0] > 0 and sizes == sorted(sizes)


@pytest.mark.parametrize("nh,kv,longest", [(4, 4, 16), (4, 4, 32), (32, 8, 4), (32, 8, 8), (32, 8, 512), (16, 8, 9)])
def test_one_for_the_longest_call_serves_shorter_ones(ctx, nh, kv, longest):
    g = torch.Generator(device="cuda").manual_seed(0)
    bs, lens = 16, [400, 37, longest]
    cache = ops.Fp4Cache.zeros(64, bs, kv)
    ops.store_kvcache_fp4(ctx, *(torch.randn(64 * bs, kv * 128, generator=g, device="cuda").to(BF16) for _ in range(2)), cache, torch.arange(64 * bs, dtype=I32, device="cuda"))
    tables = torch.randint(0, 64, (3, 100), generator=g, device="cuda", dtype=I32)
    context = torch.tensor(lens, dtype=I32, device="cuda")
    size = ctx.l.nvc_attn_fp4_workspace_bytes(ctx.h, nh, kv, longest)
    ws, stream = torch.empty(size, dtype=U8, device="cuda"), torch.cuda.current_stream().cuda_stream
    q = torch.randn(3 * longest, nh * 128, generator=g, device="cuda").to(BF16)
    out = torch.empty_like(q)
    assert ctx.l.nvc_paged_decode_attn_fp4(ctx.h, q.data_ptr(), nh * 128, cache.c, tables.data_ptr(), 100, context.data_ptr(), 3, nh, 0.1, out.data_ptr(), nh * 128, ws.data_ptr(), size, stream) == 0
    assert torch.equal(out[:3], ops.paged_decode_attn_fp4(ctx, q[:3], cache, tables, context, nh, 0.1))
    for n in sorted({1, 2, 3, longest // 2, longest}):
        cu = torch.arange(4, dtype=I32, device="cuda") * n
        assert ctx.l.nvc_prefill_attn_paged_fp4(ctx.h, q.data_ptr(), nh * 128, cache.c, tables.data_ptr(), 100, context.data_ptr(), cu.data_ptr(), 3, 3 * n, n, nh, 0.1, out.data_ptr(), nh * 128,
                                                ws.data_ptr(), size, stream) == 0
        assert torch.equal(out[:3 * n], ops.prefill_attn_paged_fp4(ctx, q[:3 * n], cache, tables, context, cu, n, nh, 0.1))
    assert ctx.l.nvc_paged_decode_attn_fp4(ctx.h, q.data_ptr(), nh * 128, cache.c, tables.data_ptr(), 100, context.data_ptr(), 3, nh, 0.1, out.data_ptr(), nh * 128, ws.data_ptr(), 1024, stream) != 0
