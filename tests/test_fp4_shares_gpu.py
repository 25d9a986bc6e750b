"""What a rank of several does over a 4-bit cache: its share of the heads, alone.  (Ranks meet only behind the attention, in the output projection's sum.)"""
import importlib

import pytest
import torch

import fp4_ref as ref

pytestmark = pytest.mark.gpu
ops = importlib.import_module("nano-vllm-candle_b200.ops")
BF16, F64, I32 = torch.bfloat16, torch.float64, torch.int32


@pytest.mark.parametrize("ranks,nh,kv", [(2, 16, 8), (8, 32, 8), (4, 20, 4)])
def test_a_share_of_the_heads(ctx, ranks, nh, kv):
    """Queries and cached rows of a share are the whole's, bit by bit; its attention is the definition's."""
    g = torch.Generator(device="cuda").manual_seed(0)
    bs, lens, new = 16, [40, 0, 133], [9, 0, 70]
    tables = torch.randperm(24, generator=g, device="cuda").to(I32).view(2, 12)[[0, 0, 1]].contiguous()
    slots = torch.cat([tables[b, torch.arange(n, device="cuda") // bs] * bs + torch.arange(n, device="cuda") % bs for b, n in enumerate(lens)]).to(I32)
    pos = torch.cat([torch.arange(n) for n in lens]).to(I32).cuda()
    q, k, v = (torch.randn(sum(lens), h, 128, generator=g, device="cuda").to(BF16) for h in (nh, kv, kv))
    qw, kw = ((torch.randn(128, generator=g, device="cuda") * 0.2 + 1).to(BF16) for _ in range(2))
    turns = ctx.rope_table(1e4, 128, 256)

    def run(heads, keys):
        cache = ops.Fp4Cache.zeros(24, bs, k[:, keys].shape[1])
        qkv = torch.cat([x.flatten(1) for x in (q[:, heads], k[:, keys], v[:, keys])], 1)
        n = q[:, heads].shape[1]
        out = ops.qk_norm_rope_store_fp4(ctx, qkv, qw, kw, 1e-6, turns, pos, n, cache, slots, q_out=torch.empty(len(pos), n * 128, dtype=BF16, device="cuda"))
        rows = torch.cat([out[a - m:a] for a, m in zip(torch.tensor(lens).cumsum(0).tolist(), new)])
        cu, context = torch.tensor([0] + new).cumsum(0).to(I32).cuda(), torch.tensor(lens, dtype=I32, device="cuda")
        last = torch.cat([out[39:40], out[:1], out[-1:]])
        for got, x, n_new in ((ops.prefill_attn_paged_fp4(ctx, rows, cache, tables, context, cu, max(new), n, 128 ** -0.5), rows, new),
                              (ops.paged_decode_attn_fp4(ctx, last, cache, tables, context, n, 128 ** -0.5), last, [1, 1, 1])):
            want, far = ref.attention(x, cache, tables.cpu(), lens, n_new, 128 ** -0.5, n)
            assert bool(((got.cpu().to(F64).view(want.shape) - want).abs() <= far).all())
        return out.view(-1, n, 128), cache

    whole, cache = run(slice(None), slice(None))
    for r in range(ranks):
        heads, keys = slice(r * nh // ranks, (r + 1) * nh // ranks), slice(r * kv // ranks, (r + 1) * kv // ranks)
        mine, part = run(heads, keys)
        assert torch.equal(mine, whole[:, heads])
        for a, b in ((part.k, cache.k), (part.k_scale, cache.k_scale), (part.v, cache.v), (part.v_scale, cache.v_scale)):
            assert torch.equal(a, b[:, keys])
