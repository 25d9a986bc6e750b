"""Rows into the 4-bit cache and back, against the format's definition in 64 bits: bit by bit."""
import importlib

import pytest
import torch

import fp4_ref as ref

pytestmark = pytest.mark.gpu
ops = importlib.import_module("nano-vllm-candle_b200.ops")
BF16, F32, F64, I32, U8 = torch.bfloat16, torch.float32, torch.float64, torch.int32, torch.uint8
DEV = "cuda:0"
NAN, INF = float("nan"), float("inf")


def _g(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _cache(blocks, kv, bs, seed=0):
    """A cache full of other bytes."""
    r = lambda w: torch.randint(0, 256, (blocks, kv, bs, w), generator=_g(seed + w), device=DEV, dtype=U8)     # noqa: E731
    return ops.Fp4Cache(r(64), r(8), r(64), r(8))


def _rows(cache, name, slots):
    codes, scales = getattr(cache, name), getattr(cache, name + "_scale")
    s = slots.long()
    return codes[s // cache.block_size, :, s % cache.block_size], scales[s // cache.block_size, :, s % cache.block_size]


def _is(cache, name, slots, rows):
    """The rows at these slots are the 4-bit form of `rows` [N, kv, 128]."""
    codes, scales = _rows(cache, name, slots)
    want, byte = ref.to_fp4(rows)
    assert torch.equal(scales.cpu().long(), byte)
    got = ref.numbers(codes, torch.full_like(scales, 15 * 8))             # scales of one: the codes' own numbers
    fine = (byte != 255)[..., None].expand(*byte.shape, 16).flatten(-2)
    assert torch.equal(torch.where(fine, got, 0.0), torch.where(fine, want, 0.0))


def _slots(n, blocks, bs, seed):
    return torch.randperm(blocks * bs, generator=_g(seed), device=DEV)[:n].to(I32)


def _hard(n, kv):
    """Rows of all sizes, ties among them, and blocks of zeros, of the largest and smallest numbers, of infinities and NaN."""
    x = torch.randn(n, kv, 8, 16, generator=_g(3), device=DEV) * torch.exp2(torch.randint(-30, 20, (n, kv, 8, 1), generator=_g(4), device=DEV).float())
    ties = torch.tensor([6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5, 0], device=DEV)
    x[0::7, :, 0] = ties
    x[1::7, :, 1] = ties * 1.125 * 2 ** -9
    x[2::7, :, 2] = 0
    x[3::7, :, 3, 5] = 3.3e38
    x[4::7, :, 4] = 1e-7
    x[5::7, :, 5, 3] = INF
    x[5::7, :, 6, 15] = -INF
    x[6::7, :, 7, 0] = NAN
    # largest magnitudes whose sixth is half way between two scales
    x[0::7, :, 6] = 0
    x[0::7, :, 6, 2] = 6 * (1 + 1 / 16)
    x[1::7, :, 6] = 0
    x[1::7, :, 6, 2] = -6 * (1 + 3 / 16)
    x[2::7, :, 5] = 0
    x[2::7, :, 5, 9] = 6 * 2.5 * 2.0 ** -17          # below 2^-14: between steps 2 and 3
    return x.flatten(-2).to(BF16)


@pytest.mark.parametrize("n,kv,bs", [(1, 1, 16), (7, 8, 16), (33, 3, 48), (64, 8, 256), (515, 2, 32)])
def test_rows_as_they_are(ctx, n, kv, bs):
    blocks = -(-n // bs) + 2
    cache, slots = _cache(blocks, kv, bs), _slots(n, blocks, bs, 1)
    before = [t.clone() for t in (cache.k, cache.k_scale, cache.v, cache.v_scale)]
    k, v = _hard(n, kv), _hard(n, kv).flip(0)
    wide = torch.full((n, 2 * kv * 128 + 24), NAN, dtype=BF16, device=DEV)
    wide[:, 8:8 + kv * 128], wide[:, 8 + kv * 128:8 + 2 * kv * 128] = k.flatten(1), v.flatten(1)
    ops.store_kvcache_fp4(ctx, wide[:, 8:8 + kv * 128], wide[:, 8 + kv * 128:8 + 2 * kv * 128], cache, slots)
    _is(cache, "k", slots, k)
    _is(cache, "v", slots, v)
    rest = torch.ones(blocks * bs, dtype=torch.bool, device=DEV)
    rest[slots.long()] = False
    rest = torch.nonzero(rest).flatten()
    for t, old in zip((cache.k, cache.k_scale, cache.v, cache.v_scale), before):
        assert torch.equal(t[rest // bs, :, rest % bs], old[rest // bs, :, rest % bs])
    # back: e4m3 numbers and scales, exact
    kq, ks, vq, vs = ops.read_kvcache_fp4(ctx, cache, slots)
    for name, q, s in (("k", kq, ks), ("v", vq, vs)):
        codes, scales = _rows(cache, name, slots)
        assert torch.equal(torch.nan_to_num(ref.numbers(codes, scales), nan=9e9),
                           torch.nan_to_num((q.cpu().to(F64).unflatten(-1, (8, 16)) * s.cpu().to(F64)[..., None]).flatten(-2), nan=9e9))


def test_every_scale_and_code_comes_back(ctx):
    """All 256 scale bytes that a cache may hold, each with all 16 codes."""
    cache = ops.Fp4Cache.zeros(2, 16, 1)
    cache.k_scale.view(-1)[:256] = torch.arange(256, device=DEV, dtype=U8)
    cache.k.view(-1, 8)[:] = torch.tensor([0x10, 0x32, 0x54, 0x76, 0x98, 0xba, 0xdc, 0xfe], dtype=U8, device=DEV)
    slots = torch.arange(32, dtype=I32, device=DEV)
    q, s, _, vs = ops.read_kvcache_fp4(ctx, cache, slots)
    assert torch.equal(q.cpu().to(F64).view(-1, 16)[0], torch.cat((ref.MAGNITUDES, -ref.MAGNITUDES))) and bool((q.view(U8) == q.view(U8).view(-1, 16)[0].repeat(8)).all())
    bits = torch.arange(256, dtype=torch.int16) << 7
    assert torch.equal(torch.nan_to_num(s.cpu().float().flatten(), nan=-1.0), torch.nan_to_num(bits.view(torch.float16).float(), nan=-1.0)) and not vs.any()


def test_slots_that_the_cache_does_not_have(ctx):
    n, kv, bs = 9, 2, 16
    cache = _cache(2, kv, bs)
    before = [t.clone() for t in (cache.k, cache.k_scale, cache.v, cache.v_scale)]
    rows = torch.randn(n, kv * 128, generator=_g(5), device=DEV).to(BF16)
    slots = torch.tensor([-1, 32, 2 ** 31 - 1, -2 ** 31, -5, 33, 1000, 5, -1], dtype=I32, device=DEV)
    ops.store_kvcache_fp4(ctx, rows, rows, cache, slots)
    _is(cache, "k", slots[7:8], rows[7:8].view(1, kv, 128))
    at = torch.tensor([i for i in range(32) if i != 5], device=DEV)
    for t, old in zip((cache.k, cache.k_scale, cache.v, cache.v_scale), before):
        assert torch.equal(t[at // bs, :, at % bs], old[at // bs, :, at % bs])
    k, ks, v, vs = ops.read_kvcache_fp4(ctx, cache, slots)
    for t in (k.view(U8), ks, v.view(U8), vs):
        assert not t[torch.arange(9) != 7].any() and t[7].any()


@pytest.mark.parametrize("n,nh,kv,bs,norm", [(1, 16, 8, 256, True), (3, 5, 1, 16, True), (37, 8, 2, 16, False), (64, 32, 8, 256, True), (259, 40, 8, 32, True)])
def test_norm_rotation_and_store(ctx, n, nh, kv, bs, norm):
    """q and k are those of the kernel with a bf16 cache, bit by bit, and the cache holds the 4-bit form of that one's rows; out of place nothing but q_out is written."""
    blocks = -(-n // bs) + 1
    slots = _slots(n, blocks, bs, 6)
    slots[n // 2:n // 2 + n // 9] = -1
    width = (nh + 2 * kv) * 128
    qkv = (torch.randn(n, width, generator=_g(7), device=DEV) * 3).to(BF16)
    qw, kw = ((torch.randn(128, generator=_g(8 + i), device=DEV) * 0.3 + 1).to(BF16) if norm else None for i in range(2))
    table = ctx.rope_table(1e6, 128, 300)
    pos = torch.randint(0, 300, (n,), generator=_g(10), device=DEV).to(I32)
    kc = torch.zeros(blocks, bs, kv, 128, dtype=BF16, device=DEV)
    vc = torch.zeros_like(kc)
    want = ctx.qk_norm_rope_store(qkv.clone(), qw, kw, 1e-6, table, pos, nh, kv, 128, slots, kc, vc)
    for how in ("in place", "out", "wide"):
        cache = _cache(blocks, kv, bs, 20)
        live = slots[slots >= 0]
        if how == "in place":
            x = qkv.clone()
            assert ops.qk_norm_rope_store_fp4(ctx, x, qw, kw, 1e-6, table, pos, nh, cache, slots) is x
            assert torch.equal(x, want)
        else:
            pad = torch.full((n, width + 8), NAN, dtype=BF16, device=DEV)
            pad[:, :width] = qkv
            x = pad[:, :width] if how == "wide" else qkv.clone()
            q = torch.full((n, nh * 128 + 16), -7.0, dtype=BF16, device=DEV)[:, :nh * 128] if how == "wide" else torch.empty(n, nh * 128, dtype=BF16, device=DEV)
            assert ops.qk_norm_rope_store_fp4(ctx, x, qw, kw, 1e-6, table, pos, nh, cache, slots, q_out=q) is q
            assert torch.equal(x, qkv) and torch.equal(q, want[:, :nh * 128])
            if how == "wide":
                assert bool((q.as_strided((n, 16), (nh * 128 + 16, 1), nh * 128) == -7).all())
        flat = lambda c: c.view(-1, kv, 128)[live.long()]          # noqa: E731
        _is(cache, "k", live, flat(kc))
        _is(cache, "v", live, flat(vc))


def test_positions_that_the_table_does_not_have(ctx):
    """Rows of NaN, not rows of another position."""
    cache, table = ops.Fp4Cache.zeros(1, 16, 1), ctx.rope_table(1e4, 128, 8)
    qkv = torch.ones(4, 3 * 128, dtype=BF16, device=DEV)
    slots, pos = torch.arange(4, dtype=I32, device=DEV), torch.tensor([7, 8, -1, 2 ** 31 - 1], dtype=I32, device=DEV)
    q = ops.qk_norm_rope_store_fp4(ctx, qkv, None, None, 1e-6, table, pos, 1, cache, slots, q_out=torch.empty(4, 128, dtype=BF16, device=DEV))
    assert torch.isfinite(q[0]).all() and torch.isnan(q[1:]).all()
    assert (cache.k_scale[0, 0, 1:4] == 255).all() and (cache.k_scale[0, 0, 0] != 255).all() and (cache.v_scale[0, 0, :4] != 255).all()


def test_slots_far_into_a_long_cache(ctx):
    """Codes beyond 2^32 bytes of the cache."""
    kv, bs, blocks = 8, 256, 36000                       # 4.7 GB of codes a side
    k = torch.empty(blocks, kv, bs, 64, dtype=U8, device=DEV)
    ks = torch.empty(blocks, kv, bs, 8, dtype=U8, device=DEV)
    cache = ops.Fp4Cache(k, ks, torch.empty_like(k), torch.empty_like(ks))
    slots = torch.tensor([blocks * bs - 1, 0, (blocks - 1) * bs, 33000 * bs + 7], dtype=I32, device=DEV)
    rows = torch.randn(4, kv * 128, generator=_g(11), device=DEV).to(BF16)
    ops.store_kvcache_fp4(ctx, rows, rows.flip(0), cache, slots)
    _is(cache, "k", slots, rows.view(4, kv, 128))
    _is(cache, "v", slots, rows.flip(0).view(4, kv, 128))
