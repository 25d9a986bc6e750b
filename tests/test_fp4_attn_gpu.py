"""Attention over the 4-bit paged cache against the definition in 64 bits; the bounds stand in fp4_ref.attention."""
import importlib

import pytest
import torch

import fp4_ref as ref

pytestmark = pytest.mark.gpu
ops = importlib.import_module("nano-vllm-candle_b200.ops")
BF16, F32, F64, I32, U8 = torch.bfloat16, torch.float32, torch.float64, torch.int32, torch.uint8
DEV = "cuda:0"


def _g(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _case(lens, nh, kv, bs, seed=0, size=1.0, new=None, wide=False):
    """q rows, a cache whose unused rows and pages are NaN, tables with -1 behind a sequence's last page, lengths."""
    new = new or [1] * len(lens)
    per = [-(-max(n, 0) // bs) for n in lens]
    blocks = sum(per) + 2
    order = torch.randperm(blocks, generator=_g(seed + 1), device=DEV)
    cache = ops.Fp4Cache(*(torch.full((blocks, kv, bs, w), 255, dtype=U8, device=DEV) for w in (64, 8, 64, 8)))
    tables = torch.full((len(lens), max(max(per), 1) + 1), -1, dtype=I32)
    at = 0
    for b, n in enumerate(lens):
        tables[b, :per[b]] = order[at:at + per[b]].cpu()
        at += per[b]
    slots = torch.cat([tables[b].repeat_interleave(bs)[:max(n, 0)] * bs + torch.arange(max(n, 0)) % bs for b, n in enumerate(lens)]).to(I32).to(DEV)
    if slots.numel():
        k, v = (torch.randn(slots.numel(), kv * 128, generator=_g(seed + 2 + i), device=DEV) * (size if i == 0 else 1.0) for i in range(2))
        ops.store_kvcache_fp4(CTX[0], k.to(BF16), v.to(BF16), cache, slots)
    rows = sum(new)
    q = torch.randn(rows, nh * 128 + (16 if wide else 0), generator=_g(seed + 4), device=DEV).to(BF16)[:, :nh * 128]
    return dict(q=q, cache=cache, tables=tables.to(DEV), lens=torch.tensor(lens, dtype=I32, device=DEV), cu=torch.tensor([0] + new).cumsum(0).to(I32).to(DEV), new=new, nh=nh)


CTX = [None]


@pytest.fixture(autouse=True)
def _with_ctx(ctx):
    CTX[0] = ctx


def _near(got, c, scale=128 ** -0.5, rows=None):
    want, far = ref.attention(c["q"], c["cache"], c["tables"].cpu(), c["lens"].tolist(), c["new"], scale, c["nh"])
    off = (got.cpu().to(F64).view(want.shape) - want).abs()
    assert torch.isfinite(got).all() and bool((off <= far).all()), f"{float((off / far.clamp_min(1e-300)).max())} times what it may be off"


def _decode(ctx, c, scale=128 ** -0.5, **kw):
    return ops.paged_decode_attn_fp4(ctx, c["q"], c["cache"], c["tables"], c["lens"], c["nh"], scale, **kw)


def _portions(ctx, c, scale=128 ** -0.5, **kw):
    return ops.prefill_attn_paged_fp4(ctx, c["q"], c["cache"], c["tables"], c["lens"], c["cu"], max(c["new"]), c["nh"], scale, **kw)


@pytest.mark.parametrize("lens,nh,kv,bs", [
    ([1], 1, 1, 16), ([16], 2, 1, 16), ([17], 8, 8, 16), ([255, 256, 257], 16, 8, 256), ([1, 0, 33, 700], 32, 8, 48), ([5, 64, 63, 65, 0, 0, 129], 40, 8, 32),
    ([1000, 3], 64, 8, 64), ([90], 12, 1, 16), ([300, 31], 16, 1, 256), ([70, 200], 24, 1, 16), ([100] * 37, 4, 4, 16), ([2500], 8, 1, 256), ([0, 0], 8, 2, 16)])
def test_decode(ctx, lens, nh, kv, bs):
    c = _case(lens, nh, kv, bs, wide=True)
    got = _decode(ctx, c)
    _near(got, c)
    assert not got[[i for i, n in enumerate(lens) if not n]].any()
    assert torch.equal(got, _decode(ctx, c))                            # bit by bit


@pytest.mark.parametrize("size,scale", [(0.01, 1.0), (30.0, 128 ** -0.5), (1.0, -0.1), (1.0, 0.0), (300.0, 1.0)])
def test_decode_of_flat_and_peaked_rows(ctx, size, scale):
    c = _case([1, 77, 640], 8, 2, 16, seed=9, size=size)
    _near(_decode(ctx, c, scale), c, scale)


@pytest.mark.parametrize("size", [2.0 ** -60, 2.0 ** -20, 2.0 ** 15, 2.0 ** 60])
def test_decode_of_queries_of_any_size(ctx, size):
    """Queries beyond what fp16 holds."""
    c = _case([50, 3], 8, 2, 16, seed=12)
    c["q"] = (c["q"].float() * size).to(BF16)
    _near(_decode(ctx, c, 128 ** -0.5 / size), c, 128 ** -0.5 / size)


@pytest.mark.parametrize("new,before,nh,kv,bs", [
    ([1], [0], 4, 2, 16), ([5], [0], 8, 8, 16), ([3, 1, 8], [0, 40, 500], 32, 8, 256), ([17, 2], [1, 200], 8, 1, 48), ([128], [0], 4, 2, 32), ([129, 1, 64], [31, 700, 0], 16, 4, 16),
    ([70], [333], 40, 8, 16), ([260, 9], [5, 77], 4, 1, 128), ([1] * 40, list(range(0, 200, 5)), 8, 8, 16), ([33], [64], 12, 1, 64), ([64, 0, 65], [0, 9, 1], 8, 2, 16)])
def test_portions(ctx, new, before, nh, kv, bs):
    c = _case([n + b for n, b in zip(new, before)], nh, kv, bs, new=new, wide=True)
    got = _portions(ctx, c)
    _near(got, c)
    assert torch.equal(got, _portions(ctx, c))


def test_portions_longer_than_their_context(ctx):
    """Rows in front of the context's first token see nothing: zeros."""
    c = _case([3, 0, 40], 4, 2, 16, new=[7, 2, 40], seed=3)
    got = _portions(ctx, c)
    _near(got, c)
    assert not got[:4].any() and not got[7:9].any()


def test_rows_behind_the_last_sequence_and_columns_beside_the_heads_stay(ctx):
    c = _case([20, 9], 8, 2, 16, new=[4, 2], seed=5)
    c["q"] = torch.cat((c["q"], torch.randn(5, 8 * 128, generator=_g(1), device=DEV).to(BF16)))
    out = torch.full((11, 8 * 128 + 32), 3.0, dtype=BF16, device=DEV)
    assert _portions(ctx, c, out=out[:, :8 * 128]).data_ptr() == out.data_ptr()
    assert bool((out[6:] == 3).all()) and bool((out[:, 8 * 128:] == 3).all())
    c["q"] = c["q"][:6]
    _near(out[:6, :8 * 128], c)
    d = _case([20, 0], 8, 2, 16, seed=6)
    wide = torch.full((2, 8 * 128 + 8), 3.0, dtype=BF16, device=DEV)
    _decode(ctx, d, out=wide[:, :8 * 128])
    assert bool((wide[:, 8 * 128:] == 3).all()) and not wide[1, :8 * 128].any()
    _near(wide[:, :8 * 128], d)


def test_pages_outside_the_pool_and_lengths_beyond_the_table(ctx):
    """A page that the pool does not have reads as rows of zeros, a length beyond the table as the table's."""
    for call, new in ((_decode, [1, 1]), (_portions, [2, 3])):
        c = _case([64, 50], 8, 2, 16, new=new, seed=7)
        c["tables"][0, 1], c["tables"][1, 2] = 1 << 28, -7
        c["lens"][0] = 10 ** 6
        c["tables"] = c["tables"][:, :4].contiguous()
        _near(call(ctx, c), c)


def test_numbers_that_are_none(ctx):
    """A NaN in a cached row reaches the heads that read it, and no other; one behind the context reaches nobody (the unused rows of every test here are NaN)."""
    for call, new in ((_decode, [1, 1]), (_portions, [4, 2])):
        c = _case([30, 18], 8, 2, 16, new=new, seed=8)
        clean = call(ctx, c)
        blk = int(c["tables"][1, 0])
        c["cache"].v_scale[blk, 1, 3, 5] = 255
        got = call(ctx, c).view(-1, 8, 128)
        n = new[0]
        assert torch.equal(got[:n], clean.view(-1, 8, 128)[:n]) and torch.equal(got[n:, :4], clean.view(-1, 8, 128)[n:, :4])
        assert torch.isnan(got[n:, 4:, 80:96]).all() and torch.isfinite(got[n:, 4:, :80]).all() and torch.isfinite(got[n:, 4:, 96:]).all()
        c["cache"].k_scale[blk, 0, 7, 0] = 255
        got = call(ctx, c).view(-1, 8, 128)
        assert torch.isnan(got[n:, :4]).all() and torch.equal(got[:n], clean.view(-1, 8, 128)[:n])


def test_queries_that_are_none(ctx):
    c = _case([30, 18], 8, 2, 16, seed=8)
    clean = _decode(ctx, c).view(2, 8, 128)
    c["q"][0, 130], c["q"][1, 5 * 128] = float("nan"), float("inf")
    got = _decode(ctx, c).view(2, 8, 128)
    assert torch.isnan(got[0, 1]).all() and torch.isnan(got[1, 5]).all()
    for b, h in ((0, 1), (1, 5)):
        rest = [i for i in range(8) if i != h]
        assert torch.equal(got[b, rest], clean[b, rest])


def test_a_step_as_it_is_used(ctx):
    """A prompt, a second chunk of it, and decode steps, through the cache: q, k, v normed, rotated and stored, then read, against attention in 64 bits over the rows read back."""
    nh, kv, bs, n = 8, 2, 16, 61
    cache, table = ops.Fp4Cache.zeros(8, bs, kv), ctx.rope_table(1e4, 128, 128)
    tables = torch.tensor([[5, 2, 7, 0, 3, -1]], dtype=I32, device=DEV)
    qw, kw = ((torch.randn(128, generator=_g(i), device=DEV) * 0.2 + 1).to(BF16) for i in range(2))
    done = 0
    for count in (37, 20, 1, 1, 1, 1):
        pos = torch.arange(done, done + count, device=DEV)
        slots = (tables[0, pos // bs] * bs + pos % bs).to(I32)
        qkv = torch.randn(count, (nh + 2 * kv) * 128, generator=_g(50 + done), device=DEV).to(BF16)
        q = ops.qk_norm_rope_store_fp4(ctx, qkv, qw, kw, 1e-6, table, pos.to(I32), nh, cache, slots, q_out=torch.empty(count, nh * 128, dtype=BF16, device=DEV))
        done += count
        c = dict(q=q, cache=cache, tables=tables, lens=torch.tensor([done], dtype=I32, device=DEV), cu=torch.tensor([0, count], dtype=I32, device=DEV), new=[count], nh=nh)
        _near(_portions(ctx, c) if count > 1 else _decode(ctx, c), c)
    assert done == n


def test_captured_and_replayed_on_other_streams(ctx):
    """Append and attention captured into two graphs that replay side by side on two streams, with other lengths than at capture."""
    nh, kv, bs = 16, 4, 32
    table = ctx.rope_table(1e4, 128, 4096)
    sides = []
    for seed in (1, 2):
        c = _case([900, 40, 333], nh, kv, bs, seed=seed)
        c["qkv"] = torch.randn(3, (nh + 2 * kv) * 128, generator=_g(seed), device=DEV).to(BF16)
        c["pos"], c["slots"] = torch.empty(3, dtype=I32, device=DEV), torch.empty(3, dtype=I32, device=DEV)

        def at(lens, c=c):
            for b, n in enumerate(lens):
                c["lens"][b], c["pos"][b], c["slots"][b] = n, n - 1, int(c["tables"][b, (n - 1) // bs]) * bs + (n - 1) % bs
            torch.cuda.synchronize()

        def step(c=c):
            c["q"] = ops.qk_norm_rope_store_fp4(ctx, c["qkv"], None, None, 1e-6, table, c["pos"], nh, c["cache"], c["slots"], q_out=c["q"])
            return _decode(ctx, c)

        at([1, 1, 1])
        stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        with torch.cuda.stream(stream):
            step()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            out = step()
        sides.append((c, at, stream, graph, out))
    for lens in ([900, 40, 333], [1, 17, 2]):
        for c, at, *_ in sides:
            at(lens)
        for _ in range(5):
            for _, _, stream, graph, _ in sides:
                with torch.cuda.stream(stream):
                    graph.replay()
        torch.cuda.synchronize()
        for c, _, _, _, out in sides:
            _near(out, c)


MANY = dict(new=[70, 33], before=[30, 150], nh=8, kv=2, bs=16)          # 280 rows of a key head: the kernel on tcgen05; 4 rows a token


def _many(seed=0, **over):
    m = {**MANY, **over}
    return _case([n + b for n, b in zip(m["new"], m["before"])], m["nh"], m["kv"], m["bs"], new=m["new"], seed=seed, size=m.get("size", 1.0))


@pytest.mark.parametrize("size,scale", [(0.01, 1.0), (30.0, 128 ** -0.5), (1.0, -0.1), (1.0, 0.0), (300.0, 1.0), (300.0, -1.0)])
def test_long_portions_of_flat_and_peaked_rows(ctx, size, scale):
    c = _many(seed=9, size=size)
    _near(_portions(ctx, c, scale), c, scale)


@pytest.mark.parametrize("size", [2.0 ** -60, 2.0 ** 15, 2.0 ** 60])
def test_long_portions_with_queries_of_any_size(ctx, size):
    c = _many(seed=12)
    c["q"] = (c["q"].float() * size).to(BF16)
    _near(_portions(ctx, c, 128 ** -0.5 / size), c, 128 ** -0.5 / size)


@pytest.mark.parametrize("new,kv,group", [([5], 2, 1), ([9, 4], 2, 4), ([70, 33], 2, 4), ([40], 1, 12)])
def test_numbers_that_are_none_behind_a_mask(ctx, new, kv, group):
    """A cached value or key that is no number, among the portion's own tokens: the rows in front of it do not see it, and are what they are without it."""
    nh = kv * group
    c = _case([n + 40 for n in new], nh, kv, 16, new=new, seed=21)
    clean = _portions(ctx, c).view(-1, nh, 128)
    at = 40 + new[0] // 2                                              # a token of the first sequence
    blk, off = int(c["tables"][0, at // 16]), at % 16
    c["cache"].v_scale[blk, 0, off, 2] = 255
    got = _portions(ctx, c).view(-1, nh, 128)
    first = at - 40
    mine = slice(0, group)
    assert torch.equal(got[:first], clean[:first]) and torch.equal(got[new[0]:], clean[new[0]:]) and torch.equal(got[:, group:], clean[:, group:])
    seen = got[first:new[0], mine]
    assert torch.isnan(seen[..., 32:48]).all() and torch.isfinite(seen[..., :32]).all() and torch.isfinite(seen[..., 48:]).all()
    c["cache"].k_scale[blk, 0, off, 7] = 255
    got = _portions(ctx, c).view(-1, nh, 128)
    assert torch.equal(got[:first], clean[:first]) and torch.isnan(got[first:new[0], mine]).all() and torch.equal(got[:, group:], clean[:, group:])


def test_queries_of_long_portions_that_are_none(ctx):
    c = _many(seed=8)
    clean = _portions(ctx, c).view(-1, 8, 128)
    c["q"][3, 130], c["q"][60, 5 * 128] = float("nan"), float("inf")
    got = _portions(ctx, c).view(-1, 8, 128)
    assert torch.isnan(got[3, 1]).all() and torch.isnan(got[60, 5]).all()
    same = torch.ones(got.shape[:2], dtype=torch.bool, device=DEV)
    same[3, 1] = same[60, 5] = False
    assert torch.equal(got[same], clean[same])


@pytest.mark.parametrize("nh,kv", [(72, 1), (130, 1), (65, 1), (96, 4)])
def test_decode_of_many_heads_to_a_key_head(ctx, nh, kv):
    c = _case([50, 0, 3], nh, kv, 16, seed=4)
    _near(_decode(ctx, c), c)


def test_many_sequences(ctx):
    """More sequences than the schedule looks at in one go: 2 100 of one token and 65 heads, and 700 of decode."""
    g = torch.Generator().manual_seed(3)
    lens = torch.randint(0, 40, (2100,), generator=g).tolist()
    c = _case(lens, 65, 1, 16, seed=5)
    _near(_portions(ctx, c), c)
    d = _case(lens[:700], 4, 2, 16, seed=6)
    _near(_decode(ctx, d), d)


def test_pages_far_into_a_long_cache(ctx):
    """Pages beyond 2^32 bytes of codes."""
    kv, bs, blocks, nh = 8, 256, 36000, 16
    k, ks = torch.empty(blocks, kv, bs, 64, dtype=U8, device=DEV), torch.empty(blocks, kv, bs, 8, dtype=U8, device=DEV)
    cache = ops.Fp4Cache(k, ks, torch.empty_like(k), torch.empty_like(ks))
    table = torch.tensor([[blocks - 1, 33333, 0]], dtype=I32, device=DEV)
    n = 300
    pos = torch.arange(n, device=DEV)
    slots = (table[0, pos // bs] * bs + pos % bs).to(I32)
    rows = [torch.randn(n, kv * 128, generator=_g(i), device=DEV).to(BF16) for i in (1, 2)]
    ops.store_kvcache_fp4(ctx, *rows, cache, slots)
    for new in ([1], [5], [40]):
        c = dict(q=torch.randn(new[0], nh * 128, generator=_g(3), device=DEV).to(BF16), cache=cache, tables=table, lens=torch.tensor([n], dtype=I32, device=DEV),
                 cu=torch.tensor([0] + new, dtype=I32, device=DEV), new=new, nh=nh)
        _near(_portions(ctx, c) if new[0] > 1 else _decode(ctx, c), c)


def test_portions_of_a_bound_that_is_too_low(ctx):
    """max_seqlen_q chooses the kernel; a row's result does not depend on its being right."""
    c = _many(seed=30)
    got = ops.prefill_attn_paged_fp4(ctx, c["q"], c["cache"], c["tables"], c["lens"], c["cu"], 2, 8, 128 ** -0.5)
    _near(got, c)


def _room(c, tokens=4096):
    """The same tables with room for more pages: decode of contexts that could be long shares its work in another way."""
    more = -(-tokens // c["cache"].block_size)
    return dict(c, tables=torch.cat((c["tables"], torch.full((len(c["new"]), more), -1, dtype=I32, device=DEV)), 1))


@pytest.mark.parametrize("lens,nh,kv,bs", [
    ([1], 1, 1, 16), ([17], 8, 8, 16), ([255, 256, 257], 16, 8, 256), ([1, 0, 33, 700], 32, 8, 48), ([5, 64, 63, 65, 0, 0, 129], 40, 8, 32), ([90], 12, 1, 16), ([300, 31], 16, 1, 256),
    ([70, 200], 24, 1, 16), ([100] * 37, 4, 4, 16), ([0, 0], 8, 2, 16), ([50, 0, 3], 96, 4, 16), ([700, 1, 0, 128], 5, 1, 16)])
def test_decode_with_room_for_more(ctx, lens, nh, kv, bs):
    c = _case(lens, nh, kv, bs, seed=21)
    for d in (c, _room(c, 600), _room(c)):
        _near(_decode(ctx, d), d)
    for blk in c["tables"][:, 0].tolist():                              # a NaN in each context's first row: its key head's rows, and no other's, whichever way
        if blk >= 0:
            c["cache"].v_scale[blk, 0, 0] = 255
    group, bad = nh // kv, torch.tensor([n > 0 for n in lens], device=DEV)
    for d in (c, _room(c)):
        got = _decode(ctx, d).view(len(lens), nh, 128)
        assert torch.isnan(got[bad, :group]).all() and torch.isfinite(got[bad, group:]).all() and not got[~bad].any()


@pytest.mark.parametrize("new,before,nh,kv,bs", [
    ([128], [0], 4, 2, 32), ([129, 1, 64], [31, 700, 0], 16, 4, 16), ([70], [333], 40, 8, 16), ([64, 0, 65], [0, 9, 1], 8, 1, 16), ([300, 2, 0, 90], [0, 100, 0, 800], 8, 8, 48),
    ([100] * 20, [0] * 20, 32, 8, 16), ([65] * 3, [1000, 0, 512], 24, 1, 128)])
def test_portions_with_room_for_more(ctx, new, before, nh, kv, bs):
    """Short portions in one way, and, with tables that have room for long ones, in the other; a bound of their length that is too low included."""
    c = _case([n + b for n, b in zip(new, before)], nh, kv, bs, new=new, seed=23)
    for d in (c, _room(c)):
        _near(_portions(ctx, d), d)
        _near(ops.prefill_attn_paged_fp4(ctx, d["q"], d["cache"], d["tables"], d["lens"], d["cu"], 64, nh, 128 ** -0.5), d)
    c["cache"].v_scale[int(c["tables"][0, 0]), 0, 0, 0] = 255              # the first context's first row: every row of its key head
    group = nh // kv
    for d in (c, _room(c)):
        got = _portions(ctx, d).view(-1, nh, 128)
        assert torch.isnan(got[:new[0], :group, :16]).all() and torch.isfinite(got[:new[0], :group, 16:]).all() and torch.isfinite(got[:new[0], group:]).all() and torch.isfinite(got[new[0]:]).all()


@pytest.mark.parametrize("new,before,nh,kv,bs", [
    ([1], [0], 4, 2, 16), ([5], [0], 8, 8, 16), ([3, 1, 8], [0, 40, 500], 32, 8, 256), ([17, 2], [1, 200], 8, 1, 48), ([1] * 40, list(range(0, 200, 5)), 8, 8, 16), ([33], [64], 4, 1, 64),
    ([2, 0, 3, 0], [0, 9, 100, 700], 12, 2, 16), ([4] * 30, [90] * 30, 32, 4, 32)])
def test_portions_of_few_rows_with_room_for_more(ctx, new, before, nh, kv, bs):
    c = _case([n + b for n, b in zip(new, before)], nh, kv, bs, new=new, seed=24)
    for d in (c, _room(c)):
        _near(_portions(ctx, d), d)
        _near(ops.prefill_attn_paged_fp4(ctx, d["q"], d["cache"], d["tables"], d["lens"], d["cu"], 1, nh, 128 ** -0.5), d)
    c["lens"][0] = 0                                                       # a context of nothing: zeros
    for d in (c, _room(c)):
        got = _portions(ctx, d)
        assert not got[:new[0]].any() and torch.isfinite(got).all()


@pytest.mark.parametrize("rows", [8, 9, 16, 17, 32, 33, 48, 64, 65])
@pytest.mark.parametrize("seqs", [1, 40])
def test_portions_around_the_kernels_ends(ctx, seqs, rows):
    """Numbers of rows of a key head at which another kernel takes them, for few sequences and for many."""
    c = _case([rows + 70] * seqs, 1, 1, 16, new=[rows] * seqs, seed=25)
    for d in (c, _room(c)):
        _near(_portions(ctx, d), d)
