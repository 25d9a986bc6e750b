"""Attention over the 4-bit cache where a warp or a CTA has several units, and a unit several CTAs: the list of all tiles, cut into stretches longer than the shortest, against the
definition in 64 bits (bounds: fp4_ref.attention)."""
import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu
ops = importlib.import_module("nano-vllm-candle_b200.ops")
BF16, F64, I32, U8 = torch.bfloat16, torch.float64, torch.int32, torch.uint8
DEV = "cuda:0"
WARPS = {8: 4 * 4 * 148, 16: 2 * 4 * 148}                             # of the grid at its largest, by columns; a stretch is 3 tiles at least


def _case(ctx, lens, new, nh, kv, bs, seed, room=8192):
    """Pages in any order, NaN in every row and page that no context has, tables with room for long contexts."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    n = torch.tensor(lens)
    per = -(-n // bs)
    blocks = int(per.sum()) + 2
    cache = ops.Fp4Cache(*(torch.full((blocks, kv, bs, w), 255, dtype=U8, device=DEV) for w in (64, 8, 64, 8)))
    tables = torch.full((len(lens), max(int(per.max()), -(-room // bs))), -1, dtype=I32)
    order, at = torch.randperm(blocks, generator=g, device=DEV).cpu().to(I32), 0
    for b, m in enumerate(per.tolist()):
        tables[b, :m] = order[at:at + m]
        at += m
    slots = torch.cat([tables[b, :int(per[b])].repeat_interleave(bs)[:m] * bs + torch.arange(m) % bs for b, m in enumerate(lens)]).to(I32).to(DEV)
    k, v = (torch.randn(slots.numel(), kv * 128, generator=g, device=DEV).to(BF16) for _ in range(2))
    ops.store_kvcache_fp4(ctx, k, v, cache, slots)
    q = torch.randn(sum(new), nh * 128, generator=g, device=DEV).to(BF16)
    return dict(q=q, cache=cache, tables=tables.to(DEV), lens=n.to(I32).to(DEV), cu=torch.tensor([0] + new).cumsum(0).to(I32).to(DEV), new=new, nh=nh, slots=slots, n=lens)


def _call(ctx, c):
    if max(c["new"]) == 1 and min(c["new"]) == 1:
        return ops.paged_decode_attn_fp4(ctx, c["q"], c["cache"], c["tables"], c["lens"], c["nh"], 128 ** -0.5)
    return ops.prefill_attn_paged_fp4(ctx, c["q"], c["cache"], c["tables"], c["lens"], c["cu"], max(c["new"]), c["nh"], 128 ** -0.5)


def _near(ctx, got, c):
    """All rows.  The cached numbers are read back (tests/test_fp4_cache_gpu.py holds that bit by bit)."""
    nh, kv = c["nh"], c["cache"].kv
    scale, group = 128 ** -0.5, nh // c["cache"].kv
    rows, at, done = ops.read_kvcache_fp4(ctx, c["cache"], c["slots"]), 0, 0
    keys, values = ((a.to(F64).unflatten(-1, (8, 16)) * s.to(F64)[..., None]).flatten(-2) for a, s in (rows[:2], rows[2:]))
    worst = 0.0
    for m, n in zip(c["n"], c["new"]):
        k, v = keys[at:at + m], values[at:at + m]
        at += m
        out = got[done:done + n].to(F64).view(n, kv, group, 128)
        q = c["q"][done:done + n].to(F64).view(n, kv, group, 128)
        done += n
        sees = torch.arange(m - n, m, device=DEV)[:, None] >= torch.arange(m, device=DEV)          # [n, m]
        none = ~sees.any(1)
        assert not out[none].any()
        if not m or bool(none.all()):
            continue
        out, q, sees = out[~none], q[~none], sees[~none]
        s = torch.einsum("nhgd,mhd->nhgm", q, k) * scale
        p = torch.softmax(s.masked_fill(~sees[:, None, None], -float("inf")), -1)
        size = (torch.einsum("nhgd,mhd->nhgm", q.abs(), k.abs()) * scale).amax(-1, keepdim=True)
        tiny = q.abs().amax(-1, keepdim=True) * 2.0 ** -25 * k.abs().sum(-1).amax() * scale
        weight = 2.0 ** -11 + 2 * (size * 132 * 2.0 ** -24 + tiny + 2.0 ** -20) + m * 2.0 ** -31 + (m / 16 + 64) * 2.0 ** -24
        want, a = torch.einsum("nhgm,mhd->nhgd", p, v), torch.einsum("nhgm,mhd->nhgd", p, v.abs())
        far = 2.0 ** -8 * want.abs() + weight * a + m * 2.0 ** -31 * v.abs().amax()
        worst = torch.maximum(torch.as_tensor(worst, device=DEV), ((out - want).abs() / far).nan_to_num(float("inf")).max())
    assert done == got.shape[0] and float(worst) <= 1, f"{float(worst)} times what it may be off"


def _stretch(c, cols):
    """Tiles of a warp's stretch in the kernel for few rows, a unit counting two more than it has."""
    kv, group = c["cache"].kv, c["nh"] // c["cache"].kv
    total = sum(kv * (-(-n * group // cols)) * (-(-m // 32) + 2) for m, n in zip(c["n"], c["new"]) if m)
    return -(-total // WARPS[cols])


def _ragged(count, low, high, seed, zeros=0):
    g = torch.Generator().manual_seed(seed)
    lens = torch.randint(low, high + 1, (count,), generator=g).tolist()
    for i in torch.randperm(count, generator=g)[:zeros].tolist():
        lens[i] = 0
    return lens


DECODES = [(200, 1, 400, 8, 8, 16, 8), (200, 1, 400, 32, 8, 256, 8), (230, 1, 300, 96, 8, 48, 16), (3000, 1, 40, 16, 4, 16, 8), (1500, 30, 34, 20, 2, 32, 16), (37, 1, 9000, 64, 8, 256, 8),
           (5, 20000, 60000, 16, 8, 64, 8)]


@pytest.mark.parametrize("count,low,high,nh,kv,bs,cols", DECODES)
def test_decode(ctx, count, low, high, nh, kv, bs, cols):
    c = _case(ctx, _ragged(count, low, high, count, zeros=count // 8), [1] * count, nh, kv, bs, 3)
    assert _stretch(c, cols) > 3
    got = _call(ctx, c)
    _near(ctx, got, c)
    assert torch.equal(got, _call(ctx, c))


@pytest.mark.parametrize("count,low,high,most,nh,kv,bs,cols", [(300, 1, 400, 2, 32, 8, 16, 8), (200, 1, 400, 4, 32, 8, 256, 16), (150, 60, 700, 8, 32, 8, 48, 16), (1000, 1, 70, 8, 4, 4, 16, 8),
                                                              (24, 500, 3000, 6, 40, 8, 256, 16)])
def test_portions_of_few_rows(ctx, count, low, high, most, nh, kv, bs, cols):
    new = _ragged(count, 0, most, 7)
    lens = [m if i % 9 else n // 2 for i, (m, n) in enumerate(zip(_ragged(count, low, high, count, zeros=count // 10), new))]         # some begin in front of their context
    c = _case(ctx, lens, new, nh, kv, bs, 4)
    assert _stretch(c, cols) > 3
    got = _call(ctx, c)
    _near(ctx, got, c)
    assert torch.equal(got, _call(ctx, c))


@pytest.mark.parametrize("count,low,high,most,nh,kv,bs", [(60, 100, 900, 100, 32, 8, 16), (9, 1000, 5000, 700, 16, 2, 256), (400, 65, 300, 65, 8, 4, 48), (2, 9000, 15000, 1500, 64, 8, 64)])
def test_long_portions(ctx, count, low, high, most, nh, kv, bs):
    c = _case(ctx, _ragged(count, low, high, count, zeros=count // 10), _ragged(count, 0, most, 8), nh, kv, bs, 5)
    got = _call(ctx, c)
    _near(ctx, got, c)
    assert torch.equal(got, _call(ctx, c))


@pytest.mark.parametrize("new,nh", [(1, 8), (1, 16), (3, 4), (8, 4), (64, 4), (200, 4)])
def test_one_context_over_many_ctas(ctx, new, nh):
    """One key head of 16 000 and of 40 000 tokens: a unit in more than 32 pieces of the kernel for few rows, in up to 19 of the other's."""
    for m in (16000, 40001):
        c = _case(ctx, [m], [new], nh, 1, 256, 6, room=65536)
        got = _call(ctx, c)
        _near(ctx, got, c)


@pytest.mark.parametrize("most,nh,cols", [(2, 32, 8), (4, 32, 16), (100, 8, 0)])
def test_numbers_that_are_none_stay_with_their_unit(ctx, most, nh, cols):
    """Units in mid-stretch whose own tokens hold a NaN: the rows that see it have it, the units that the same warp takes in front of it and behind it do not."""
    count, kv = 200, 8
    new = [most] * count
    lens = [m + most for m in _ragged(count, 1, 300, 9)]
    c = _case(ctx, lens, new, nh, kv, 16, 10)
    assert not cols or _stretch(c, cols) > 3
    clean = _call(ctx, c).view(count, most, nh, 128)
    bad = list(range(3, count, 5))
    first = most // 2                                                       # its token: the rows from this one on see it
    for b in bad:
        at = lens[b] - most + first
        c["cache"].v_scale[int(c["tables"][b, at // 16]), b % kv, at % 16, 3] = 255
    got = _call(ctx, c).view(count, most, nh, 128)
    want = torch.zeros(got.shape, dtype=torch.bool, device=DEV)
    for b in bad:
        want[b, first:, (b % kv) * (nh // kv):(b % kv + 1) * (nh // kv), 48:64] = True
    assert torch.equal(torch.isnan(got), want) and torch.equal(got[~want], clean[~want])
