"""Rows and weights in 8 bits where it is easy to go wrong: units far from one, numbers that are none, tiles behind the first.

Tolerances come from the roundings in between, each at most 2^-24 of the value in fp32 (the hardware's exponential 2^-22, its reciprocal 2^-23)."""
import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu
ops = importlib.import_module("nano-vllm-candle_b200.ops")
BF16, F32, F64, E4M3 = torch.bfloat16, torch.float32, torch.float64, torch.float8_e4m3fn
DEV = "cuda:0"
LEAST = 2.0 ** -126


def _bits(t):
    return t.view(torch.uint8) if t.dtype == E4M3 else t


def _g(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


# ----------------------------------------------------------------------------- what a call reads, whoever wrote it
@pytest.mark.parametrize("route,M", [(11, 9), (14, 9), (21, 30), (24, 30), (31, 150), (32, 150), (41, 150), (51, 300), (61, 300)])
@pytest.mark.parametrize("writer", ["copy", "rows"])
def test_weights_written_in_front_of_their_product(ctx, route, M, writer):
    """Weights and scales written over by a kernel that is none of the library's, or by one that lets its followers start early, directly in front of the product that reads them."""
    N, K, links, l, h = 784, 1296, 8, ctx.l, ctx.h
    kb, nb = (K + 127) // 128, (N + 127) // 128
    q, s = ops.quant_fp8(ctx, torch.randn(M, K, generator=_g(1), device=DEV))
    full = [torch.randn(N, K, generator=_g(2 + i), device=DEV).to(BF16) for i in range(links)]
    new_q = [ops.quant_fp8(ctx, w)[0].view(torch.uint8) for w in full]
    new_s = [torch.rand(nb, kb, generator=_g(50 + i), device=DEV) + 0.5 for i in range(links)]
    wq, ws, beside = new_q[0].clone(), new_s[0].clone(), torch.empty(N, kb, device=DEV)
    stream = torch.cuda.current_stream().cuda_stream

    def chain(wait):
        outs = [torch.empty(M, N, dtype=BF16, device=DEV) for _ in full]
        torch.cuda.synchronize()
        for i, c in enumerate(outs):
            ws.copy_(new_s[i])
            if writer == "copy":
                wq.copy_(new_q[i])
            else:
                assert l.nvc_quant_fp8_rows(h, full[i].data_ptr(), 0, K, N, ops.ACT_NONE, 0, None, None, wq.data_ptr(), K, beside.data_ptr(), kb, N, K, stream) == 0
            if wait:
                torch.cuda.synchronize()
            assert l.nvc_gemm_fp8_ex(h, q.data_ptr(), K, s.data_ptr(), kb, wq.data_ptr(), ws.data_ptr(), c.data_ptr(), N, 0, M, N, K, route, stream) == 0
            if wait:
                torch.cuda.synchronize()
        torch.cuda.synchronize()
        return outs

    want = chain(True)
    assert not torch.equal(want[0], want[1])
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(chain(False), want))


@pytest.mark.parametrize("N,H", [(3, 2048), (1200, 1024)])
def test_norm_weights_written_in_front_of_their_norm(ctx, N, H):
    x = torch.randn(N, H, generator=_g(1), device=DEV).to(BF16)
    new = [torch.randn(H, generator=_g(2 + i), device=DEV).to(BF16) for i in range(12)]
    w = new[0].clone()
    want = []
    for n in new:
        want.append(ops.add_rmsnorm_fp8(ctx, x, n, 1e-6)[:2])
    torch.cuda.synchronize()
    got = []
    for n in new:
        w.copy_(n)
        got.append(ops.add_rmsnorm_fp8(ctx, x, w, 1e-6)[:2])
    for (q, s), (q0, s0) in zip(got, want):
        assert torch.equal(_bits(q), _bits(q0)) and torch.equal(s, s0)


# ----------------------------------------------------------------------------- gated units, one number to a block
def _one_to_a_block(ctx, gate, up, act):
    """gate, up [n] fp32 -> what the scale of a block with nothing else in it says the unit gave, and the sign of its number."""
    n = gate.numel()
    x = torch.zeros(n, 256, device=DEV)
    x[:, 5], x[:, 128 + 5] = gate, up
    q, s = ops.quant_fp8(ctx, x, act=act)
    got = q.to(F64)
    assert torch.all(got[:, :5] == 0) and torch.all(got[:, 6:] == 0)
    return s.to(F64)[:, 0] * 448, torch.sign(got[:, 5])


def _unit64(gate, act):
    z = gate.to(F64)
    w = z if act == ops.ACT_SILU_MUL else z * (2 * 0.7978845608028654) * (1 + 0.044715 * z * z)
    return w, z * torch.sigmoid(w)


@pytest.mark.parametrize("act", [ops.ACT_SILU_MUL, ops.ACT_GELU_TANH_MUL])
def test_tiny_gates_keep_their_digits(ctx, act):
    """Gates down to the least normal numbers, with an up value that brings their product back: ten roundings of 2^-24 at most, and two of the scale."""
    gate = torch.tensor([1e-28, 1e-30, 1e-33, 1e-34, 1e-35, 1e-36, 1e-37, 2.4e-38], device=DEV)
    gate = torch.cat([gate, -gate, gate.to(BF16).float()])
    for up in (1.0, 1e10, -1e30):
        u = torch.full_like(gate, up)
        _, y = _unit64(gate, act)
        want = y * u.to(F64)
        keep = want.abs() >= 448 * 2 * LEAST          # else the scale is the least one
        got, sign = _one_to_a_block(ctx, gate, u, act)
        assert torch.all(((got - want.abs()).abs() <= (2.0 ** -20 + 2.0 ** -22) * want.abs())[keep]), (got / want.abs()).tolist()
        assert torch.all((sign == torch.sign(want))[keep])


@pytest.mark.parametrize("act", [ops.ACT_SILU_MUL, ops.ACT_GELU_TANH_MUL])
def test_gates_far_below_zero_keep_their_digits(ctx, act):
    """A single gate to a block, down to where the sigmoid leaves fp32.  silu: the exponential 2^-22, the reciprocal 2^-23, a second order of 2^-26 and five roundings, below
    2^-20.  gelu: its exponent is computed, four roundings of 2^-24 of itself, which the part of the sigmoid that falls carries."""
    most = 102.0 if act == ops.ACT_SILU_MUL else 10.4
    gate = torch.linspace(-most, 12.0, 20011, device=DEV)
    w, y = _unit64(gate, act)
    up = torch.exp2(torch.floor(-torch.log2(y.abs().clamp_min(2.0 ** -148)))).clamp(2.0 ** -20, 2.0 ** 120).float()
    want = (y * up.to(F64)).abs()
    got, sign = _one_to_a_block(ctx, gate, up, act)
    rel = 2.0 ** -20 + (0 if act == ops.ACT_SILU_MUL else 2.0 ** -22) * w.abs() * torch.sigmoid(-w)
    tol = (rel + 2.0 ** -22) * want + 2.0 ** -149 * up.to(F64) + 448 * LEAST          # the gate itself may be a denormal number
    err = (got - want).abs()
    worst = int((err / tol).argmax())
    assert torch.all(err <= tol), (float(gate[worst]), float(got[worst]), float(want[worst]), float((err / tol)[worst]))
    assert torch.all((sign == torch.sign(y))[want > 2.0 ** -100])


# ----------------------------------------------------------------------------- numbers that are none
@pytest.mark.parametrize("N,H", [(4, 1024), (2100, 256), (1000, 1040), (600, 4096)])
@pytest.mark.parametrize("where", [(8,), (8, 9, 10, 11), (6, 7, 8, 9, 10, 11, 12, 13), tuple(range(128))])
def test_a_norm_keeps_a_nan_to_itself(ctx, N, H, where):
    """Weights that are no numbers, alone, four neighbouring ones and a whole block: every other number has the bits that it has where they count for nothing."""
    x = torch.randn(N, H, generator=_g(N + H), device=DEV).to(BF16)
    w = 1 + 0.2 * torch.randn(H, generator=_g(7), device=DEV)
    at = torch.tensor(where, device=DEV) + 128
    nan, zero = w.clone(), w.clone()
    nan[at], zero[at] = float("nan"), 0.0
    q, s, out = ops.add_rmsnorm_fp8(ctx, x, nan, 1e-6, want_out=True)
    q0, s0, out0 = ops.add_rmsnorm_fp8(ctx, x, zero, 1e-6, want_out=True)
    assert torch.equal(s, s0)
    assert torch.all(torch.isnan(q.float()[:, at])) and torch.all(torch.isnan(out[:, at]))
    rest = torch.ones(H, dtype=torch.bool, device=DEV)
    rest[at] = False
    assert torch.equal(_bits(q)[:, rest], _bits(q0)[:, rest]) and torch.equal(out[:, rest], out0[:, rest])


@pytest.mark.parametrize("act", [ops.ACT_NONE, ops.ACT_RELU2, ops.ACT_SILU_MUL, ops.ACT_GELU_TANH_MUL])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_units_keep_a_nan(ctx, act, dtype):
    """A NaN stays one through every unit, from either half of a gated one, and counts for no scale."""
    gated = act in (ops.ACT_SILU_MUL, ops.ACT_GELU_TANH_MUL)
    x = torch.randn(9, 512 if gated else 256, generator=_g(5), device=DEV).abs().to(dtype)
    q0, s0 = ops.quant_fp8(ctx, torch.where(torch.arange(x.shape[1], device=DEV) % 256 == 40, torch.zeros((), dtype=dtype, device=DEV), x), act=act)
    for col in (40, 256 + 40) if gated else (40,):
        y = x.clone()
        y[:, col] = float("nan")
        q, s = ops.quant_fp8(ctx, y, act=act)
        assert torch.all(torch.isnan(q.float()[:, 40])), col
        assert torch.equal(s, s0)
        assert torch.equal(_bits(q)[:, :40], _bits(q0)[:, :40]) and torch.equal(_bits(q)[:, 41:], _bits(q0)[:, 41:])


# ----------------------------------------------------------------------------- strides that are never used, sizes that pass 31 bits
def test_one_row_of_any_stride(ctx):
    """A single row's distance to the next one says nothing: a column seen as a row is as good as any."""
    x, w = torch.randn(1, 256, generator=_g(1), device=DEV), torch.ones(256, device=DEV)
    wq, ws = ops.quant_fp8_weight(ctx, torch.randn(160, 256, generator=_g(2), device=DEV))
    q = torch.empty(256, 1, dtype=torch.uint8, device=DEV).view(E4M3).t()
    s, c = torch.empty(2, 1, device=DEV).t(), torch.empty(160, 1, device=DEV).t()
    assert q.stride() == (1, 1) and s.stride() == (1, 1) and c.stride() == (1, 1)
    want = ops.quant_fp8(ctx, x)
    ops.quant_fp8(ctx, x, q=q, scale=s)
    assert torch.equal(_bits(q), _bits(want[0])) and torch.equal(s, want[1])
    assert torch.equal(ops.gemm_fp8(ctx, q, s, wq, ws, out=c), ops.gemm_fp8(ctx, *want, wq, ws, out_dtype=F32))
    want = ops.add_rmsnorm_fp8(ctx, x, w, 1e-6)
    ops.add_rmsnorm_fp8(ctx, x, w, 1e-6, q=q, scale=s)
    assert torch.equal(_bits(q), _bits(want[0])) and torch.equal(s, want[1])


def test_refusals_of_widths(ctx):
    """Widths and rows whose number of blocks passes 31 bits on the way: refused before anything is read, where it became a negative number."""
    q, s = torch.empty(4, 256, dtype=torch.uint8, device=DEV), torch.ones(4, 2, device=DEV)
    w, l, h = torch.ones(128, 256, dtype=BF16, device=DEV), ctx.l, ctx.h
    top = 2 ** 31 - 16                               # the largest multiple of 16
    p, sp, wp = q.data_ptr(), s.data_ptr(), w.data_ptr()
    calls = [lambda: l.nvc_quant_fp8_rows(h, wp, 0, top, 4, ops.ACT_NONE, 0, None, None, p, top, sp, 2, 0, top, 0),
             lambda: l.nvc_quant_fp8_blocks(h, wp, 0, p, sp, 0, 2 ** 31 - 1, 256, 0), lambda: l.nvc_quant_fp8_blocks(h, wp, 0, p, sp, 0, 256, top, 0),
             lambda: l.nvc_gemm_fp8_grouped(h, p, 256, sp, 2, p, sp, wp, 128, 0, 0, 128, 256, sp, 2 ** 24 - 1, 0, 0)]
    for N, K in ((128, top), (top, 256)):
        calls += [lambda N=N, K=K: l.nvc_gemm_fp8(h, p, K, sp, 2, p, sp, wp, N, 0, 0, N, K, 0),
                  lambda N=N, K=K: l.nvc_gemm_fp8_grouped(h, p, K, sp, 2, p, sp, wp, N, 0, 0, N, K, sp, 1, 0, 0)]
    for i, call in enumerate(calls):                 # none of them has rows: nothing would be launched
        assert call() == -2, i
        assert b"too many rows or too wide" in l.nvc_last_error(h), i


# ----------------------------------------------------------------------------- tiles behind the first, bands, loops
def _whole(seed, M, N, K, groups=None):
    """Numbers of -3 to 3 with scales that are powers of two, different for every block, and the product in 64 bits' arguments: every sum is exact in fp32."""
    g, kb, nb = _g(seed), (K + 127) // 128, (N + 127) // 128
    lead = () if groups is None else (groups,)
    whole = lambda *shape: torch.randint(-3, 4, shape, generator=g, device=DEV).float()
    two = lambda *shape: torch.exp2(torch.randint(-2, 3, shape, generator=g, device=DEV).float())
    q, s, wq, ws = whole(M, K), two(M, kb), whole(*lead, N, K), two(*lead, nb, kb)
    a = q.to(F64) * s.to(F64).repeat_interleave(128, -1)[:, :K]
    w = wq.to(F64) * ws.to(F64).repeat_interleave(128, -2)[..., :N, :].repeat_interleave(128, -1)[..., :K]
    return q.to(E4M3), s, wq.to(E4M3), ws, a, w


def _forced(ctx, route, q, s, wq, ws, dtype):
    (M, K), N = q.shape, wq.shape[0]
    c = torch.full((M + 1, N + 8), 7.0, dtype=dtype, device=DEV)
    assert ctx.l.nvc_gemm_fp8_ex(ctx.h, q.data_ptr(), K, s.data_ptr(), s.shape[1], wq.data_ptr(), ws.data_ptr(), c.data_ptr(), N + 8, int(dtype == F32), M, N, K, route,
                                 torch.cuda.current_stream().cuda_stream) == 0
    assert torch.all(c[M] == 7.0) and torch.all(c[:, N:] == 7.0)
    return c[:M, :N]


@pytest.mark.parametrize("K", [128, 272, 1040])
@pytest.mark.parametrize("route", [41, 51, 61])
def test_several_tiles_to_a_cta(ctx, route, K):
    """Two and more tiles to every CTA, or pair of them: ring, accumulators and what was asked ahead go on from tile to tile.  More k-blocks than stages, and fewer."""
    M, N = 2500, 5008                            # 400 tiles of 128 x 256, 200 of 256 x 256
    q, s, wq, ws, a, w = _whole(K, M, N, K)
    want = a @ w.T
    for dtype in (F32, BF16):
        for _ in range(2):
            assert torch.equal(_forced(ctx, route, q, s, wq, ws, dtype), want.to(F32).to(dtype))
    assert torch.equal(ops.gemm_fp8(ctx, q, s, wq, ws, out_dtype=F32), want.to(F32))


@pytest.mark.parametrize("M,N,K", [(4764, 8208, 4112), (6300, 2064, 16400)])
def test_bands_of_row_tiles(ctx, M, N, K):
    """Weights above 32 MB are walked in bands of row tiles: 19 in two bands, 25 in three, the last one shorter."""
    q, s, wq, ws, a, w = _whole(M, M, N, K)
    want = (a @ w.T).to(F32)
    assert torch.equal(_forced(ctx, 61, q, s, wq, ws, F32), want)
    assert torch.equal(ops.gemm_fp8(ctx, q, s, wq, ws, out_dtype=F32), want)
    assert torch.equal(ops.gemm_fp8(ctx, q, s, wq, ws), want.to(BF16))


@pytest.mark.parametrize("counts,N,K", [([2000, 1500, 0, 77, 3000], 4112, 272), ([130] * 9 + [0, 1000], 2064, 1040), ([5] * 40, 1040, 144)])
def test_several_tiles_of_experts_to_a_cta(ctx, counts, N, K):
    tiles = sum([[e] * ((n + 127) // 128) for e, n in enumerate(counts)], [])
    tiles.insert(len(tiles) // 2, -1)
    tiles += [-1, -1]
    q, s, wq, ws, a, w = _whole(N, 128 * len(tiles), N, K, len(counts))
    group = torch.tensor(tiles, dtype=torch.int32, device=DEV)
    for dtype in (F32, BF16):
        got = ops.gemm_fp8_grouped(ctx, q, s, wq, ws, group, out_dtype=dtype)
        for t, e in enumerate(tiles):
            rows = slice(128 * t, 128 * t + 128)
            assert torch.equal(got[rows], (a[rows] @ w[e].T).to(F32).to(dtype) if e >= 0 else torch.zeros_like(got[rows])), t


@pytest.mark.parametrize("act", [ops.ACT_SILU_MUL, ops.ACT_GELU_TANH_MUL])
@pytest.mark.parametrize("N,H,dtype", [(1000, 12288, BF16), (9001, 1040, BF16), (4000, 3088, F32)])
def test_gated_rows_of_large_inputs(ctx, act, N, H, dtype):
    """Above 16 CTAs per SM a warp goes on from part to part: the bits that a hundred rows at a time give, which need no second part."""
    x = (3 * torch.randn(N, 2 * H, generator=_g(N), device=DEV)).to(dtype)
    q, s = ops.quant_fp8(ctx, x, act=act)
    for at in range(0, N, 100):
        q1, s1 = ops.quant_fp8(ctx, x[at:at + 100], act=act)
        assert torch.equal(_bits(q)[at:at + 100], _bits(q1)) and torch.equal(s[at:at + 100], s1), at


@pytest.mark.parametrize("act", [ops.ACT_NONE, ops.ACT_RELU2, ops.ACT_SILU_MUL])
@pytest.mark.parametrize("M,H", [(64, 144), (70, 1040), (9100, 1040), (20, 16)])
def test_rows_gathered_where_blocks_go_one_behind_the_other(ctx, act, M, H):
    """Widths whose blocks do not fill a warp's stretches, with rows by number and a count of them: what a gather in front gives, nothing behind the count."""
    x = torch.randn(40, 2 * H if act == ops.ACT_SILU_MUL else H, generator=_g(H), device=DEV).to(BF16)
    rows = torch.randint(0, 40, (M,), generator=_g(M), device=DEV, dtype=torch.int32)
    rows[3], rows[5], rows[6], rows[11] = -1, 40, rows[7], 2 ** 31 - 1
    there = (rows >= 0) & (rows < 40)
    want_q, want_s = ops.quant_fp8(ctx, torch.where(there[:, None], x[rows.clamp(0, 39).long()], torch.zeros((), dtype=BF16, device=DEV)), act=act)
    for used in (0, 1, M // 2, M - 1, M, M + 7, -3):
        q, s = torch.full((M, H), 0x33, dtype=torch.uint8, device=DEV).view(E4M3), torch.full(want_s.shape, 7.0, device=DEV)
        ops.quant_fp8(ctx, x, act=act, rows=rows, num_rows=torch.tensor([used], dtype=torch.int32, device=DEV), q=q, scale=s)
        n = min(max(used, 0), M)
        assert torch.equal(_bits(q)[:n], _bits(want_q)[:n]) and torch.equal(s[:n], want_s[:n]), used
        assert torch.all(_bits(q)[n:] == 0x33) and torch.all(s[n:] == 7.0), used


def test_calls_on_several_streams_at_once(ctx):
    """Three streams with products of every kernel, norms and rows in flight together: nothing is shared between calls, the bits are those of one call after the other."""
    sizes = [(3, 1056, 2048), (24, 800, 4096), (150, 1536, 1040), (300, 2080, 512), (1100, 1024, 1024), (2600, 3104, 640)]
    work = []
    for i, (M, N, K) in enumerate(sizes):
        x, w = torch.randn(M, K, generator=_g(i), device=DEV).to(BF16), torch.ones(K, dtype=BF16, device=DEV)
        work.append((x, w, ops.quant_fp8_weight(ctx, torch.randn(N, K, generator=_g(10 + i), device=DEV) * K ** -0.5)))

    def step(x, w, weight):
        q, s, _ = ops.add_rmsnorm_fp8(ctx, x, w, 1e-6)
        y = ops.gemm_fp8(ctx, q, s, *weight)
        return y, *ops.quant_fp8(ctx, y, act=ops.ACT_SILU_MUL)

    want = [step(*t) for t in work]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(3)], []
    for _ in range(4):
        for i in range(len(work)):
            for j, stream in enumerate(streams):
                with torch.cuda.stream(stream):
                    k = (i + 2 * j) % len(work)
                    got.append((k, step(*work[k])))
    torch.cuda.synchronize()
    for k, out in got:
        assert all(torch.equal(_bits(a), _bits(b)) for a, b in zip(out, want[k])), k
