"""Rows and weights in 8 bits and the products that read them, against plain forms in 64 bits.

Tolerances, all from the roundings in between:
  an 8-bit number: half a step of e4m3, 2^-4 of the value, or half of its smallest step, 2^-10, times the scale
  a scale, and a number in front of its rounding: fp32 arithmetic.  silu: the exponential 2^-22, the reciprocal 2^-23, five roundings of 2^-24: below 2^-20.
    norms: 16 squares per thread and two trees of five, 26 roundings, halved by the root, and six more: below 2^-19
  a product: e4m3 products are exact in fp32; sums of 128 of them, whatever their order, lose at most 2^-23 of the sum of magnitudes for each of at most 8
    partial sums that the tensor core keeps (32 numbers per instruction, four instructions), and K / 128 outer sums in fp32 2^-23 each for K <= 8192: 72 * 2^-23 <
    2^-16 of the sum of magnitudes; a bf16 result 2^-8 of itself on top"""
import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu
ops = importlib.import_module("nano-vllm-candle_b200.ops")
BF16, F32, F64, E4M3 = torch.bfloat16, torch.float32, torch.float64, torch.float8_e4m3fn
DEV = "cuda:0"


def _g(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(seed, *shape):
    g = _g(seed)
    t = torch.randn(*shape, generator=g, device=DEV)
    return t * torch.exp(torch.randn(*shape[:-1], 1, generator=g, device=DEV))


def _block_amax(y, rows=1):
    """[N, K] -> largest magnitudes of blocks of `rows` x 128, in y's type."""
    n, k = y.shape
    p = torch.nn.functional.pad(y.abs(), (0, -k % 128, 0, -n % rows))
    return p.view(p.shape[0] // rows, rows, -1, 128).amax((1, 3))


def _scale32(y, rows=1):
    """The definition's scale: a division by a tensor, since torch multiplies by 1 / 448 where the divisor is a plain number."""
    return (_block_amax(y, rows) / torch.full((), 448.0, device=y.device)).clamp_min(2.0 ** -126)


def _spread(s, k):
    return s.repeat_interleave(128, 1)[:, :k]


def _scale64(y):
    return (_block_amax(y) / 448).clamp_min(2.0 ** -126)


def _check_rows(q, scale, y, rel):
    """q * scale is y up to its 8-bit rounding, the scale is the definition's, both beside `rel` from the arithmetic in front."""
    y = y.to(F64)
    want = _scale64(y)
    assert torch.all((scale.to(F64) - want).abs() <= (rel + 2.0 ** -23) * want)
    s = _spread(scale.to(F64), y.shape[1])
    err = (q.to(F64) * s - y).abs()
    assert torch.all(err <= (2.0 ** -4 + 2 * rel + 2.0 ** -22) * y.abs() + 2.0 ** -10 * s * (1 + 2.0 ** -20)), float((err / (y.abs() + 1e-30)).max())


def _dequant(q, scale):
    return q.to(F64) * _spread(scale.to(F64), q.shape[1])


def _dequant_w(q, scale):
    n, k = q.shape
    return q.to(F64) * scale.to(F64).repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]


def _bits(t):
    return t.view(torch.uint8) if t.dtype == E4M3 else t


# ----------------------------------------------------------------------------- rows
WIDTHS = [16, 112, 128, 144, 512, 528, 1024, 2560, 12288]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("N,H", [(1, w) for w in WIDTHS] + [(3, 1008), (77, 768), (300, 4096)])
def test_rows_as_they_are(ctx, N, H, dtype):
    x = _randn(N + H, N, H).to(dtype)
    q, s = ops.quant_fp8(ctx, x)
    assert q.shape == (N, H) and s.shape == (N, (H + 127) // 128)
    # nothing but exact steps and two roundings: the same bits as these
    f = x.float()
    want = _scale32(f)
    assert torch.equal(s, want)
    assert torch.equal(_bits(q), _bits((f * _spread(1.0 / want, H)).to(E4M3)))
    _check_rows(q, s, x, 0.0)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("act", ["silu", "gelu", "relu2"])
@pytest.mark.parametrize("N,H", [(1, 16), (5, 144), (64, 768), (31, 6144)])
def test_rows_through_a_unit(ctx, N, H, act, dtype):
    x = (3 * _randn(N + H, N, H if act == "relu2" else 2 * H)).to(dtype)
    d = x.to(F64)
    if act == "relu2":
        y, kind = d.clamp_min(0).square(), ops.ACT_RELU2
    elif act == "silu":
        y, kind = d[:, :H] * torch.sigmoid(d[:, :H]) * d[:, H:], ops.ACT_SILU_MUL
    else:
        y, kind = torch.nn.functional.gelu(d[:, :H], approximate="tanh") * d[:, H:], ops.ACT_GELU_TANH_MUL
    q, s = ops.quant_fp8(ctx, x, act=kind)
    if act == "gelu":       # 1 + tanh loses digits where tanh is near -1: 2^-22 of the gate, whatever is left of it
        slack = 2.0 ** -21 * (d[:, :H] * d[:, H:]).abs()
        sc = _spread(s.to(F64), H)
        assert torch.all((q.to(F64) * sc - y).abs() <= 2.0 ** -4 * (y.abs() + slack) + slack + 2.0 ** -10 * sc * 1.001)
        top = _scale64(y)
        assert torch.all((s.to(F64) - top).abs() <= 2.0 ** -19 * top + _block_amax(slack) / 448)
    else:
        _check_rows(q, s, y, 2.0 ** -20)


def test_silu_far_from_zero(ctx):
    """Gates whose exponential leaves fp32, and zeros."""
    gate = torch.tensor([0.0, -0.0, 88.0, -88.0, 200.0, -200.0, 3e38, -3e38, 1e-30, -1e-30, -20.0, -60.0, 20.0, 1.0, -1.0, -103.0], device=DEV)
    for i in range(16):       # each alone in its block, so that its own scale shows it
        x = torch.zeros(1, 256, device=DEV)
        x[0, 5], x[0, 128 + 5] = gate[i], 0.5
        q, s = ops.quant_fp8(ctx, x, act=ops.ACT_SILU_MUL)
        want = gate[i].to(F64) * torch.sigmoid(gate[i].to(F64)) * 0.5
        got = q.to(F64)[0, 5] * s.to(F64)[0, 0]
        assert abs(float(got - want)) <= 2.0 ** -4 * abs(float(want)) + 2.0 ** -130, (float(gate[i]), float(got), float(want))
        assert int((q.float() != 0).sum()) <= 1


def test_rows_of_zeros_tiny_and_not_numbers(ctx):
    x = torch.zeros(6, 256, device=DEV)
    x[1, 3] = 1e-42                                   # a block whose scale would not be a normal number
    x[2, :] = 2.0 ** -126
    x[3, 7], x[3, 8] = float("nan"), 2.0              # the NaN stays where it is
    x[4, 200] = float("inf")
    x[5, 0] = 3.4e38
    q, s = ops.quant_fp8(ctx, x)
    least = 2.0 ** -126
    assert torch.all(s[0] == least) and torch.all(q[0].float() == 0)
    assert float(s[1, 0]) == least and torch.all(q[1].float() == 0)
    assert torch.all(s[2] == least) and torch.all(q[2].float() == 1)
    nan = torch.isnan(q[3].float())
    assert bool(nan[7]) and int(nan.sum()) == 1 and float(q[3].float()[8]) == 448 and float(s[3, 0]) == float(torch.tensor(2.0) / torch.tensor(448.0))
    assert torch.isinf(s[4, 1]) and torch.isnan((q[4].float()[200] * s[4, 1])) and torch.all(s[4, 0] == least)
    assert float(q[5].float()[0]) == 448


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rows_gathered_and_limited(ctx, dtype):
    """Rows taken by index, the same one twice, none for negative ones and for those beyond; rows behind the count stay as they were."""
    N, H = 40, 400
    x = _randn(3, N, H).to(dtype)
    rows = torch.randint(0, N, (64,), generator=_g(4), device=DEV, dtype=torch.int32)
    rows[5], rows[17], rows[6], rows[30], rows[31] = -1, -7, rows[7], N, 2 ** 31 - 1        # none for those that x has not, either
    for used in (0, 1, 50, 64, 100):
        q = torch.full((64, H), 0x33, dtype=torch.uint8, device=DEV).view(E4M3)
        s = torch.full((64, 4), 7.0, device=DEV)
        count = torch.tensor([used], dtype=torch.int32, device=DEV)
        ops.quant_fp8(ctx, x, rows=rows, num_rows=count, q=q, scale=s)
        f = torch.where((rows[:, None] < 0) | (rows[:, None] >= N), torch.zeros((), device=DEV), x.float()[rows.clamp(0, N - 1).long()])
        want = _scale32(f)
        wq = _bits((f * _spread(1.0 / want, H)).to(E4M3))
        n = min(used, 64)
        assert torch.equal(s[:n], want[:n]) and torch.equal(_bits(q)[:n], wq[:n])
        assert torch.all(s[n:] == 7.0) and torch.all(_bits(q)[n:] == 0x33)


def test_rows_with_strides(ctx):
    """Columns of wider rows in, columns of wider rows out, nothing beside them touched."""
    N, H = 9, 272
    wide = _randn(5, N, 2 * H + 48).to(BF16)
    qb = torch.full((N + 2, H + 64), 0x11, dtype=torch.uint8, device=DEV)
    sb = torch.full((N + 2, 9), -1.0, device=DEV)
    x = wide[:, 16:16 + 2 * H]
    q, s = qb[1:1 + N, 16:16 + H].view(E4M3), sb[1:1 + N, 2:5]
    ops.quant_fp8(ctx, x, act=ops.ACT_SILU_MUL, q=q, scale=s)
    q2, s2 = ops.quant_fp8(ctx, x.contiguous(), act=ops.ACT_SILU_MUL)
    assert torch.equal(_bits(q), _bits(q2)) and torch.equal(s, s2)
    qb[1:1 + N, 16:16 + H] = 0x11
    sb[1:1 + N, 2:5] = -1.0
    assert torch.all(qb == 0x11) and torch.all(sb == -1.0)


# ----------------------------------------------------------------------------- norm
@pytest.mark.parametrize("N,H", [(1, 16), (1, 1024), (2, 128), (3, 1040), (64, 2560), (33, 4096), (5, 12288), (2, 16384), (40000, 16), (2100, 256), (700, 1040), (1000, 4096), (297, 16384)])
@pytest.mark.parametrize("with_res", [False, True])
@pytest.mark.parametrize("dtype,wdtype", [(BF16, BF16), (F32, F32), (BF16, F32), (F32, BF16)])
def test_add_rmsnorm_fp8(ctx, N, H, with_res, dtype, wdtype):
    x = _randn(N + H, N, H).to(dtype)
    w = (1 + 0.2 * torch.randn(H, generator=_g(7), device=DEV)).to(wdtype)
    res = _randn(N + H + 1, N, H) if with_res else None
    out_res = torch.empty(N, H, device=DEV) if with_res else None
    q, s, out = ops.add_rmsnorm_fp8(ctx, x, w, 1e-6, residual=res, residual_out=out_res, want_out=True)
    v = x.to(F64) + (res.to(F64) if with_res else 0)
    y = v / torch.sqrt(v.square().mean(1, keepdim=True) + 1e-6) * w.to(F64)
    if with_res:
        assert torch.equal(out_res, x.float() + res)
        # the sum's own rounding, 2^-24 of its two parts, is part of y
        y = out_res.to(F64) / torch.sqrt(out_res.to(F64).square().mean(1, keepdim=True) + 1e-6) * w.to(F64)
    _check_rows(q, s, y, 2.0 ** -19)
    assert torch.all((out.to(F64) - y).abs() <= (2.0 ** -8 + 2.0 ** -18) * y.abs())
    # in place, and without the bf16 row: the same bits
    if with_res:
        q2, s2, none = ops.add_rmsnorm_fp8(ctx, x, w, 1e-6, residual=res, residual_out=res)
        assert none is None and torch.equal(_bits(q), _bits(q2)) and torch.equal(s, s2) and torch.equal(res, out_res)


def test_norm_of_zeros_and_its_strides(ctx):
    qb = torch.full((4, 128 + 32), 0x22, dtype=torch.uint8, device=DEV)
    sb = torch.full((4, 3), 5.0, device=DEV)
    w = torch.ones(128, dtype=BF16, device=DEV)
    q, s, _ = ops.add_rmsnorm_fp8(ctx, torch.zeros(4, 128, dtype=BF16, device=DEV), w, 1e-6, q=qb[:, 16:144].view(E4M3), scale=sb[:, 1:2])
    assert torch.all(q.float() == 0) and torch.all(s == 2.0 ** -126)
    assert torch.all(qb[:, :16] == 0x22) and torch.all(qb[:, 144:] == 0x22) and torch.all(sb[:, ::2] == 5.0)


# ----------------------------------------------------------------------------- weights
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("shape", [(1, 16), (16, 128), (128, 128), (130, 144), (1000, 1008), (3, 130, 272), (5, 1, 16), (2, 256, 512), (6144, 1024)])
def test_weights(ctx, shape, dtype):
    w = _randn(sum(shape), *shape).to(dtype)
    q, s = ops.quant_fp8_weight(ctx, w)
    assert q.shape == w.shape and s.shape == (*shape[:-2], (shape[-2] + 127) // 128, (shape[-1] + 127) // 128)
    for wg, qg, sg in zip(*(t if len(shape) == 3 else t[None] for t in (w, q, s))):
        f = wg.float()
        want = _scale32(f, 128)
        assert torch.equal(sg, want)
        inv = (1.0 / want).repeat_interleave(128, 0)[:f.shape[0]].repeat_interleave(128, 1)[:, :f.shape[1]]
        assert torch.equal(_bits(qg), _bits((f * inv).to(E4M3)))


# ----------------------------------------------------------------------------- products
def _operands(seed, M, N, K, groups=None):
    q, s = _rows_8bit(_randn(seed, M, K))
    if groups is None:
        w = [_weight_8bit(_randn(seed + 1, N, K) * K ** -0.5)]
        return q, s, w[0][0], w[0][1]
    w = [_weight_8bit(_randn(seed + 1 + g, N, K) * K ** -0.5) for g in range(groups)]
    return q, s, torch.stack([a.view(torch.uint8) for a, _ in w]).view(E4M3), torch.stack([b for _, b in w])


def _whole_numbers(seed, M, N, K):
    """Numbers of -3 to 3 with scales that are powers of two, different for every block."""
    g = _g(seed)
    q = torch.randint(-3, 4, (M, K), generator=g, device=DEV).float().to(E4M3)
    wq = torch.randint(-3, 4, (N, K), generator=g, device=DEV).float().to(E4M3)
    kb = (K + 127) // 128
    s = torch.exp2(torch.randint(-2, 3, (M, kb), generator=g, device=DEV).float())
    ws = torch.exp2(torch.randint(-2, 3, ((N + 127) // 128, kb), generator=g, device=DEV).float())
    return q, s, wq, ws


def _rows_8bit(x):
    s = _scale32(x)
    return (x * _spread(1.0 / s, x.shape[1])).to(E4M3), s


def _weight_8bit(x):
    s = _scale32(x, 128)
    inv = (1.0 / s).repeat_interleave(128, 0)[:x.shape[0]].repeat_interleave(128, 1)[:, :x.shape[1]]
    return (x * inv).to(E4M3), s


def _check_product(got, a, w):
    want, size = a @ w.T, a.abs() @ w.abs().T
    tol = 2.0 ** -16 * size + (2.0 ** -8 * want.abs() if got.dtype == BF16 else 0)
    err = (got.to(F64) - want).abs()
    assert torch.all(err <= tol), (float((err / (tol + 1e-300)).max()), (err > tol).nonzero()[:4].tolist())


SIZES = [(1, 16, 16), (1, 1024, 2048), (2, 48, 128), (3, 4096, 144), (7, 144, 1008), (8, 2048, 8192), (16, 272, 512), (17, 1040, 1024), (33, 6144, 640), (64, 1024, 1024), (65, 128, 2048),
         (100, 640, 4096), (127, 256, 256), (128, 512, 384), (129, 2048, 1040), (200, 1536, 2048), (256, 256, 4096), (257, 4096, 1024), (300, 784, 2560), (513, 272, 128),
         (1000, 2048, 1024), (1500, 4096, 768), (2111, 1008, 1536), (4096, 1024, 512)]


@pytest.mark.parametrize("out_dtype", [BF16, F32])
@pytest.mark.parametrize("M,N,K", SIZES)
def test_product(ctx, M, N, K, out_dtype):
    q, s, wq, ws = _operands(M + N + K, M, N, K)
    got = ops.gemm_fp8(ctx, q, s, wq, ws, out_dtype=out_dtype)
    assert got.dtype == out_dtype and got.shape == (M, N)
    _check_product(got, _dequant(q, s), _dequant_w(wq, ws))
    assert torch.equal(got, ops.gemm_fp8(ctx, q, s, wq, ws, out_dtype=out_dtype))        # bit by bit


@pytest.mark.parametrize("M,N,K", [(1, 272, 1040), (5, 1024, 4096), (64, 640, 2048), (130, 400, 1040), (300, 1040, 2064), (1030, 784, 1040)])
def test_product_of_whole_numbers_is_exact(ctx, M, N, K):
    """Small whole numbers and scales that are powers of two, different for every block: every sum is exact, so every index is the right one."""
    q, s, wq, ws = _whole_numbers(M, M, N, K)
    got = ops.gemm_fp8(ctx, q, s, wq, ws, out_dtype=F32)
    assert torch.equal(got.to(F64), _dequant(q, s) @ _dequant_w(wq, ws).T)


ROUTES = [10 * tile + shares for tile in (1, 2, 3) for shares in range(1, 9)] + [41, 51, 61]


@pytest.mark.parametrize("M,N,K", [(1, 16, 16), (5, 272, 1040), (17, 640, 2064), (64, 1024, 8192), (130, 400, 1040), (140, 176, 128), (257, 400, 272), (600, 48, 256), (1030, 784, 1040)])
def test_every_kernel_and_share(ctx, M, N, K):
    """Every kernel of a dense product with every share of K, for sizes it would not be chosen for too: exact sums, nothing written beside them."""
    q, s, wq, ws = _whole_numbers(M, M, N, K)
    want = _dequant(q, s) @ _dequant_w(wq, ws).T
    for route in ROUTES:
        for dt in (F32, BF16):
            c = torch.full((M + 2, N + 8), 7.0, dtype=dt, device=DEV)
            for _ in range(3):
                c[1:1 + M, :N] = -1.0
                assert ctx.l.nvc_gemm_fp8_ex(ctx.h, q.data_ptr(), K, s.data_ptr(), s.shape[1], wq.data_ptr(), ws.data_ptr(), c[1:].data_ptr(), N + 8, int(dt == F32), M, N, K, route,
                                             torch.cuda.current_stream().cuda_stream) == 0
                assert torch.equal(c[1:1 + M, :N], want.to(dt)), (route, dt)
            assert torch.all(c[0] == 7.0) and torch.all(c[1 + M] == 7.0) and torch.all(c[:, N:] == 7.0), (route, dt)


@pytest.mark.parametrize("out_dtype", [BF16, F32])
@pytest.mark.parametrize("M,N,K", [(1, 144, 272), (13, 272, 400), (70, 400, 1024), (140, 144, 272), (400, 1040, 640)])
def test_product_with_strides(ctx, M, N, K, out_dtype):
    """Columns of wider rows; nothing beside the result is written."""
    q, s, wq, ws = _operands(M + N, M, N, K)
    kb = s.shape[1]
    qb = torch.randint(0, 255, (M, K + 48), generator=_g(1), device=DEV, dtype=torch.uint8)
    sb = torch.full((M, kb + 3), float("nan"), device=DEV)
    qv, sv = qb[:, 16:16 + K].view(E4M3), sb[:, 1:1 + kb]
    qv.view(torch.uint8).copy_(q.view(torch.uint8))
    sv.copy_(s)
    cb = torch.full((M + 2, N + 24), 3.0, dtype=out_dtype, device=DEV)
    c = cb[1:1 + M, 8:8 + N]
    ops.gemm_fp8(ctx, qv, sv, wq, ws, out=c)
    assert torch.equal(c, ops.gemm_fp8(ctx, q, s, wq, ws, out_dtype=out_dtype))
    c.fill_(3.0)
    assert torch.all(cb == 3.0)


def test_product_of_no_rows(ctx):
    q, s, wq, ws = _operands(1, 4, 128, 256)
    assert ops.gemm_fp8(ctx, q[:0], s[:0], wq, ws).shape == (0, 128)
    assert ops.quant_fp8(ctx, torch.empty(0, 64, device=DEV))[0].shape == (0, 64)
    assert ops.add_rmsnorm_fp8(ctx, torch.empty(0, 64, device=DEV), torch.ones(64, device=DEV), 1e-6)[1].shape == (0, 1)
    assert ops.quant_fp8_weight(ctx, torch.empty(0, 16, 64, device=DEV))[1].shape == (0, 1, 1)


def test_nothing_crosses_rows_or_columns(ctx):
    """A NaN row, a NaN scale and a NaN weight row spoil their own results only."""
    for M, N, K in ((7, 272, 512), (200, 400, 512), (600, 2048, 512)):
        q, s, wq, ws = _operands(M, M, N, K)
        clean = ops.gemm_fp8(ctx, q, s, wq, ws, out_dtype=F32)
        q2, s2, w2 = q.clone(), s.clone(), wq.clone()
        q2.view(torch.uint8)[M // 2, 5] = 0x7F
        s2[M - 1, 1] = float("inf")
        w2.view(torch.uint8)[N - 3, 300] = 0x7F
        got = ops.gemm_fp8(ctx, q2, s2, w2, ws, out_dtype=F32)
        assert torch.all(torch.isnan(got[M // 2])) and torch.all(torch.isnan(got[:, N - 3]))
        assert not torch.any(torch.isfinite(got[M - 1]))
        keep = torch.ones(M, N, dtype=torch.bool, device=DEV)
        keep[M // 2] = keep[M - 1] = False
        keep[:, N - 3] = False
        assert torch.equal(got[keep], clean[keep])


# ----------------------------------------------------------------------------- products of experts
def _layout(counts, spare):
    """Groups of these many rows, each from a multiple of 128 on: (expert of each tile, first row of each group)."""
    group, first = [], []
    for e, n in enumerate(counts):
        first.append(128 * len(group))
        group += [e] * ((n + 127) // 128)
    return torch.tensor(group + [-1] * spare, dtype=torch.int32, device=DEV), first


@pytest.mark.parametrize("out_dtype", [BF16, F32])
@pytest.mark.parametrize("counts,N,K", [([1], 16, 16), ([0, 5, 0, 128, 129, 0], 144, 272), ([300, 1, 0, 77, 2], 1040, 640), ([3] * 24, 768, 2048), ([700, 900, 10, 0], 2048, 1008),
                                        ([0, 0, 0], 256, 256)])
def test_grouped_product(ctx, counts, N, K, out_dtype):
    group, first = _layout(counts, 2)
    M = 128 * group.numel()
    q, s, wq, ws = _operands(N, M, N, K, groups=len(counts))
    got = ops.gemm_fp8_grouped(ctx, q, s, wq, ws, group, out_dtype=out_dtype)
    a = _dequant(q, s)
    for e, n in enumerate(counts):
        if n:
            rows = slice(first[e], first[e] + (n + 127) // 128 * 128)
            _check_product(got[rows], a[rows], _dequant_w(wq[e], ws[e]))
    assert torch.all(got[M - 256:] == 0)
    mine = torch.full((M, N + 16), 5.0, dtype=out_dtype, device=DEV)
    ops.gemm_fp8_grouped(ctx, q, s, wq, ws, group, out=mine[:, 8:8 + N])
    assert torch.equal(mine[:M - 256, 8:8 + N], got[:M - 256])
    assert torch.all(mine[M - 256:] == 5.0) and torch.all(mine[:, :8] == 5.0) and torch.all(mine[:, 8 + N:] == 5.0)


def test_grouped_tiles_in_any_order(ctx):
    """Tiles of one expert apart, tiles without one in between."""
    group = torch.tensor([2, -1, 0, 2, 3, 1, 0], dtype=torch.int32, device=DEV)          # there are three
    N, K = 400, 384
    q, s, wq, ws = _operands(9, 7 * 128, N, K, groups=3)
    got = ops.gemm_fp8_grouped(ctx, q, s, wq, ws, group, out_dtype=F32)
    a = _dequant(q, s)
    for t, e in enumerate(group.tolist()):
        rows = slice(128 * t, 128 * t + 128)
        if e < 0 or e > 2:
            assert torch.all(got[rows] == 0)
        else:
            _check_product(got[rows], a[rows], _dequant_w(wq[e], ws[e]))


# ----------------------------------------------------------------------------- together
def _mlp(ctx, x, res, w, gu, down):
    q, s, _ = ops.add_rmsnorm_fp8(ctx, x, w, 1e-6, residual=res, residual_out=res)
    h = ops.gemm_fp8(ctx, q, s, *gu)
    q2, s2 = ops.quant_fp8(ctx, h, act=ops.ACT_SILU_MUL)
    return ops.gemm_fp8(ctx, q2, s2, *down), (q, s, h, q2, s2)


@pytest.mark.parametrize("M,H,I", [(1, 1024, 2048), (64, 1024, 1536), (333, 512, 1040)])
def test_feed_forward_in_8_bits(ctx, M, H, I):
    x, res = _randn(1, M, H).to(BF16), _randn(2, M, H)
    w = (1 + 0.1 * torch.randn(H, generator=_g(3), device=DEV)).to(BF16)
    full = [torch.randn(2 * I, H, generator=_g(4), device=DEV) * H ** -0.5, torch.randn(H, I, generator=_g(5), device=DEV) * I ** -0.5]
    gu, down = (ops.quant_fp8_weight(ctx, t) for t in full)
    y, (q, s, h, q2, s2) = _mlp(ctx, x, res.clone(), w, gu, down)
    # each step against its own inputs
    _check_product(h, _dequant(q, s), _dequant_w(*gu))
    hd = h.to(F64)
    _check_rows(q2, s2, hd[:, :I] * torch.sigmoid(hd[:, :I]) * hd[:, I:], 2.0 ** -20)
    _check_product(y, _dequant(q2, s2), _dequant_w(*down))
    # the whole against numbers that were never rounded: four operands in 8 bits, each off by at most 2^-4 of itself and evenly spread, 2^-4 / sqrt(3) = 3.6 % of
    # the norm; a product's sum carries the two relative errors of its operands, 5.1 %; twice, and the unit in between (slope at most 1.1, two factors): below 16 %
    v = x.to(F64) + res.to(F64)
    n = v / torch.sqrt(v.square().mean(1, keepdim=True) + 1e-6) * w.to(F64)
    f = n @ full[0].to(F64).T
    want = (f[:, :I] * torch.sigmoid(f[:, :I]) * f[:, I:]) @ full[1].to(F64).T
    assert float((y.to(F64) - want).norm() / want.norm()) < 0.16


def test_experts_in_8_bits(ctx):
    """Router, sort, rows of experts, both products, gated unit, combination."""
    N, H, I, E, top = 150, 512, 400, 6, 2
    x = _randn(1, N, H).to(BF16)
    w = torch.ones(H, dtype=BF16, device=DEV)
    up = [torch.randn(E, 2 * I, H, generator=_g(4), device=DEV) * H ** -0.5, torch.randn(E, H, I, generator=_g(5), device=DEV) * I ** -0.5]
    (wg, sg), (wd, sd) = (ops.quant_fp8_weight(ctx, t) for t in up)
    router = torch.randn(E, H, generator=_g(6), device=DEV) * H ** -0.5
    router[4] -= 100.0 * router[4]                  # an expert that few like
    _, _, h = ops.add_rmsnorm_fp8(ctx, x, w, 1e-6, want_out=True)
    idx, tw, _ = ops.moe_route(ctx, h, router, torch.tensor([0, 0, 0, 0, -9.0, 0], device=DEV), None, top, 1.0)
    offsets, src, pos, tiles = ops.moe_sort_padded(ctx, idx, E)
    used = offsets[E:]
    q, s = ops.quant_fp8(ctx, h, rows=src, num_rows=used)
    g = ops.gemm_fp8_grouped(ctx, q, s, wg, sg, tiles)
    q2, s2 = ops.quant_fp8(ctx, g, act=ops.ACT_SILU_MUL, num_rows=used)
    y = ops.moe_combine(ctx, ops.gemm_fp8_grouped(ctx, q2, s2, wd, sd, tiles), pos, tw)
    want = torch.zeros(N, H, dtype=F64, device=DEV)
    q1, s1 = ops.quant_fp8(ctx, h)
    a = _dequant(q1, s1)
    size = torch.zeros_like(want)
    assert not torch.any(idx == 4)
    for e in range(E):
        f = (a @ _dequant_w(wg[e], sg[e]).T).to(BF16).to(F64)
        u = f[:, :I] * torch.sigmoid(f[:, :I]) * f[:, I:]
        qe, se = _rows_8bit(u.float())
        o = _dequant(qe, se) @ _dequant_w(wd[e], sd[e]).T
        weight = torch.where(idx == e, tw, torch.zeros((), device=DEV)).sum(1, keepdim=True).to(F64)
        want += weight * o
        size += weight * (_dequant(qe, se).abs() @ _dequant_w(wd[e], sd[e]).abs().T)
    # a number of the middle that falls on the other side of a rounding moves by a step: 2^-7 in bf16, 2^-3 in 8 bits, for a few of the numbers summed; in norm below 1 %
    assert float((y.to(F64) - want).norm() / want.norm()) < 0.01
    assert torch.all((y.to(F64) - want).abs() <= 2.0 ** -7 * want.abs() + 2.0 ** -3 * size)


def test_another_stream_and_replays(ctx):
    """The chain on a stream of its own, and captured twice: two graphs over the same weights, replayed in turn with new inputs, give what direct calls give."""
    M, H, I = 24, 1024, 1536
    w = torch.ones(H, dtype=BF16, device=DEV)
    gu = ops.quant_fp8_weight(ctx, _randn(4, 2 * I, H) * H ** -0.5)
    down = ops.quant_fp8_weight(ctx, _randn(5, H, I) * I ** -0.5)
    xs = [_randn(10 + i, M, H).to(BF16) for i in range(4)]
    want = [_mlp(ctx, x, None, w, gu, down)[0] for x in xs]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = [_mlp(ctx, x, None, w, gu, down)[0] for x in xs]
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs = []
    for _ in range(2):
        x = xs[0].clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = _mlp(ctx, x, None, w, gu, down)[0]
        graphs.append((g, x, y))
    for a, b in ((0, 1), (2, 3), (3, 0)):
        graphs[0][1].copy_(xs[a]); graphs[1][1].copy_(xs[b])
        graphs[0][0].replay(); graphs[1][0].replay()
        torch.cuda.synchronize()
        assert torch.equal(graphs[0][2], want[a]) and torch.equal(graphs[1][2], want[b])


def test_chains_without_a_wait(ctx):
    """Kernels start ahead of their predecessors' end: long chains, every link from the one in front, weights fresh from their conversion."""
    for rep in range(3):
        M, H = 40, 1024
        x = _randn(20 + rep, M, H).to(BF16)
        w = torch.ones(H, dtype=BF16, device=DEV)
        full = _randn(30 + rep, H, H) * H ** -0.5
        torch.cuda.synchronize()
        weight = ops.quant_fp8_weight(ctx, full)
        y = x
        for _ in range(12):
            q, s, _ = ops.add_rmsnorm_fp8(ctx, y, w, 1e-6)
            y = ops.gemm_fp8(ctx, q, s, *weight)
        z = x
        for _ in range(12):
            q, s, _ = ops.add_rmsnorm_fp8(ctx, z, w, 1e-6)
            torch.cuda.synchronize()
            z = ops.gemm_fp8(ctx, q, s, *weight)
            torch.cuda.synchronize()
        assert torch.equal(y, z)


# ----------------------------------------------------------------------------- refusals
def test_refusals(ctx):
    q, s, wq, ws = _operands(1, 8, 128, 256)
    l, h = ctx.l, ctx.h

    def product(A=q.data_ptr(), lda=256, lds=2, W=wq.data_ptr(), ldc=128, dt=0, M=8, N=128, K=256, C=torch.empty(8, 128, device=DEV)):
        return l.nvc_gemm_fp8(h, A, lda, s.data_ptr(), lds, W, ws.data_ptr(), C.data_ptr() if C is not None else None, ldc, dt, M, N, K, 0)

    assert product() == 0 and product(M=0) == 0
    for bad, code in ((dict(A=None), -1), (dict(C=None), -1), (dict(M=-1), -1), (dict(dt=2), -1), (dict(A=q.data_ptr() + 8), -1), (dict(W=wq.data_ptr() + 1), -1),
                      (dict(K=250), -2), (dict(N=120), -2), (dict(lda=240), -2), (dict(lda=264), -2), (dict(lds=1), -2), (dict(ldc=100), -2), (dict(ldc=132), -2), (dict(N=0), -1)):
        assert product(**bad) == code, bad
        assert b"nvc_gemm_fp8" in l.nvc_last_error(h)
    x = torch.zeros(4, 64, dtype=BF16, device=DEV)
    w = torch.ones(64, dtype=BF16, device=DEV)
    for fn, args, exc in (
        (ops.gemm_fp8, (q, s, wq, ws[:, :1]), ValueError), (ops.gemm_fp8, (q.view(torch.uint8), s, wq, ws), TypeError), (ops.gemm_fp8, (q, s.double(), wq, ws), TypeError),
        (ops.gemm_fp8, (q.cpu(), s, wq, ws), ValueError), (ops.gemm_fp8, (q, s[:4], wq, ws), ValueError), (ops.gemm_fp8, (q[:, :128], s, wq, ws), ValueError),
        (ops.gemm_fp8, (q, s, wq[::2], ws), ValueError),
        (ops.quant_fp8, (x[:, :24],), RuntimeError), (ops.quant_fp8, (x.half(),), TypeError), (ops.quant_fp8, (x.t(),), ValueError),
        (ops.quant_fp8, (x[:, :24], ops.ACT_SILU_MUL), RuntimeError), (ops.quant_fp8, (x, 9), RuntimeError), (ops.quant_fp8, (x[:, 4:36],), RuntimeError),
        (ops.quant_fp8, (x, 0, torch.zeros(3, device=DEV)), TypeError),
        (ops.add_rmsnorm_fp8, (x, w[:32], 1e-6), ValueError), (ops.add_rmsnorm_fp8, (x[:, :32], w[:32], 1e-6), ValueError), (ops.add_rmsnorm_fp8, (x, w, 1e-6, x), TypeError),
        (ops.add_rmsnorm_fp8, (torch.zeros(1, 16400, device=DEV), torch.ones(16400, device=DEV), 1e-6), RuntimeError),
        (ops.quant_fp8_weight, (x[:, :32],), ValueError), (ops.quant_fp8_weight, (torch.zeros(4, 24, device=DEV),), RuntimeError),
    ):
        with pytest.raises(exc):
            fn(ctx, *args)
    qg, sg, wg, wsg = _operands(3, 256, 64, 128, groups=2)
    tiles = torch.zeros(2, dtype=torch.int32, device=DEV)
    assert ops.gemm_fp8_grouped(ctx, qg, sg, wg, wsg, tiles).shape == (256, 64)
    for args in ((qg[:200], sg[:200], wg, wsg, tiles), (qg, sg, wg, wsg, tiles[:1]), (qg, sg, wg[0], wsg[0], tiles), (qg, sg, wg, wsg[:1], tiles)):
        with pytest.raises(ValueError):
            ops.gemm_fp8_grouped(ctx, *args)
    with pytest.raises(TypeError):
        ops.gemm_fp8_grouped(ctx, qg, sg, wg, wsg, tiles.long())


def test_refusals_of_extents_and_routes(ctx):
    """More rows than the last tile's row numbers have room for, and routes that do not exist: refused before anything is read."""
    q, s, wq, ws = _operands(1, 8, 128, 256)
    c = torch.empty(8, 128, dtype=BF16, device=DEV)
    l, h = ctx.l, ctx.h

    def product(M=8, route=0):
        return l.nvc_gemm_fp8_ex(h, q.data_ptr(), 256, s.data_ptr(), 2, wq.data_ptr(), ws.data_ptr(), c.data_ptr(), 128, 0, M, 128, 256, route, 0)

    assert [product(M=2**31 - 1 - d) for d in (0, 128, 255)] == [-2] * 3
    assert [product(route=r) for r in (1, 10, 19, 40, 60, 71, -11)] == [-1] * 7
    assert [product(route=r) for r in (0, 11, 28, 32, 41, 51, 61)] == [0] * 7


def test_rows_of_nothing(ctx):
    """A gather from no rows at all (a step without tokens): every row is one that does not exist."""
    x = torch.empty(0, 256, dtype=BF16, device=DEV)
    q, s = ops.quant_fp8(ctx, x, rows=torch.full((128,), -1, dtype=torch.int32, device=DEV))
    assert q.shape == (128, 256) and not q.view(torch.uint8).any() and torch.equal(s, torch.full((128, 2), 2.0**-126, device=DEV))
    q, s = ops.quant_fp8(ctx, x, act=ops.ACT_SILU_MUL, rows=torch.arange(3, dtype=torch.int32, device=DEV))
    assert q.shape == (3, 128) and not q.view(torch.uint8).any() and torch.equal(s, torch.full((3, 1), 2.0**-126, device=DEV))
    q, s = ops.quant_fp8(ctx, x)
    assert q.shape == (0, 256) and s.shape == (0, 2)


@pytest.mark.parametrize("route,M", [(11, 9), (14, 9), (21, 30), (24, 30), (31, 150), (32, 150), (41, 150), (51, 300), (61, 300)])
def test_weights_converted_in_place_between_products(ctx, route, M):
    """Products fetch weights ahead of their predecessors' end, and weights are converted into the place that the product in front still reads: no product sees another's."""
    N, K, links = 784, 1296, 8
    (q, s), l, h = ops.quant_fp8(ctx, _randn(40, M, K).to(BF16)), ctx.l, ctx.h
    ws = [_randn(50 + i, N, K).to(BF16) for i in range(links)]
    wq, wscale = ops.quant_fp8_weight(ctx, ws[0])
    stream = torch.cuda.current_stream().cuda_stream

    def chain(wait):
        outs = [torch.empty(M, N, dtype=BF16, device=DEV) for _ in ws]
        torch.cuda.synchronize()
        for w, c in zip(ws, outs):
            for call in (lambda: l.nvc_quant_fp8_blocks(h, w.data_ptr(), 0, wq.data_ptr(), wscale.data_ptr(), 1, N, K, stream),
                         lambda: l.nvc_gemm_fp8_ex(h, q.data_ptr(), K, s.data_ptr(), s.shape[1], wq.data_ptr(), wscale.data_ptr(), c.data_ptr(), N, 0, M, N, K, route, stream)):
                assert call() == 0
                if wait:
                    torch.cuda.synchronize()
        torch.cuda.synchronize()
        return outs

    want = chain(True)
    assert not torch.equal(want[0], want[1])
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(chain(False), want))
