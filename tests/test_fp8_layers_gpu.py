"""The linear layers, the norm and the gated unit in 8 bits: the same bits as the kernels' own entry points, near what the bf16 layers give."""
import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu
L = importlib.import_module("nano-vllm-candle_b200.layers")
ops = importlib.import_module("nano-vllm-candle_b200.ops")
BF16 = torch.bfloat16


def _bits(t):
    return t.view(torch.uint8) if t.dtype == ops.FP8 else t


def test_feed_forward_of_layers(ctx):
    g = torch.Generator(device="cuda").manual_seed(3)
    H, I, shape = 512, 768, (2, 17, 512)
    x, res = (torch.randn(shape, generator=g, device="cuda") for _ in range(2))
    x = x.to(BF16)
    gate, up, down = (torch.randn(n, k, generator=g, device="cuda") * k ** -0.5 for n, k in ((I, H), (I, H), (H, I)))

    def layers():
        gu, dn = L.MergedColumnParallelLinear(ctx, H, [I, I]), L.RowParallelLinear(ctx, I, H)
        gu.load_weights(gate, loaded_shard_id=0)
        gu.load_weights(up, loaded_shard_id=1)
        dn.load_weights(down)
        return gu, dn

    norm, act = L.RMSNorm(ctx, H), L.SiluAndMul(ctx)
    gu, dn = layers()
    want_res = None
    n, want_res = norm.forward(x, res)
    want = dn.forward(act.forward(gu.forward(n)))
    gu8, dn8 = (layer.to_fp8() for layer in layers())
    assert gu8.weight is None and gu8.weight_fp8[0].shape == (2 * I, H)
    rows, new_res = norm.forward_fp8(x, res)
    assert torch.equal(new_res, want_res)
    got = dn8.forward(act.forward_fp8(gu8.forward(rows)))
    # the steps by themselves
    q, s, _ = ops.add_rmsnorm_fp8(ctx, x.reshape(-1, H), norm.weight, norm.eps, residual=res.reshape(-1, H))
    w1, w2 = (ops.quant_fp8_weight(ctx, w.to(BF16)) for w in (torch.cat([gate, up]), down))
    h = ops.gemm_fp8(ctx, q, s, *w1)
    direct = ops.gemm_fp8(ctx, *ops.quant_fp8(ctx, h, act=ops.ACT_SILU_MUL), *w2)
    assert torch.equal(got, direct)
    # four operands in 8 bits, each 2^-4 / sqrt(3) of its norm off at most: two products of 5.1 % each, the unit between them with two factors and a slope of at most 1.1
    far = (got.float() - want.reshape(-1, H).float()).norm() / want.float().norm()
    assert float(far) < 0.16
    # a tensor in place of rows, more than two dimensions, no residual
    plain, none = norm.forward_fp8(x)
    assert none is None and torch.equal(_bits(plain[0]), _bits(ops.add_rmsnorm_fp8(ctx, x.reshape(-1, H), norm.weight, norm.eps)[0]))
    y = gu8.forward(x)
    assert y.shape == (2, 17, 2 * I) and torch.equal(y.reshape(-1, 2 * I), ops.gemm_fp8(ctx, *ops.quant_fp8(ctx, x.reshape(-1, H)), *w1))


def test_a_checkpoints_own_weights_and_refusals(ctx):
    w = torch.randn(300, 256, device="cuda")
    q, s = ops.quant_fp8_weight(ctx, w)
    lin = L.ReplicatedLinear(ctx, 256, 304)
    with pytest.raises(RuntimeError):
        lin.to_fp8()
    with pytest.raises(ValueError):
        lin.load_fp8(q, s[:2])
    with pytest.raises(ValueError):
        lin.load_fp8(w, s)
    q, s = ops.quant_fp8_weight(ctx, torch.randn(304, 256, device="cuda"))
    lin.load_fp8(q, s.to(BF16))
    x = torch.randn(5, 256, device="cuda", dtype=BF16)
    rows = ops.quant_fp8(ctx, x)
    assert torch.equal(lin.forward(x), ops.gemm_fp8(ctx, *rows, q, s.to(BF16).float()))
    lin.load_weights(torch.randn(304, 256, device="cuda"))          # back to bf16
    with pytest.raises(ValueError):
        lin.forward(rows)
    assert lin.forward(x).shape == (5, 304)


def test_gated_unit_of_any_layout(ctx):
    """Rows that SiluAndMul.forward takes: a transposed view, rows at an odd distance, three dimensions."""
    act = L.SiluAndMul(ctx)
    base = torch.randn(256, 24, device="cuda").to(BF16)
    for x in (base.t(), torch.randn(7, 261, device="cuda").to(BF16)[:, 3:259], torch.randn(2, 5, 256, device="cuda").to(BF16).transpose(0, 1)):
        whole = x.reshape(-1, 256).contiguous()
        want, got = ops.quant_fp8(ctx, whole, act=ops.ACT_SILU_MUL), act.forward_fp8(x)
        assert all(torch.equal(_bits(a), _bits(b)) for a, b in zip(want, got))
