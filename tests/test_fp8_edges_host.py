"""What the 8-bit entry points and layers decide before they reach a device, with a library that only notes its calls."""
import importlib
import types

import pytest
import torch

ops = importlib.import_module("nano-vllm-candle_b200.ops")
E4M3 = torch.float8_e4m3fn


class _Calls(list):
    def __getattr__(self, name):
        def call(*args):
            self.append((name, args))
            return 0
        return call


@pytest.fixture
def fake(monkeypatch):
    """A context on no device: its tensors have memory or none ("meta"), its library notes calls."""
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda device: 0, raising=False)
    return types.SimpleNamespace(device=-1, h=0, l=_Calls(), tp_size=1, tp_rank=0)


def _meta(*shape, dtype=torch.bfloat16):
    return torch.empty(*shape, dtype=dtype, device="meta")


def test_one_row_has_its_own_width_as_distance(fake):
    """A column seen as a row: what its stride says is not handed on."""
    x, q, s, c = torch.zeros(1, 256), torch.zeros(256, 1, dtype=torch.uint8).view(E4M3).t(), torch.zeros(2, 1).t(), torch.zeros(160, 1).t()
    assert q.stride() == (1, 1) and s.stride() == (1, 1) and c.stride() == (1, 1)
    ops.quant_fp8(fake, x, q=q, scale=s)
    ops.add_rmsnorm_fp8(fake, x, torch.ones(256), 1e-6, q=q, scale=s)
    ops.gemm_fp8(fake, q, s, torch.zeros(160, 256, dtype=torch.uint8).view(E4M3), torch.zeros(2, 2), out=c)
    (_, rows), (_, norm), (_, product) = fake.l
    assert (rows[10], rows[12]) == (256, 2) and (norm[9], norm[11]) == (256, 2) and (product[2], product[4], product[8]) == (256, 2, 160)


BIG = 2 ** 32 + 128                              # 128, if only its lowest 32 bits are looked at


def test_sizes_beyond_31_bits_are_refused(fake):
    """Sizes and strides go to the library as 32-bit numbers: one that does not fit is refused, where its low bits named another call."""
    wq, ws = _meta(128, 256, dtype=E4M3), _meta(1, 2, dtype=torch.float32)
    far = lambda n, w, dtype: torch.empty_strided((n, w), (BIG, 1), dtype=dtype, device="meta")
    f32 = torch.float32
    for call in (
        lambda: ops.quant_fp8(fake, _meta(BIG, 256)),
        lambda: ops.quant_fp8(fake, far(4, 256, torch.bfloat16)),
        lambda: ops.quant_fp8(fake, _meta(BIG, 256), rows=_meta(4, dtype=torch.int32)),
        lambda: ops.quant_fp8(fake, _meta(4, 256), rows=_meta(BIG, dtype=torch.int32)),
        lambda: ops.quant_fp8(fake, _meta(1, BIG)),
        lambda: ops.quant_fp8(fake, _meta(4, 256), q=far(4, 256, E4M3)),
        lambda: ops.quant_fp8(fake, _meta(4, 256), scale=far(4, 2, f32)),
        lambda: ops.quant_fp8_weight(fake, _meta(BIG, 256)),
        lambda: ops.quant_fp8_weight(fake, _meta(BIG, 16, 256)),
        lambda: ops.add_rmsnorm_fp8(fake, _meta(BIG, 256), _meta(256), 1e-6),
        lambda: ops.add_rmsnorm_fp8(fake, _meta(4, 256), _meta(256), 1e-6, q=far(4, 256, E4M3)),
        lambda: ops.gemm_fp8(fake, _meta(BIG, 256, dtype=E4M3), _meta(BIG, 2, dtype=f32), wq, ws),
        lambda: ops.gemm_fp8(fake, far(4, 256, E4M3), _meta(4, 2, dtype=f32), wq, ws),
        lambda: ops.gemm_fp8(fake, _meta(4, 256, dtype=E4M3), _meta(4, 2, dtype=f32), _meta(BIG, 256, dtype=E4M3), _meta(BIG // 128, 2, dtype=f32)),
        lambda: ops.gemm_fp8(fake, _meta(4, 256, dtype=E4M3), _meta(4, 2, dtype=f32), wq, ws, out=far(4, 128, f32)),
        lambda: ops.gemm_fp8_grouped(fake, _meta(BIG, 256, dtype=E4M3), _meta(BIG, 2, dtype=f32), wq[None], ws[None], _meta(BIG // 128, dtype=torch.int32)),
        lambda: ops.gemm_fp8_grouped(fake, _meta(128, 256, dtype=E4M3), _meta(128, 2, dtype=f32), _meta(BIG, 128, 256, dtype=E4M3), _meta(BIG, 1, 2, dtype=f32),
                                     _meta(1, dtype=torch.int32)),
    ):
        with pytest.raises(ValueError, match="31 bits"):
            call()
    assert not fake.l
    ops.quant_fp8(fake, _meta(128, 256))
    assert len(fake.l) == 1


# ----------------------------------------------------------------------------- layers
layers = importlib.import_module("nano-vllm-candle_b200.layers")
tp = importlib.import_module("nano-vllm-candle_b200.tp")


def _loaded(ctx, kind):
    """A layer of 64 inputs with its weight loaded shard by shard, and how to load its first shard again."""
    full = torch.randn(96, 64)
    if kind == "merged":
        layer = layers.MergedColumnParallelLinear(ctx, 64, [48, 48])
        layer.load_weights(full[:48], loaded_shard_id=0)
        layer.load_weights(full[48:], loaded_shard_id=1)
        return layer, lambda w: layer.load_weights(w, loaded_shard_id=0), full
    layer = layers.QKVParallelLinear(ctx, 64, 16, 4, 1)
    for name, w in zip("qkv", full.split([64, 16, 16])):
        layer.load_qkv_weight(w, name)
    return layer, lambda w: layer.load_qkv_weight(w, "q"), full


@pytest.mark.parametrize("kind", ["merged", "qkv"])
@pytest.mark.parametrize("how", ["to_fp8", "load_fp8"])
def test_8_bits_give_up_the_loaded_shards(fake, kind, how):
    """Merged layers hold their shards, views of whole tensors: converted, they hold none of them; a later load starts with all of them."""
    import gc
    import weakref
    layer, again, full = _loaded(fake, kind)
    parts = [weakref.ref(p) for p in (layer._parts if kind == "merged" else layer._parts.values())]
    assert all(p() is not None for p in parts)
    if how == "to_fp8":
        assert layer.to_fp8() is layer
    else:
        layer.load_fp8(torch.zeros(96, 64, dtype=torch.uint8).view(E4M3), torch.ones(1, 1))
    gc.collect()
    assert layer.weight is None and layer.weight_fp8[0].shape == (96, 64) and not any(p() is not None for p in parts)
    again(torch.randn(48 if kind == "merged" else 64, 64))
    assert layer.weight is None and layer.weight_fp8 is not None          # the other shards are gone
    if kind == "merged":
        layer.load_weights(torch.randn(48, 64), loaded_shard_id=1)
    else:
        layer.load_weights(torch.randn(96, 64))
    assert layer.weight.shape == (96, 64) and layer.weight_fp8 is None


def _layer_of(ctx, kind, size, rank):
    cfg = tp.TPConfig(size, rank, 0)
    return {"replicated": lambda: layers.ReplicatedLinear(ctx, 256, 384),
            "column": lambda: layers.ColumnParallelLinear(ctx, 256, 384, cfg),
            "merged": lambda: layers.MergedColumnParallelLinear(ctx, 256, [256, 128], cfg),
            "qkv": lambda: layers.QKVParallelLinear(ctx, 256, 32, 8, 2, cfg),
            "row": lambda: layers.RowParallelLinear(ctx, 256, 384, cfg)}[kind]()


@pytest.mark.parametrize("kind", ["replicated", "column", "merged", "qkv", "row"])
@pytest.mark.parametrize("size", [1, 2])
def test_load_fp8_takes_this_ranks_share_alone(fake, kind, size):
    """Another layer's weight, a whole one for a rank's share, one that lies on its side, wrong scales, another device: refused, and the weight of before stays."""
    n, k = {"replicated": (384, 256), "row": (384, 256 // size)}.get(kind, (384 // size, 256))
    weight = lambda n, k, device="cpu": torch.zeros(n, k, dtype=torch.uint8, device=device).view(E4M3)
    scale = lambda n, k, device="cpu": torch.ones((n + 127) // 128, (k + 127) // 128, device=device)
    layer = _layer_of(fake, kind, size, size - 1)
    before = torch.zeros(n, k, dtype=torch.bfloat16)
    layer._set(before, None)
    others = {(384, 256), (256, 384), (192, 256), (384, 128), (n + 128, k), (n, k + 128), (n // 2, k)} - {(n, k)}
    for shape in sorted(others):
        with pytest.raises(ValueError):
            layer.load_fp8(weight(*shape), scale(*shape))
    for w, s in ((weight(n, k), scale(n + 128, k)), (weight(n, k), scale(n, k).T.contiguous()[:, :1]), (weight(n, k).view(torch.uint8), scale(n, k)),
                 (weight(n, k, "meta"), scale(n, k)), (weight(n, k)[None], scale(n, k)), (weight(n, k), scale(n, k).to(torch.int32))):
        if w.device.type == "meta":
            fake.device = 0                      # a tensor of no device of ours
        with pytest.raises(ValueError):
            layer.load_fp8(w, s)
        fake.device = -1
    assert torch.equal(layer.weight, before) and layer.weight_fp8 is None
    layer.load_fp8(weight(n, k), scale(n, k).to(torch.bfloat16))
    assert layer.weight is None and layer.weight_fp8[1].dtype == torch.float32
    kept = layer.weight_fp8
    with pytest.raises(ValueError):
        layer.load_fp8(weight(k, n + 16), scale(k, n + 16))
    assert layer.weight_fp8 is kept


@pytest.mark.parametrize("n,k", [(300, 256), (304, 264)])
def test_to_fp8_keeps_a_weight_that_no_product_takes(fake, n, k):
    """Products take sizes that are multiples of 16: refused where the bf16 weight is still there, not at the first product."""
    layer = layers.ReplicatedLinear(fake, k, n)
    weight = torch.randn(n, k).to(torch.bfloat16)
    layer.load_weights(weight)
    with pytest.raises(ValueError, match="multiples of 16"):
        layer.to_fp8()
    assert torch.equal(layer.weight, weight) and layer.weight_fp8 is None
    with pytest.raises(ValueError, match="multiples of 16"):
        layer.load_fp8(torch.zeros(n, k, dtype=torch.uint8).view(E4M3), torch.ones(3, 3 if k > 256 else 2))
    assert torch.equal(layer.weight, weight) and not fake.l
