"""What the entry points of the 4-bit cache decide before they reach a device, with a library that only notes its calls."""
import importlib
import types

import pytest
import torch

import fp4_ref as ref

ops = importlib.import_module("nano-vllm-candle_b200.ops")
layers = importlib.import_module("nano-vllm-candle_b200.layers")
_lib = importlib.import_module("nano-vllm-candle_b200._lib")
BF16, F32, I32, U8 = torch.bfloat16, torch.float32, torch.int32, torch.uint8
BIG = 2 ** 32 + 128                              # 128, if only its lowest 32 bits are looked at


class _Calls(list):
    def __getattr__(self, name):
        def call(*args):
            if name == "nvc_attn_fp4_workspace_bytes":
                return 0
            self.append((name, args))
            return 0
        return call


@pytest.fixture
def fake(monkeypatch):
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda device: 0, raising=False)
    return types.SimpleNamespace(device=-1, h=0, l=_Calls(), tp_size=1, tp_rank=0)


def _meta(*shape, dtype=BF16):
    return torch.empty(*shape, dtype=dtype, device="meta")


def _far(n, w, dtype=BF16):
    return torch.empty_strided((n, w), (BIG, 1), dtype=dtype, device="meta")


def _cache(blocks=3, kv=2, bs=16):
    return ops.Fp4Cache(*(_meta(blocks, kv, bs, w, dtype=U8) for w in (64, 8, 64, 8)))


def _ints(*shape):
    return _meta(*shape, dtype=I32)


def test_no_context_is_an_invalid_argument():
    l = _lib.lib()
    assert l.nvc_qk_norm_rope_store_fp4(None, 16, 640, None, None, 1e-6, 16, 8, 16, 16, None, None, 0, 1, 1, None) == -1
    assert l.nvc_store_kvcache_fp4(None, 16, 128, 16, 128, None, 16, 1, None) == -1
    assert l.nvc_read_kvcache_fp4(None, None, 16, 16, 16, 16, 16, 1, None) == -1
    assert l.nvc_paged_decode_attn_fp4(None, 16, 128, None, 16, 1, 16, 1, 1, 1.0, 16, 128, None, 0, None) == -1
    assert l.nvc_prefill_attn_paged_fp4(None, 16, 128, None, 16, 1, 16, 16, 1, 1, 1, 1, 1.0, 16, 128, None, 0, None) == -1
    assert l.nvc_last_error(None)


def test_a_cache_s_parts_belong_together():
    k, s = torch.zeros(3, 2, 16, 64, dtype=U8), torch.zeros(3, 2, 16, 8, dtype=U8)
    c = ops.Fp4Cache(k, s, k, s)
    assert (c.num_blocks, c.kv, c.block_size) == (3, 2, 16)
    for parts in ((k[..., :32], s, k, s), (k, s[:2], k, s), (k, s, k[:, :1], s), (k, s, k, s.transpose(0, 1)), (k[:, :, :8], s[:, :, :8], k[:, :, :8], s[:, :, :8]),
                  (k[:0], s[:0], k[:0], s[:0]), (k[0], s[0], k[0], s[0]), (k, s, k.to("meta"), s)):
        with pytest.raises(ValueError):
            ops.Fp4Cache(*parts)
    with pytest.raises(TypeError, match="uint8"):
        ops.Fp4Cache(k, s.float(), k, s)
    with pytest.raises(ValueError, match="31 bits"):
        _cache(2 ** 27, 1, 16)


def _calls(ctx, **over):
    """Each entry point with arguments that fit, and some of them replaced."""
    c, a = _cache(), dict(qkv=_meta(5, 8 * 128), w=_meta(128), table=_meta(9, 128, dtype=F32), pos=_ints(5), slots=_ints(5), k=_meta(5, 256), v=_meta(5, 256), q=_meta(5, 512),
                          tables=_ints(5, 4), lens=_ints(5), cu=_ints(6), q_out=None, nh=4)
    a.update(over)
    c = a.get("cache", c)
    return {
        "norm": lambda: ops.qk_norm_rope_store_fp4(ctx, a["qkv"], a["w"], a["w"], 1e-6, a["table"], a["pos"], a["nh"], c, a["slots"], q_out=a["q_out"]),
        "store": lambda: ops.store_kvcache_fp4(ctx, a["k"], a["v"], c, a["slots"]),
        "read": lambda: ops.read_kvcache_fp4(ctx, c, a["slots"]),
        "decode": lambda: ops.paged_decode_attn_fp4(ctx, a["q"], c, a["tables"], a["lens"], a["nh"], 0.1, out=a.get("out")),
        "prefill": lambda: ops.prefill_attn_paged_fp4(ctx, a["q"], c, a["tables"], a["lens"], a["cu"], a.get("most", 3), a["nh"], 0.1, out=a.get("out")),
    }


def test_calls_that_fit_reach_the_library(fake):
    for call in _calls(fake).values():
        call()
    assert [name for name, _ in fake.l] == ["nvc_qk_norm_rope_store_fp4", "nvc_store_kvcache_fp4", "nvc_read_kvcache_fp4", "nvc_paged_decode_attn_fp4", "nvc_prefill_attn_paged_fp4"]


@pytest.mark.parametrize("where,over", [
    ("norm", dict(qkv=_meta(5, 7 * 128))), ("norm", dict(qkv=_meta(5, 8 * 128, dtype=F32))), ("norm", dict(w=_meta(64))), ("norm", dict(table=_meta(9, 64, dtype=F32))),
    ("norm", dict(table=_meta(9, 128))), ("norm", dict(pos=_ints(4))), ("norm", dict(pos=_meta(5, dtype=torch.int64))), ("norm", dict(slots=_ints(6))), ("norm", dict(q_out=_meta(5, 4 * 100))),
    ("norm", dict(q_out=_meta(4, 512))), ("norm", dict(nh=5)), ("norm", dict(qkv=_meta(8 * 128, 5).t())), ("norm", dict(cache=(1, 2, 3, 4))),
    ("store", dict(k=_meta(5, 128))), ("store", dict(v=_meta(4, 256))), ("store", dict(k=_meta(5, 256, dtype=torch.float16))), ("store", dict(slots=_ints(4))), ("store", dict(slots=_ints(10)[::2])),
    ("read", dict(slots=_meta(5, dtype=torch.int64))), ("read", dict(slots=_ints(5, 1))),
    ("decode", dict(q=_meta(5, 500))), ("decode", dict(q=_meta(5, 512, dtype=F32))), ("decode", dict(tables=_ints(4, 4))), ("decode", dict(tables=_ints(5))), ("decode", dict(lens=_ints(4))),
    ("decode", dict(tables=_ints(4, 5).t())), ("decode", dict(out=_meta(5, 511))), ("decode", dict(out=_meta(5, 512, dtype=F32))),
    ("prefill", dict(cu=_ints(5))), ("prefill", dict(cu=_ints(0))), ("prefill", dict(lens=_ints(6))), ("prefill", dict(q=_meta(5, 511))), ("prefill", dict(cu=_meta(6, dtype=torch.int64)))])
def test_arguments_that_do_not_fit_are_refused(fake, where, over):
    with pytest.raises((ValueError, TypeError)):
        _calls(fake, **over)[where]()
    assert not fake.l


def test_tensors_elsewhere_are_refused():
    ctx = types.SimpleNamespace(device=0, h=None, l=None)      # nothing of the library is reached
    for call in _calls(ctx).values():
        with pytest.raises(ValueError, match="must be on cuda:0"):
            call()


@pytest.mark.parametrize("where,over", [
    ("norm", dict(qkv=_far(5, 8 * 128))), ("norm", dict(q_out=_far(5, 512))), ("norm", dict(table=_meta(BIG, 128, dtype=F32))), ("store", dict(k=_far(5, 256))), ("store", dict(v=_far(5, 256))),
    ("read", dict(slots=_ints(BIG))), ("decode", dict(q=_far(5, 512))), ("decode", dict(out=_far(5, 512))), ("decode", dict(tables=_ints(5, BIG))), ("prefill", dict(q=_far(5, 512))),
    ("prefill", dict(most=BIG))])
def test_sizes_beyond_31_bits_are_refused(fake, where, over):
    with pytest.raises(ValueError, match="31 bits"):
        _calls(fake, **over)[where]()
    assert not fake.l


def test_no_rows_reach_nothing(fake):
    none = dict(qkv=_meta(0, 8 * 128), pos=_ints(0), slots=_ints(0), k=_meta(0, 256), v=_meta(0, 256), q=_meta(0, 512), tables=_ints(0, 4), lens=_ints(0), cu=_ints(1))
    got = {name: call() for name, call in _calls(fake, **none).items()}
    assert not fake.l and got["decode"].shape == got["prefill"].shape == (0, 512) and got["read"][0].shape == (0, 2, 128) and got["read"][1].shape == (0, 2, 8)


def test_one_row_has_its_own_width_as_distance(fake):
    """A row whose stride says nothing: its width goes on."""
    q = torch.zeros(512, 1, dtype=BF16).t()
    c = ops.Fp4Cache(*(torch.zeros(1, 2, 16, w, dtype=U8) for w in (64, 8, 64, 8)))
    fake.device = -1
    ops.paged_decode_attn_fp4(fake, q, c, torch.zeros(1, 4, dtype=I32), torch.zeros(1, dtype=I32), 4, 0.1, out=torch.zeros(512, 1, dtype=BF16).t())
    args = fake.l[0][1]
    assert args[2] == 512 and args[11] == 512


def test_the_definition_s_own_ends():
    """The reference of the tests: ties, the ends of the range, the relative error that 4 bits leave."""
    x = torch.zeros(1, 128)
    x[0, :8] = torch.tensor([6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    c, s = ref.to_fp4(x)
    assert c[0, :8].tolist() == [6, 0, 0.5, 1, 1.5, 2, 3, 4] and ref.SCALES[s[0, 0]] == 1 and not s[0, 1:].any()
    x = torch.randn(64, 128, generator=torch.Generator().manual_seed(0))
    c, s = ref.to_fp4(x)
    back = (c.unflatten(-1, (8, 16)) * ref.SCALES[s][..., None]).flatten(-2)
    assert 0.05 < float((back - x).norm() / x.norm()) < 0.12
    top = torch.full((1, 128), 1e6)
    c, s = ref.to_fp4(top)
    assert bool((c == 6).all()) and bool((ref.SCALES[s] == 10240).all())
