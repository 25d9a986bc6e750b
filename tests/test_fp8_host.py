"""The 8-bit entry points refuse before they reach a device: no context, tensors that are not on one."""
import importlib
import types

import pytest
import torch

ops = importlib.import_module("nano-vllm-candle_b200.ops")
_lib = importlib.import_module("nano-vllm-candle_b200._lib")


def test_no_context_is_an_invalid_argument():
    l = _lib.lib()
    assert l.nvc_gemm_fp8(None, 16, 128, 16, 1, 16, 16, 16, 128, 0, 1, 128, 128, None) == -1
    assert l.nvc_gemm_fp8_grouped(None, 16, 128, 16, 1, 16, 16, 16, 128, 0, 128, 128, 128, 16, 1, 0, None) == -1
    assert l.nvc_quant_fp8_rows(None, 16, 0, 128, 1, 0, 0, None, None, 16, 128, 16, 1, 1, 128, None) == -1
    assert l.nvc_quant_fp8_blocks(None, 16, 0, 16, 16, 1, 128, 128, None) == -1
    assert l.nvc_add_rmsnorm_fp8(None, 16, 0, None, None, 16, 0, 1e-6, 16, 128, 16, 1, None, 1, 128, None) == -1
    assert l.nvc_last_error(None)


def test_tensors_elsewhere_are_refused():
    ctx = types.SimpleNamespace(device=0, h=None, l=None)      # nothing of the library is reached
    x, w = torch.zeros(4, 128), torch.ones(128)
    q, s = torch.zeros(4, 128, dtype=torch.uint8).view(ops.FP8), torch.ones(4, 1)
    for call in (lambda: ops.quant_fp8(ctx, x), lambda: ops.quant_fp8_weight(ctx, x), lambda: ops.add_rmsnorm_fp8(ctx, x, w, 1e-6),
                 lambda: ops.gemm_fp8(ctx, q, s, q, s[:1]), lambda: ops.gemm_fp8_grouped(ctx, q, s, q[None], s[None, :1], torch.zeros(1, dtype=torch.int32))):
        with pytest.raises(ValueError, match="must be on cuda:0"):
            call()
    with pytest.raises(TypeError):
        ops.quant_fp8(ctx, x.half())
