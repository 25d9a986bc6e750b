"""The Qwen3 runner over a 4-bit cache: its timing hook, and whole generations against the model in 64 bits."""
import importlib

import numpy as np
import pytest
import torch

from oracle import qwen3_oracle as O
from oracle import synth

pytestmark = pytest.mark.gpu
eng = importlib.import_module("nano-vllm-candle_b200.engine")
CFG = O.MODEL_CONFIGS["qwen3-tiny"]


def _runner(ctx, bits, **kw):
    w = synth.make_weights(CFG, seed=0, norm_jitter=0.1)
    args = dict(num_kvcache_blocks=64, kvcache_block_size=16, max_num_seqs=8, max_num_batched_tokens=512, max_model_len=512)
    return eng.Qwen3ModelRunner.from_weights(ctx, CFG, w.items(), kv_cache_bits=bits, **{**args, **kw})


def _kernels(call):
    from torch.profiler import ProfilerActivity, profile
    with profile(activities=[ProfilerActivity.CUDA]) as p:
        call()
        torch.cuda.synchronize()
    return {e.key for e in p.key_averages()}


def test_timed_operators_are_the_step_s_own(ctx):
    """What time_op times over a 4-bit cache is what a decode step runs, and the cached rows stay as they are."""
    table, at = np.array([[3, 9, 1]], dtype=np.int32), lambda a, b: [int((3, 9, 1)[t // 16]) * 16 + t % 16 for t in range(a, b)]          # noqa: E731
    logits = []
    for timed in (False, True):
        runner = _runner(ctx, 4, use_cuda_graph=False)
        runner.prefill(list(range(5, 35)), range(30), [0, 30], at(0, 30))
        step = _kernels(lambda: runner.decode([7], [30], at(30, 31), table, [31]))
        if timed:
            for op, part in (("qk_norm_rope", "store_fp4_kernel"), ("paged_decode", "attn_kernel")):
                mine = [k for k in _kernels(lambda: runner.time_op(op, 2)) if part in k]
                assert len(mine) == 1 and mine[0] in step, (op, mine, step)
                ms, launches = runner.time_op(op, 3)
                assert ms > 0 and launches == 3 * CFG.num_hidden_layers
        runner.decode([11], [31], at(31, 32), table, [32])
        logits.append(runner.last_logits(1).copy())
        runner.close()
    assert np.array_equal(*logits)
