"""The 4-bit cache behind the layer and runner interfaces: Attention with an Fp4Cache, Qwen3ModelRunner and LLMEngine with kv_cache_bits=4."""
import importlib

import numpy as np
import pytest
import torch

import fp4_ref as ref
from oracle import qwen3_oracle as O
from oracle import synth

pytestmark = pytest.mark.gpu
ops = importlib.import_module("nano-vllm-candle_b200.ops")
eng = importlib.import_module("nano-vllm-candle_b200.engine")
L = importlib.import_module("nano-vllm-candle_b200.layers")
BF16, F64, I32 = torch.bfloat16, torch.float64, torch.int32


def _i(*v):
    return torch.tensor(v, dtype=I32, device="cuda")


def test_attention_layer(ctx):
    """A prompt attends to its own rows as without a cache, a portion behind it and a decode step to the cached ones."""
    nh, kv, hd, bs = 4, 2, 128, 16
    g = torch.Generator().manual_seed(6)
    attn = L.Attention(ctx, nh, hd, hd ** -0.5, kv, block_size=bs)
    attn.fp4_cache = ops.Fp4Cache.zeros(8, bs, kv)
    table, done = _i(5, 2, 7, 0)[None], 0
    for n, kind in ((21, "prompt"), (9, "portion"), (1, "decode")):
        q, k, v = (torch.randn(n, h * hd, generator=g).to(BF16).cuda() for h in (nh, kv, kv))
        pos = torch.arange(done, done + n, device="cuda")
        slots, done = (table[0, pos // bs] * bs + pos % bs).to(I32), done + n
        lens, cu = _i(done), _i(0, n)
        if kind == "prompt":
            L.set_context(is_prefill=True, cu_seqlens=cu, max_seqlen=n, slot_mapping=slots)
            assert torch.equal(attn.forward(q, k, v), ctx.prefill_attn(q, k, v, cu, n, nh, kv, hd, hd ** -0.5))
            continue
        L.set_context(is_prefill=kind == "portion", cu_seqlens=cu, max_seqlen=n, slot_mapping=slots, context_lens=lens, block_tables=table)
        got = attn.forward(q, k, v)
        want, far = ref.attention(q, attn.fp4_cache, table.cpu(), [done], [n], hd ** -0.5, nh)
        assert bool(((got.cpu().to(F64).view(want.shape) - want).abs() <= far).all())
    attn.k_cache = torch.zeros(8, bs, kv, hd, dtype=BF16, device="cuda")
    with pytest.raises(RuntimeError, match="one cache"):
        attn.forward(q, k, v)


CFG = O.MODEL_CONFIGS["qwen3-tiny"]


def _runner(ctx, bits, **kw):
    w = synth.make_weights(CFG, seed=0, norm_jitter=0.1)
    args = dict(num_kvcache_blocks=64, kvcache_block_size=16, max_num_seqs=8, max_num_batched_tokens=512, max_model_len=512)
    return eng.Qwen3ModelRunner.from_weights(ctx, CFG, w.items(), kv_cache_bits=bits, **{**args, **kw}), {k: v.to(F64) for k, v in w.items()}


class _Model:
    """Qwen3 in 64 bits, a step at a time, with the cached rows of every layer as they are or as their 4-bit forms."""

    def __init__(self, w, fp4):
        self.w, self.fp4, self.rows = w, fp4, [None] * CFG.num_hidden_layers
        self.nh, self.kv, self.hd = CFG.num_attention_heads, CFG.num_key_value_heads, CFG.head_dim

    def _norm(self, x, w):
        return x / torch.sqrt(x.square().mean(-1, keepdim=True) + CFG.rms_norm_eps) * w

    def _turn(self, x, pos):
        f = CFG.rope_theta ** (-torch.arange(0, self.hd, 2, dtype=F64) / self.hd)
        c, s = torch.cos(pos[:, None] * f)[:, None], torch.sin(pos[:, None] * f)[:, None]
        a, b = x.chunk(2, -1)
        return torch.cat((a * c - b * s, b * c + a * s), -1)

    def _kept(self, x):
        if not self.fp4:
            return x
        c, s = ref.to_fp4(x.to(BF16))
        return (c.unflatten(-1, (8, 16)) * ref.SCALES[s][..., None]).flatten(-2)

    def step(self, ids, first):
        """Logits of the last token; a step from position 0 attends to its own rows, the others to the cached ones."""
        w, n = self.w, len(ids)
        x, pos = w["model.embed_tokens.weight"][torch.tensor(ids)], torch.arange(first, first + n, dtype=F64)
        for i in range(CFG.num_hidden_layers):
            p = f"model.layers.{i}."
            h = self._norm(x, w[p + "input_layernorm.weight"])
            q, k, v = ((h @ w[p + f"self_attn.{c}_proj.weight"].T).view(n, -1, self.hd) for c in "qkv")
            q = self._turn(self._norm(q, w[p + "self_attn.q_norm.weight"]), pos)
            k = self._turn(self._norm(k, w[p + "self_attn.k_norm.weight"]), pos)
            new = torch.stack((self._kept(k), self._kept(v)))
            self.rows[i] = new if first == 0 else torch.cat((self.rows[i], new), 1)
            ks, vs = (k, v) if first == 0 else self.rows[i]
            group = self.nh // self.kv
            s = torch.einsum("qhd,khd->hqk", q, ks.repeat_interleave(group, 1)) * self.hd ** -0.5
            s = s.masked_fill(torch.arange(first + n)[None] > torch.arange(first, first + n)[:, None], -float("inf"))
            o = torch.einsum("hqk,khd->qhd", torch.softmax(s, -1), vs.repeat_interleave(group, 1)).flatten(1)
            x = x + o @ w[p + "self_attn.o_proj.weight"].T
            h = self._norm(x, w[p + "post_attention_layernorm.weight"])
            gate, up = h @ w[p + "mlp.gate_proj.weight"].T, h @ w[p + "mlp.up_proj.weight"].T
            x = x + (gate / (1 + torch.exp(-gate)) * up) @ w[p + "mlp.down_proj.weight"].T
        head = w.get("lm_head.weight", w["model.embed_tokens.weight"])
        return self._norm(x[-1], w["model.norm.weight"]) @ head.T


def test_runner_steps(ctx):
    """A prompt's logits are those with a bf16 cache, bit by bit; a portion's and decode steps' are those of the model with 4-bit rows.

    Bound: what the bf16 path is held to elsewhere (2e-2), and half of what the 4 bits themselves move.  A cached row has gone through three roundings to bf16 (2^-9 of a number in the mean)
    in each of up to three layers, sqrt(9) 2^-9 = 0.6 %; steps between codes are a third of a number, so that 1.8 % of the codes are others, each by a step, where the format's own roundings are off
    by a step / sqrt(12) at every place: sqrt(12 * 0.018) = 0.46 of what those move."""
    runner, w = _runner(ctx, 4)
    wide, _ = _runner(ctx, 16)
    prompt = synth.make_prompts(1, 45, CFG.vocab_size, 7)[0]
    table = np.array([[3, 9, 1, 12, 30]], dtype=np.int32)
    four, plain = _Model(w, True), _Model(w, False)
    at = lambda a, b: [int(table[0, t // 16]) * 16 + t % 16 for t in range(a, b)]          # noqa: E731

    def near(got, first, ids):
        a, b = four.step(ids, first), plain.step(ids, first)
        moved = float((a - b).abs().max())
        off = float((got - a).abs().max())
        assert off <= 2e-2 + moved / 2, f"{off} with {moved} moved by the 4 bits"
        return float((got - a).norm()), float((got - b).norm())

    for r in (runner, wide):
        r.prefill(prompt[:30], range(30), [0, 30], at(0, 30))
    got = torch.from_numpy(runner.last_logits(1))[0].to(F64)
    assert torch.equal(got, torch.from_numpy(wide.last_logits(1))[0].to(F64))
    near(got, 0, prompt[:30])
    runner.step_mixed(prompt[30:45], range(30, 45), [0, 15], at(30, 45), table, [45], 0)
    nearer = [near(torch.from_numpy(runner.last_logits(1))[0].to(F64), 30, prompt[30:45])]
    for i, t in enumerate((5, 77, 1234, 9, 300)):
        runner.decode([t], [45 + i], at(45 + i, 46 + i), table, [46 + i])
        nearer.append(near(torch.from_numpy(runner.last_logits(1))[0].to(F64), 45 + i, [t]))
    assert sum(a for a, _ in nearer) < sum(b for _, b in nearer)                            # the 4-bit rows are what it reads
    runner.close()
    wide.close()


@pytest.mark.parametrize("prefix,chunked", [(False, False), (True, False), (True, True)])
def test_engine_generates(ctx, prefix, chunked):
    """Whole generations over a small pool (sequences are put back and begun again on the way), with cached prefixes and chunked prompts, repeat themselves."""
    runner, _ = _runner(ctx, 4, num_kvcache_blocks=24)
    prompts = [synth.make_prompts(1, n, CFG.vocab_size, 100 + n)[0] for n in (7, 33, 70, 50)]
    prompts.append(prompts[2][:64] + [5, 6, 7])
    runs = []
    for _ in range(2):
        sch = eng.Scheduler(eng.SchedulerConfig(4, 64 if chunked else 512, CFG.eos_token_id, 24, 16, enable_prefix_caching=prefix, enable_chunked_prefill=chunked))
        outs = eng.LLMEngine(sch, runner, greedy=True).generate(prompts, eng.SamplingParams(1.0, 24, True))
        runs.append([o.token_ids for o in outs])
        assert all(len(t) == 24 for t in runs[-1])
    assert runs[0] == runs[1]
    runner.close()


def test_other_widths_are_refused(ctx):
    with pytest.raises(Exception, match="kv_cache_bits"):
        _runner(ctx, 8)


def test_bytes_of_a_token(ctx):
    sizes = {}
    for bits in (16, 4):
        runner, _ = _runner(ctx, bits)
        sizes[bits] = runner.kv_bytes_per_token()
        runner.close()
    assert sizes[4] * 256 == sizes[16] * 72
