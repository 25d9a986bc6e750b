"""The Qwen3 runner over a 4-bit cache: its timing hook, and whole generations against the model in 64 bits."""
import importlib

import numpy as np
import pytest
import torch

import fp4_ref as ref
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
    with profile(activities=[ProfilerActivity.CUDA], acc_events=True) as p:
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


F64 = torch.float64
POOL, BS = 14, 16


class Paged:
    """Qwen3 in 64 bits over a pool of slots, with the cached rows as they are or as their 4-bit forms; a step is what the runner is told, and nothing else."""

    def __init__(self, w, fp4):
        self.w, self.fp4 = w, fp4
        self.nh, self.kv, self.hd = CFG.num_attention_heads, CFG.num_key_value_heads, CFG.head_dim
        self.pool = [[torch.full((POOL * BS, self.kv, self.hd), float("nan"), dtype=F64) for _ in range(2)] for _ in range(CFG.num_hidden_layers)]

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
        c, s = ref.to_fp4(x.to(torch.bfloat16))
        return (c.unflatten(-1, (8, 16)) * ref.SCALES[s][..., None]).flatten(-2)

    def step(self, ids, positions, cu, slots, tables, lens, paged):
        """Logits of each sequence's last row.  paged: rows attend to their context in the pool; else to the step's own rows."""
        w, pos, group = self.w, torch.from_numpy(positions).to(F64), self.nh // self.kv
        x = w["model.embed_tokens.weight"][torch.from_numpy(ids).long()]
        for i, pool in enumerate(self.pool):
            p = f"model.layers.{i}."
            h = self._norm(x, w[p + "input_layernorm.weight"])
            q, k, v = ((h @ w[p + f"self_attn.{c}_proj.weight"].T).unflatten(-1, (-1, self.hd)) for c in "qkv")
            q = self._turn(self._norm(q, w[p + "self_attn.q_norm.weight"]), pos)
            k = self._turn(self._norm(k, w[p + "self_attn.k_norm.weight"]), pos)
            for side, rows in zip(pool, (k, v)):
                side[torch.from_numpy(slots).long()] = self._kept(rows)
            out = []
            for b in range(len(cu) - 1):
                mine = slice(int(cu[b]), int(cu[b + 1]))
                n, m = int(cu[b + 1] - cu[b]), int(lens[b])
                if paged:
                    at = torch.tensor([int(tables[b, t // BS]) * BS + t % BS for t in range(m)])
                    ks, vs = pool[0][at], pool[1][at]
                else:
                    assert n == m
                    ks, vs = k[mine], v[mine]
                s = torch.einsum("qhd,khd->hqk", q[mine], ks.repeat_interleave(group, 1)) * self.hd ** -0.5
                s = s.masked_fill(torch.arange(m)[None] > torch.arange(m - n, m)[:, None], -float("inf"))
                out.append(torch.einsum("hqk,khd->qhd", torch.softmax(s, -1), vs.repeat_interleave(group, 1)).flatten(1))
            x = x + torch.cat(out) @ w[p + "self_attn.o_proj.weight"].T
            h = self._norm(x, w[p + "post_attention_layernorm.weight"])
            gate, up = h @ w[p + "mlp.gate_proj.weight"].T, h @ w[p + "mlp.up_proj.weight"].T
            x = x + (gate / (1 + torch.exp(-gate)) * up) @ w[p + "mlp.down_proj.weight"].T
        last = torch.from_numpy(cu[1:]).long() - 1
        return self._norm(x[last], w["model.norm.weight"]) @ w.get("lm_head.weight", w["model.embed_tokens.weight"]).T


def _config(prefix, chunked):
    return eng.SchedulerConfig(4, 64 if chunked else 512, CFG.eos_token_id, POOL, BS, enable_prefix_caching=prefix, enable_chunked_prefill=chunked)


def follow(runner, w, prompts, count, prefix, chunked):
    """Whole generations, a scheduled step at a time: the runner's logits against the two models', the tokens behind every slot that a step reads against the sequence's own.
    Gives the tokens, the worst error by its bound, and what happened on the way."""
    sch = eng.LLMEngine(eng.Scheduler(_config(prefix, chunked)), eng.DummyModelRunner())
    four, plain = Paged(w, True), Paged(w, False)
    said = {sch.add_request(p, eng.SamplingParams(1.0, count, True)): list(p) for p in prompts}
    written, seen, worst = np.full(POOL * BS, -1), dict(paged=0, plain=0, decode=0, mixed=0, again=0), 0.0
    while not sch.is_finished():
        si = sch.schedule()
        decode = si.num_decode_seqs == len(si.seq_ids) if chunked else not si.is_prefill
        cu = np.arange(len(si.seq_ids) + 1, dtype=np.int32) if decode else si.cu_seqlens
        paged = decode or chunked or bool((si.context_lens != np.diff(cu)).any())
        if decode:
            tokens = runner.decode(si.ids, si.positions, si.slot_mapping, si.block_tables, si.context_lens)
        elif paged:
            tokens = runner.step_mixed(si.ids, si.positions, cu, si.slot_mapping, si.block_tables, si.context_lens, si.num_decode_seqs)
        else:
            tokens = runner.prefill(si.ids, si.positions, cu, si.slot_mapping)
        seen["decode" if decode else "mixed" if si.num_decode_seqs else "paged" if paged else "plain"] += 1
        written[si.slot_mapping] = si.ids
        for b, sid in enumerate(si.seq_ids):
            m = int(si.context_lens[b])
            seen["again"] += not decode and b >= si.num_decode_seqs and len(said[sid]) > len(prompts[list(said).index(sid)])       # put back on the way
            assert [written[int(si.block_tables[b, t // BS]) * BS + t % BS] for t in range(m)] == said[sid][:m]
        step = (si.ids, si.positions, cu, si.slot_mapping, si.block_tables, si.context_lens, paged)
        got, a, c = torch.from_numpy(runner.last_logits(len(si.seq_ids))).to(F64), four.step(*step), plain.step(*step)
        bound = 2e-2 / 3 * CFG.vocab_size ** 0.5 + 0.6 * (a - c).norm(dim=-1)
        worst = max(worst, float(((got - a).norm(dim=-1) / bound).max()))
        for b, sid in enumerate(si.seq_ids):
            if si.emit is None or not chunked or si.emit[b]:
                said[sid].append(int(tokens[b]))
        sch.post_process(tokens)
    return [s[len(p):] for s, p in zip(said.values(), prompts)], worst, seen


def _prompts():
    prompts = [synth.make_prompts(1, n, CFG.vocab_size, 100 + n)[0] for n in (7, 33, 70, 50)]
    return prompts + [prompts[2][:64] + [5, 6, 7]]


@pytest.mark.parametrize("prefix,chunked", [(False, False), (True, False), (True, True)])
def test_generations_against_the_model(ctx, prefix, chunked):
    """Every step of generations over a pool that does not hold all sequences, with cached prefixes and chunked prompts, against the model in 64 bits with 4-bit rows; the engine's own run says
    the same tokens.

    Bound, of a sequence's logits as a vector: what the bf16 path is held to at every logit elsewhere (2e-2, three deviations of an error spread over 2 048 of them), and 0.6 of what the 4 bits
    themselves move.  Up to 1.8 % of a cached row's codes are others than the model's, as bf16 rows next to a border fall on its other side, each by a whole step, where the format's own roundings
    are off by a step / sqrt(12) at every place: sqrt(12 * 0.018) = 0.46, and three deviations of a tenth for the number of independent terms (a context of 7 tokens has 130 such codes)."""
    runner = _runner(ctx, 4, num_kvcache_blocks=POOL)
    w = {k: v.to(F64) for k, v in synth.make_weights(CFG, seed=0, norm_jitter=0.1).items()}
    prompts = _prompts()
    said, worst, seen = follow(runner, w, prompts, 24, prefix, chunked)
    assert worst <= 1, f"{worst} times the bound, {seen}"
    assert seen["decode"] and seen["again"] and (seen["mixed"] if chunked else seen["plain"]) and (not prefix or chunked or seen["paged"])
    outs = eng.LLMEngine(eng.Scheduler(_config(prefix, chunked)), runner, greedy=True).generate(prompts, eng.SamplingParams(1.0, 24, True))
    assert [o.token_ids for o in outs] == said
    runner.close()


def test_registry_runner(ctx, tmp_path):
    """ModelRunner over a Qwen3 directory with a 4-bit cache is Qwen3ModelRunner with one; an architecture with caches of its own refuses it."""
    import test_hf_loader as H
    import test_vizotar_model_gpu as V
    w = synth.make_weights(CFG, seed=4, norm_jitter=0.1)
    H._write_config(tmp_path, CFG, head_dim=CFG.head_dim, tie_word_embeddings=False)
    H.save_file({k: v.to(torch.bfloat16).contiguous() for k, v in w.items()}, str(tmp_path / "model.safetensors"))
    kw = dict(num_kvcache_blocks=16, kvcache_block_size=16, max_num_seqs=2, max_num_batched_tokens=256, max_model_len=256, kv_cache_bits=4)
    logits = []
    for kind in (lambda: eng.ModelRunner.from_dir(ctx, str(tmp_path), **kw), lambda: eng.Qwen3ModelRunner.from_hf_dir(ctx, str(tmp_path), **kw)):
        r = kind()
        assert r.kv_bytes_per_token() == CFG.num_hidden_layers * CFG.num_key_value_heads * 2 * 72
        r.prefill(range(10, 31), range(21), [0, 21], range(16, 37))
        r.decode([5], [21], [37], np.array([[1, 2]], dtype=np.int32), [22])
        logits.append(r.last_logits(1).copy())
        r.close()
    assert np.array_equal(*logits)
    cfg = V.Z.make_config(vocab=70, width=64, streams=2, layers=[V.Z.with_dense(V.Z.delta_cfg())])
    with pytest.raises(Exception, match="formats"):
        eng.ModelRunner.from_config(ctx, cfg, [], num_kvcache_blocks=2, kvcache_block_size=BS, max_num_seqs=1, max_num_batched_tokens=32, max_model_len=32, dtype="float32", kv_cache_bits=4)
