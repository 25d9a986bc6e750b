"""The reference's layer API (src/layers/*.rs) on the B200 kernels.  Same class names, constructor
arguments and method meaning; tensors are bf16 CUDA tensors used as device-memory handles, every
computation is a call through the C ABI (ops.Context).  No CPU path: a CPU tensor raises.

  RMSNorm            src/layers/layernorm.rs:3-61       forward(x, residual) -> (out, new_residual)
  RotaryEmbedding    src/layers/rotary_embedding.rs     apply(q, k) on [B, heads, T, hd], positions 0..T
  SiluAndMul         src/layers/activation.rs:4-18
  *ParallelLinear    src/layers/linear.rs:4-223         load_weights(weight, bias) / forward(x)
  Attention          src/layers/attention.rs:4-16       forward(q, k, v) + per-step Context

Beyond the reference: the linear layers run in 8 bits after to_fp8() (their loaded weights are converted) or load_fp8() (a checkpoint's own e4m3 weights with
a scale for each 128 x 128), and take rows that are in 8 bits already - (q, scale), as RMSNorm.forward_fp8 and SiluAndMul.forward_fp8 give them - in place of
a tensor.  Attention.fp4_cache keeps keys and values in 4 bits (ops.Fp4Cache), 72 bytes a row of 128 numbers in place of 256.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import List, Optional, Tuple

import torch

from . import ops
from .tp import TPConfig, get_tp

BF16 = torch.bfloat16


class RMSNorm:
    def __init__(self, ctx, hidden_size: int, eps: Optional[float] = None, device="cuda"):
        self.ctx = ctx
        self.weight = torch.ones(hidden_size, dtype=BF16, device=device)      # layernorm.rs:29 (ones)
        self.eps = 1e-6 if eps is None else eps

    @classmethod
    def from_weight(cls, ctx, weight: torch.Tensor, eps: float) -> "RMSNorm":
        self = cls.__new__(cls)
        self.ctx, self.weight, self.eps = ctx, weight.reshape(-1).to(BF16).contiguous(), eps
        return self

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None):
        """(x + residual) normalised; returns (out bf16, new_residual f32 or None) like
        layernorm.rs:44-60 (the sum is kept in f32)."""
        shape = x.shape
        x2 = x.reshape(-1, shape[-1]).contiguous()
        if residual is None:
            return self.ctx.fused_add_rmsnorm(x2, self.weight, self.eps).reshape(shape), None
        r2 = residual.reshape(-1, shape[-1]).to(torch.float32).contiguous()
        new_res = torch.empty_like(r2)
        out = self.ctx.fused_add_rmsnorm(x2, self.weight, self.eps, residual_in=r2, residual_out=new_res)
        return out.reshape(shape), new_res.reshape(shape)

    def forward_fp8(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None):
        """The same with the normed rows in 8 bits: ((q [rows, hidden], scale [rows, ceil(hidden / 128)]), new_residual f32 or None)."""
        shape = x.shape
        x2 = x.reshape(-1, shape[-1]).contiguous()
        if residual is None:
            q, scale, _ = ops.add_rmsnorm_fp8(self.ctx, x2, self.weight, self.eps)
            return (q, scale), None
        r2 = residual.reshape(-1, shape[-1]).to(torch.float32).contiguous()
        new_res = torch.empty_like(r2)
        q, scale, _ = ops.add_rmsnorm_fp8(self.ctx, x2, self.weight, self.eps, residual=r2, residual_out=new_res)
        return (q, scale), new_res.reshape(shape)


class RotaryEmbedding:
    def __init__(self, ctx, head_size: int, max_position: int, base: float):
        if head_size != 128:
            raise ValueError("the B200 kernels support head_size 128 (all Qwen3 dense models)")
        self.ctx, self.head_size, self.max_position, self.base = ctx, head_size, max_position, base
        self.table = ctx.rope_table(base, head_size, max_position)      # built once (reference: per call)

    def apply(self, q: torch.Tensor, k: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
        """q [B, nh, T, hd], k [B, kv, T, hd]; position of token t is t (rotary_embedding.rs:93-107)."""
        B, nh, T, hd = q.shape
        kv = k.shape[1]
        if T > self.max_position:
            raise ValueError("sequence longer than max_position")
        # plumbing only: token-major fused rows [q heads | k heads | (unused v heads)]
        rows = torch.cat([q.permute(0, 2, 1, 3).reshape(B * T, nh * hd), k.permute(0, 2, 1, 3).reshape(B * T, kv * hd),
                          torch.zeros(B * T, kv * hd, dtype=BF16, device=q.device)], dim=1).contiguous()
        pos = torch.arange(T, dtype=torch.int32, device=q.device).repeat(B)
        self.ctx.qk_norm_rope_store(rows, None, None, 0.0, self.table, pos, nh, kv, hd)
        qo = rows[:, :nh * hd].reshape(B, T, nh, hd).permute(0, 2, 1, 3)
        ko = rows[:, nh * hd:(nh + kv) * hd].reshape(B, T, kv, hd).permute(0, 2, 1, 3)
        return qo, ko


class SiluAndMul:
    def __init__(self, ctx):
        self.ctx = ctx

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        shape = x.shape
        out = self.ctx.silu_and_mul(x.reshape(-1, shape[-1]).contiguous())
        return out.reshape(*shape[:-1], shape[-1] // 2)

    def forward_fp8(self, x: torch.Tensor):
        """The same with rows in 8 bits: (q [rows, width / 2], scale)."""
        return ops.quant_fp8(self.ctx, x.reshape(-1, x.shape[-1]).contiguous(), act=ops.ACT_SILU_MUL)


# ----------------------------------------------------------------------------- linear family
class LinearBase:
    """weight [out, in] (the reference's layout, linear.rs:16)."""

    def __init__(self, ctx, tp_dim: int, input_size: int, output_size: int, tp: Optional[TPConfig] = None):
        self.ctx = ctx
        tp = tp or TPConfig(ctx.tp_size, ctx.tp_rank, tp_dim)
        self.tp_dim, self.tp_rank, self.tp_size = tp_dim, tp.rank, tp.size
        self.input_size, self.output_size = input_size, output_size
        self.weight: Optional[torch.Tensor] = None
        self.weight_fp8: Optional[Tuple[torch.Tensor, torch.Tensor]] = None       # (e4m3 [out, in], scale [ceil(out / 128), ceil(in / 128)])

    def to_fp8(self) -> "LinearBase":
        """Converts the loaded weight (this rank's share of it) to 8 bits, once; the bf16 weight is given up, and the shards it came from: to load one again takes all."""
        if self.weight is None:
            raise RuntimeError("load_weights has not been called")
        self._multiples_of_16("to_fp8", *self.weight.shape)
        self.weight_fp8, self.weight = ops.quant_fp8_weight(self.ctx, self.weight), None
        self._forget_shards()
        return self

    @staticmethod
    def _multiples_of_16(name: str, n: int, k: int) -> None:
        if n % 16 or k % 16:
            raise ValueError(f"{name}: products in 8 bits take multiples of 16, the weight is [{n}, {k}]")

    def _share(self) -> Tuple[int, int]:
        """(out, in) of the weight that this rank has."""
        return self.output_size, self.input_size

    def _forget_shards(self) -> None:
        """Layers that are loaded in shards hold them until all are there, and after: a shard may be loaded again."""

    def load_fp8(self, weight: torch.Tensor, scale: torch.Tensor) -> None:
        """This rank's share of the weight as e4m3 [out, in] with its scales [ceil(out / 128), ceil(in / 128)], on the context's device."""
        n, k = self._share()
        if weight.dtype != ops.FP8 or tuple(weight.shape) != (n, k) or not scale.is_floating_point() or tuple(scale.shape) != ((n + 127) // 128, (k + 127) // 128):
            raise ValueError(f"load_fp8: this rank has an e4m3 weight [{n}, {k}] and scales [{(n + 127) // 128}, {(k + 127) // 128}], "
                             f"got {weight.dtype} {list(weight.shape)} and {scale.dtype} {list(scale.shape)}")
        self._multiples_of_16("load_fp8", n, k)
        if weight.get_device() != self.ctx.device or scale.get_device() != self.ctx.device:
            raise ValueError(f"load_fp8: weight and scales must be on cuda:{self.ctx.device}")
        self.weight_fp8, self.weight = (weight.contiguous(), scale.to(torch.float32).contiguous()), None
        self._forget_shards()

    def _set(self, w: torch.Tensor, bias):
        if bias is not None:
            raise NotImplementedError("bias: the Qwen3 path has none (every call site passes None, qwen3.rs:121,123)")
        self.weight, self.weight_fp8 = w.to(BF16).contiguous(), None

    def forward(self, x) -> torch.Tensor:
        """x: [..., in], or rows in 8 bits (q, scale) for a layer whose weight is in 8 bits."""
        if self.weight_fp8 is not None:
            rows = x if isinstance(x, tuple) else ops.quant_fp8(self.ctx, x.reshape(-1, x.shape[-1]))
            y = ops.gemm_fp8(self.ctx, *rows, *self.weight_fp8)
            return y if isinstance(x, tuple) else y.reshape(*x.shape[:-1], y.shape[1])
        if self.weight is None:
            raise RuntimeError("load_weights has not been called")
        if isinstance(x, tuple):
            raise ValueError("rows in 8 bits need a weight in 8 bits: to_fp8() or load_fp8()")
        shape = x.shape
        y = self.ctx.gemm(x.reshape(-1, shape[-1]), self.weight)
        return y.reshape(*shape[:-1], self.weight.shape[0])


class ReplicatedLinear(LinearBase):
    def __init__(self, ctx, input_size, output_size):
        super().__init__(ctx, 0, input_size, output_size)

    def load_weights(self, weight, bias=None):
        self._set(weight, bias)


class ColumnParallelLinear(LinearBase):
    """Output features sharded: rank r keeps rows [r*out/tp, (r+1)*out/tp) of the FULL weight.
    (The reference computes shard_size from the already-full dim, linear.rs:81-84, which only
    works at tp_size 1.)"""

    def __init__(self, ctx, input_size, output_size, tp: Optional[TPConfig] = None):
        super().__init__(ctx, 0, input_size, output_size, tp)

    def load_weights(self, weight, bias=None):
        n = weight.shape[0] // self.tp_size
        self._set(weight[self.tp_rank * n:(self.tp_rank + 1) * n], bias)

    def _share(self):
        return self.output_size // self.tp_size, self.input_size


class MergedColumnParallelLinear(LinearBase):
    """Several column-parallel matrices fused along the output dim (gate_up): each is sharded
    separately, linear.rs:106-119."""

    def __init__(self, ctx, input_size, output_sizes: List[int], tp: Optional[TPConfig] = None):
        super().__init__(ctx, 0, input_size, sum(output_sizes), tp)
        self.output_sizes = output_sizes
        self._parts: List[Optional[torch.Tensor]] = [None] * len(output_sizes)

    def load_weights(self, weight, bias=None, loaded_shard_id: int = 0):
        n = self.output_sizes[loaded_shard_id] // self.tp_size
        self._parts[loaded_shard_id] = weight[self.tp_rank * n:(self.tp_rank + 1) * n]
        if all(p is not None for p in self._parts):
            self._set(torch.cat(self._parts, dim=0), bias)

    def _share(self):
        return sum(n // self.tp_size for n in self.output_sizes), self.input_size

    def _forget_shards(self):
        self._parts = [None] * len(self.output_sizes)


class QKVParallelLinear(LinearBase):
    """Fused q/k/v rows, sharded by head group (linear.rs:121-176)."""

    def __init__(self, ctx, hidden_size, head_size, num_heads, num_kv_heads, tp: Optional[TPConfig] = None):
        super().__init__(ctx, 0, hidden_size, (num_heads + 2 * num_kv_heads) * head_size, tp)
        self.head_size, self.num_heads, self.num_kv_heads = head_size, num_heads, num_kv_heads
        self._parts = {}

    def load_qkv_weight(self, w, shard_id: str):
        heads = self.num_heads if shard_id == "q" else self.num_kv_heads
        n = heads // self.tp_size * self.head_size
        self._parts[shard_id] = w[self.tp_rank * n:(self.tp_rank + 1) * n]
        if len(self._parts) == 3:
            self._set(torch.cat([self._parts["q"], self._parts["k"], self._parts["v"]], dim=0), None)

    def _share(self):
        return (self.num_heads // self.tp_size + 2 * (self.num_kv_heads // self.tp_size)) * self.head_size, self.input_size

    def _forget_shards(self):
        self._parts = {}

    def load_weights(self, weight, bias=None):
        """Full fused [q; k; v] weight (qwen3.rs:171-173)."""
        hs = self.head_size
        q, k, v = weight.split([self.num_heads * hs, self.num_kv_heads * hs, self.num_kv_heads * hs], dim=0)
        for name, w in (("q", q), ("k", k), ("v", v)):
            self.load_qkv_weight(w, name)


class RowParallelLinear(LinearBase):
    """Input features sharded (columns of the [out, in] weight); partial outputs are summed with
    an all-reduce - the reference stops before the reduce (linear.rs:184-198) and shards dim 0
    (:217), which is wrong for a row-parallel layer."""

    def __init__(self, ctx, input_size, output_size, tp: Optional[TPConfig] = None):
        super().__init__(ctx, 1, input_size, output_size, tp)

    def load_weights(self, weight, bias=None):
        n = weight.shape[1] // self.tp_size
        self._set(weight[:, self.tp_rank * n:(self.tp_rank + 1) * n], bias)

    def _share(self):
        return self.output_size, self.input_size // self.tp_size

    def forward(self, x):
        y = super().forward(x)
        if self.tp_size > 1:
            self.ctx.allreduce(y)
        return y


# ----------------------------------------------------------------------------- attention
@dataclass
class Context:
    """Per-step attention inputs (upstream nano-vllm's Context): the integer contract N1/N2."""
    is_prefill: bool = False
    cu_seqlens: Optional[torch.Tensor] = None      # i32 [B+1]
    max_seqlen: int = 0
    slot_mapping: Optional[torch.Tensor] = None    # i32 [N]
    context_lens: Optional[torch.Tensor] = None    # i32 [B]
    block_tables: Optional[torch.Tensor] = None    # i32 [B, max_blocks]


_CONTEXT = Context()


def set_context(**kw) -> None:
    global _CONTEXT
    _CONTEXT = Context(**kw)


def get_context() -> Context:
    return _CONTEXT


class Attention:
    """Attention{num_heads, head_dim, scale, softcapping} (attention.rs:4-9) + num_kv_heads and the
    paged KV cache.  forward(q, k, v): q [N, nh*hd], k / v [N, kv*hd] token-major (views into a
    fused qkv buffer are fine); writes k, v to the cache at slot_mapping, then varlen causal flash
    (prefill) or paged attention over block_tables (decode).
    fp4_cache (ops.Fp4Cache) in place of k_cache / v_cache keeps the rows in 4 bits; a prefill with block_tables then reads its
    whole context from there (portions behind a cached prefix), one without attends to its own k, v."""

    def __init__(self, ctx, num_heads: int, head_dim: int, scale: float, num_kv_heads: int, softcapping: float = 1.0,
                 block_size: int = 256):
        if softcapping != 1.0:
            raise NotImplementedError("softcapping is unused by Qwen3")
        self.ctx, self.num_heads, self.head_dim, self.scale = ctx, num_heads, head_dim, scale
        self.num_kv_heads, self.block_size = num_kv_heads, block_size
        self.k_cache: Optional[torch.Tensor] = None      # [num_blocks, block_size, kv, hd]
        self.v_cache: Optional[torch.Tensor] = None
        self.fp4_cache: Optional[ops.Fp4Cache] = None    # num_blocks pages of its own block_size

    def forward(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> torch.Tensor:
        c = get_context()
        nh, kv, hd = self.num_heads, self.num_kv_heads, self.head_dim
        if self.fp4_cache is not None:
            if self.k_cache is not None:
                raise RuntimeError("one cache: fp4_cache, or k_cache and v_cache")
            if c.slot_mapping is not None:
                ops.store_kvcache_fp4(self.ctx, k, v, self.fp4_cache, c.slot_mapping)
            if not c.is_prefill:
                return ops.paged_decode_attn_fp4(self.ctx, q, self.fp4_cache, c.block_tables, c.context_lens, nh, self.scale)
            if c.block_tables is not None:
                return ops.prefill_attn_paged_fp4(self.ctx, q, self.fp4_cache, c.block_tables, c.context_lens, c.cu_seqlens, c.max_seqlen, nh, self.scale)
        if self.k_cache is not None and c.slot_mapping is not None:
            self.ctx.store_kvcache(k, v, self.k_cache, self.v_cache, c.slot_mapping, kv, hd)
        if c.is_prefill:
            return self.ctx.prefill_attn(q, k, v, c.cu_seqlens, c.max_seqlen, nh, kv, hd, self.scale)
        if self.k_cache is None:
            raise RuntimeError("decode needs a KV cache")
        return self.ctx.paged_decode_attn(q, self.k_cache, self.v_cache, c.block_tables, c.context_lens, nh, kv, hd,
                                          self.block_size, self.scale)
