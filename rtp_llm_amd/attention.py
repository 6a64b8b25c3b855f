"""Decode attention strategy — the reference's FMHA plug-in surface
(rtp_llm/models_py/modules/factory/attention/{fmha_impl_base.py:99-178, attn_factory.py:100-254}):

    DECODE_MHA_IMPS.append(cls); cls.support(attn_configs, attn_inputs);
    impl = cls(attn_configs, attn_inputs, parallelism_config); impl.forward(qkv, LayerKVCache, layer_idx)

Data-contract mirrors (bindings/OpDefs.h:29-51,281-327; cpp/model_utils/AttentionConfig.h:24-85):
LayerKVCache, PyAttentionInputs, AttentionConfigs — same field names, decode fields only.
"""
import math
from dataclasses import dataclass, field
from typing import List, Optional

import torch

from . import ops


@dataclass
class AttentionConfigs:       # cpp/model_utils/AttentionConfig.h:24-85 (per-rank values)
    head_num: int
    kv_head_num: int
    size_per_head: int
    rope_dim: int = 0
    rope_theta: float = 1e6
    max_seq_len: int = 4096
    softmax_extra_scale: float = 1.0
    kernel_tokens_per_block: int = 16
    softcap: float = 0.0                           # > 0: scores become softcap * tanh(score / softcap)
    slopes: Optional[torch.Tensor] = None          # fp32 [head_num]: distance biases in place of the rotation
    kv_budget: int = 0                             # > 0: tokens that a sequence keeps per kv head; the least attended go first
    kv_sinks: int = 4                              # ... of which the first and the newest tokens always stay
    kv_recent: int = 32
    kv_decay: float = 1.0                          # what earlier attention weights count at every step

    @property
    def scored(self) -> bool:
        return self.softcap != 0 or self.slopes is not None or self.kv_budget != 0


@dataclass
class LayerKVCache:           # bindings/OpDefs.h:29-51
    kv_cache_base: torch.Tensor                    # [blocks, 2, nkv, page, hd]
    kv_scale_base: Optional[torch.Tensor] = None   # [blocks, 2*nkv*page] fp32 (8-bit caches)
    seq_size_per_block: int = 0
    layer_id: int = -1
    weights: Optional[torch.Tensor] = None         # planes of a cache that evicts (kvcache.alloc_planes): attention weights,
    key_pos: Optional[torch.Tensor] = None         # and the positions of the tokens in its slots


@dataclass
class PyAttentionInputs:      # bindings/OpDefs.h:281-327, decode fields
    is_prefill: bool = False
    sequence_lengths: torch.Tensor = None              # int32 [B]: tokens already in the cache
    input_lengths: torch.Tensor = None
    kv_cache_kernel_block_id_device: torch.Tensor = None   # int32 [B, M]
    is_cuda_graph: bool = False
    sequence_lengths_plus_1_device: torch.Tensor = None    # filled by prepare()
    token_positions: Optional[torch.Tensor] = None         # int32 [B]: the new tokens' positions where they are not sequence_lengths (after evictions)


class FMHAImplBase:
    def forward(self, qkv, kv_cache, layer_idx: int = 0):
        raise NotImplementedError

    @staticmethod
    def support(attn_configs, attn_inputs) -> bool:
        return False

    def support_cuda_graph(self) -> bool:       # fmha_impl_base.py:165-172
        return callable(getattr(self, "prepare_cuda_graph", None))


class Mi355PagedDecodeImpl(FMHAImplBase):
    """RoPE+KV-write op followed by the paged flash-decoding op (the pairing of
    AiterDecodeImpl*, rocm_impl/aiter.py:1960-2031)."""

    def __init__(self, attn_configs: AttentionConfigs, attn_inputs: PyAttentionInputs, parallelism_config=None,
                 cos_sin: Optional[torch.Tensor] = None, qkv_bias: Optional[torch.Tensor] = None):
        self.cfg = attn_configs
        self.cos_sin = cos_sin
        self.prepare(attn_inputs)

    @staticmethod
    def support(attn_configs: AttentionConfigs, attn_inputs: PyAttentionInputs) -> bool:
        g = attn_configs.head_num // max(1, attn_configs.kv_head_num)
        return (not attn_inputs.is_prefill and not attn_configs.scored and attn_configs.size_per_head in (64, 128) and g <= 16
                and attn_configs.head_num % attn_configs.kv_head_num == 0
                and attn_configs.rope_dim in (0, attn_configs.size_per_head))

    def prepare(self, attn_inputs: PyAttentionInputs):
        """Host-side prep (FMHAParams, aiter.py:205-209: seq_lens = sequence_lengths + 1 on device)."""
        self.inputs = attn_inputs
        dev = attn_inputs.kv_cache_kernel_block_id_device.device
        self.positions = attn_inputs.sequence_lengths.to(device=dev, dtype=torch.int32).contiguous()
        self.seq_lens = (self.positions + 1).contiguous()
        attn_inputs.sequence_lengths_plus_1_device = self.seq_lens
        self.block_table = attn_inputs.kv_cache_kernel_block_id_device.to(torch.int32).contiguous()

    def prepare_cuda_graph(self, attn_inputs: PyAttentionInputs):
        """In-place refresh of the address-stable device buffers for graph replay (aiter.py:1964-1981)."""
        self.positions.copy_(attn_inputs.sequence_lengths.to(self.positions.device, torch.int32))
        torch.add(self.positions, 1, out=self.seq_lens)
        self.block_table.copy_(attn_inputs.kv_cache_kernel_block_id_device)

    def forward(self, qkv: torch.Tensor, kv_cache: LayerKVCache, layer_idx: int = 0) -> torch.Tensor:
        c = self.cfg
        page = kv_cache.seq_size_per_block or kv_cache.kv_cache_base.shape[3]
        q = ops.rope_kv_write(qkv.contiguous(), None, self.cos_sin, self.positions, self.block_table, kv_cache.kv_cache_base,
                              kv_cache.kv_scale_base, c.head_num, c.kv_head_num, c.size_per_head, page)
        return ops.paged_decode_attention(q, kv_cache.kv_cache_base, kv_cache.kv_scale_base, self.block_table, self.seq_lens,
                                          c.kv_head_num, page, c.max_seq_len,
                                          c.softmax_extra_scale / math.sqrt(c.size_per_head))


class Mi355ScoredDecodeImpl(Mi355PagedDecodeImpl):
    """The same pairing for capped or biased scores and for a cache with a budget: the writer puts a token at the next slot, whatever its position, the attention adds up what every cached token
    draws, and evict() brings the cache back to the budget."""

    def __init__(self, attn_configs: AttentionConfigs, attn_inputs: PyAttentionInputs, parallelism_config=None, cos_sin: Optional[torch.Tensor] = None, qkv_bias: Optional[torch.Tensor] = None):
        if not attn_configs.softcap >= 0:
            raise ValueError(f"softcap={attn_configs.softcap} (0: none, or above)")
        if attn_configs.kv_budget < 0:
            raise ValueError(f"kv_budget={attn_configs.kv_budget} (0: none, or above)")
        # no table means no rotation to the writer: that has to be the model's choice (slopes, or no rotated channels)
        if attn_configs.slopes is None and attn_configs.rope_dim != 0 and cos_sin is None:
            raise ValueError(f"rope_dim={attn_configs.rope_dim} needs cos_sin (models with slopes do not rotate)")
        super().__init__(attn_configs, attn_inputs, parallelism_config, cos_sin, qkv_bias)

    @staticmethod
    def support(attn_configs: AttentionConfigs, attn_inputs: PyAttentionInputs) -> bool:
        return (not attn_inputs.is_prefill and attn_configs.scored and attn_configs.size_per_head in (64, 128) and attn_configs.head_num % max(1, attn_configs.kv_head_num) == 0
                and attn_configs.rope_dim in (0, attn_configs.size_per_head))

    def prepare(self, attn_inputs: PyAttentionInputs):
        super().prepare(attn_inputs)
        # prepare_cuda_graph writes into these: not into the caller's
        own = lambda t, given: t.clone() if attn_inputs.is_cuda_graph and t.data_ptr() == given.data_ptr() else t
        self.slots, self.block_table, given = own(self.positions, attn_inputs.sequence_lengths), own(self.block_table, attn_inputs.kv_cache_kernel_block_id_device), attn_inputs.token_positions
        self.positions = (self.slots if given is None else given.to(device=self.slots.device, dtype=torch.int32)).clone()

    def prepare_cuda_graph(self, attn_inputs: PyAttentionInputs):
        given = attn_inputs.token_positions
        self.slots.copy_(attn_inputs.sequence_lengths.to(self.slots.device, torch.int32))
        self.positions.copy_(self.slots if given is None else given.to(self.slots.device, torch.int32))
        torch.add(self.slots, 1, out=self.seq_lens)
        self.block_table.copy_(attn_inputs.kv_cache_kernel_block_id_device)

    def forward(self, qkv: torch.Tensor, kv_cache: LayerKVCache, layer_idx: int = 0) -> torch.Tensor:
        c = self.cfg
        page = kv_cache.seq_size_per_block or kv_cache.kv_cache_base.shape[3]
        if c.kv_budget > 0 and (kv_cache.weights is None or kv_cache.key_pos is None):
            raise ValueError("a cache with a budget needs its planes (kvcache.alloc_planes)")
        q = ops.rope_kv_write_slots(qkv.contiguous(), None, None if c.slopes is not None else self.cos_sin, self.positions, self.slots, self.block_table, kv_cache.kv_cache_base,
                                    kv_cache.kv_scale_base, c.head_num, c.kv_head_num, c.size_per_head, page, key_pos=kv_cache.key_pos, weights=kv_cache.weights)
        # slots are bounded by the block table, as evict() has them, not by max_seq_len: that is of positions, and a budget's table may be shorter
        return ops.paged_attention_scored(q, kv_cache.kv_cache_base, kv_cache.kv_scale_base, self.block_table, self.seq_lens, c.kv_head_num, page, self.block_table.shape[1] * page,
                                          scale=c.softmax_extra_scale / math.sqrt(c.size_per_head), softcap=c.softcap, slopes=c.slopes,
                                          positions=self.positions if c.slopes is not None else None, key_pos=kv_cache.key_pos if c.slopes is not None else None,
                                          weights=kv_cache.weights if c.kv_budget > 0 else None, decay=c.kv_decay)

    def evict(self, kv_cache: LayerKVCache) -> torch.Tensor:
        """Behind forward() of a step: sequences over the budget go back to it, in this layer.  -> the lengths (int32 [B], the same for every layer); the next step's sequence_lengths, with
        token_positions one above this step's."""
        c = self.cfg
        if c.kv_budget <= 0:
            raise ValueError("evict() is for a cache with a budget (kv_budget)")
        if kv_cache.weights is None or kv_cache.key_pos is None:
            raise ValueError("a cache with a budget needs its planes (kvcache.alloc_planes)")
        kv = kv_cache.kv_cache_base
        page = kv_cache.seq_size_per_block or kv.shape[3]
        return ops.kv_evict(kv_cache.weights, kv_cache.key_pos, self.block_table, self.seq_lens, self.positions + 1, kv.view(-1, 2, c.kv_head_num, page, c.size_per_head),
                            kv_cache.kv_scale_base, c.kv_budget, sinks=c.kv_sinks, recent=c.kv_recent)


DECODE_MHA_IMPS: List[type] = [Mi355PagedDecodeImpl, Mi355ScoredDecodeImpl]   # attention/__init__.py:47-49 registration list


class AttnImplFactory:
    """attn_factory.py:226-254: first registered impl whose support() accepts the inputs."""

    @staticmethod
    def get_fmha_impl(attn_configs, attn_inputs, parallelism_config=None, **kw) -> FMHAImplBase:
        for impl in DECODE_MHA_IMPS:
            if impl.support(attn_configs, attn_inputs):
                inst = impl(attn_configs, attn_inputs, parallelism_config, **kw)
                if attn_inputs.is_cuda_graph and not inst.support_cuda_graph():
                    continue
                return inst
        raise RuntimeError("no decode FMHA implementation supports these inputs")
