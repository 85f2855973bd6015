"""Deterministic attention backend bound to vLLM's CUSTOM slot
(reference: fxpr_vllm/vllm_modules/attention_backend.py:42-228).

Metadata and its builder are vLLM's Triton-attention ones (query_start_loc,
seq_lens, block_table, max_query_len, max_seq_len); the paged KV cache layout
``[num_blocks, 2, block_size, num_kv_heads, head_size]`` and the cache update
(``reshape_and_cache_flash``) are vLLM's. The attention itself is
``unified_attention_fxp`` on the B200 kernel, split over
``VLLM_FXP_NUM_KV_SPLITS`` KV splits (results do not depend on the count).

An addition to the reference's backend: when the engine's cascade attention is
on (``disable_cascade_attn=False``) and all requests of a step share a prefix,
``shared_prefix_attention_fxp`` runs instead, with the same bits.

The rotary position stays vLLM's in the engine. vLLM 0.22 fuses rotary and cache
update on ROCm only, and there only for steps of up to 256 tokens, so offering
it would give a token another rotation in a larger step. The method that it
would call, ``do_rope_and_kv_cache_update``, is for callers of the layer itself.
"""

from __future__ import annotations

import logging

import torch
from vllm.v1.attention.backend import AttentionImpl, AttentionLayer, AttentionType
from vllm.v1.attention.backends.triton_attn import TritonAttentionBackend, TritonAttentionMetadataBuilder

from ..fixed_point_kernels.attention import (shared_prefix_attention_fxp, shared_prefix_takes_prefix_kernels,
                                              unified_attention_fxp)
from ..fixed_point_kernels.fixed_point import RCP_LN2
from ..fixed_point_kernels.rope import rope_append_kv_fxp
from .config import get_runtime_config

logger = logging.getLogger("fxpr_vllm")


class DeterministicAttentionMetadataBuilder(TritonAttentionMetadataBuilder):
    """The Triton backend's metadata, with cascade attention for the steps in
    which the shared-prefix operator runs its prefix kernels, by the operator's
    own rule. In the others it would run the unified kernels, and the engine
    only lose its full CUDA graph. The engine does not say how many keys the
    requests have behind the prefix: the rule is asked for the fewest possible
    (their queries), and with many the operator runs the unified kernels after
    all."""

    # of an instance: what its layers have
    headdim = 128
    block_size = 16
    q_dtype = kv_dtype = torch.bfloat16
    logits_soft_cap = 0.0

    def __init__(self, kv_cache_spec, layer_names, vllm_config, device):
        super().__init__(kv_cache_spec, layer_names, vllm_config, device)
        self.headdim, self.kv_dtype = kv_cache_spec.head_size, kv_cache_spec.dtype
        self.q_dtype = vllm_config.model_config.dtype
        layers = vllm_config.compilation_config.static_forward_context
        caps = [getattr(layers[n].impl, "logits_soft_cap", 0.0) for n in layer_names if n in layers]
        self.logits_soft_cap = max(caps, default=0.0)

    def use_cascade_attention(self, common_prefix_len: int, query_lens, num_query_heads: int,
                              num_kv_heads: int, use_alibi: bool, use_sliding_window: bool,
                              use_local_attention: bool, num_sms: int, dcp_world_size: int) -> bool:
        if len(query_lens) < 2 or use_local_attention or dcp_world_size > 1:
            return False
        cfg = get_runtime_config()
        prefix, longest = int(common_prefix_len), int(max(query_lens))
        return shared_prefix_takes_prefix_kernels(
            prefix, len(query_lens), int(sum(query_lens)), longest, prefix + longest, num_query_heads,
            num_kv_heads, self.headdim, self.block_size, dtype=self.q_dtype, kv_dtype=self.kv_dtype,
            fxp_dtype=cfg.fxp_int_bits, frac_bits=cfg.frac_bits, logits_soft_cap=self.logits_soft_cap,
            window_size=int(use_sliding_window), alibi=bool(use_alibi))

    def build(self, common_prefix_len: int, common_attn_metadata, fast_build: bool = False):
        # the Triton builder's own cascade fields are not used (it leaves some
        # of them unset): built without a prefix, which is then noted
        metadata = super().build(0, common_attn_metadata, fast_build)
        if common_prefix_len > 0:
            metadata.use_cascade, metadata.common_prefix_len = True, common_prefix_len
        return metadata


class DeterministicAttentionBackend(TritonAttentionBackend):
    """Fixed-point deterministic attention backend."""

    accept_output_buffer: bool = True
    forward_includes_kv_cache_update: bool = False

    @staticmethod
    def get_name() -> str:
        return "CUSTOM"

    @staticmethod
    def get_impl_cls() -> type["DeterministicAttentionImpl"]:
        return DeterministicAttentionImpl

    @staticmethod
    def get_builder_cls() -> type["DeterministicAttentionMetadataBuilder"]:
        return DeterministicAttentionMetadataBuilder

    @classmethod
    def supports_head_size(cls, head_size: int) -> bool:
        return head_size in (32, 64, 128, 256)

    @classmethod
    def supports_sink(cls) -> bool:
        return False


class DeterministicAttentionImpl(AttentionImpl):
    def __init__(self, num_heads: int, head_size: int, scale: float, num_kv_heads: int,
                 alibi_slopes: list[float] | None, sliding_window: int | None,
                 kv_cache_dtype: str = "auto", logits_soft_cap: float | None = None,
                 attn_type: AttentionType | None = AttentionType.DECODER,
                 *_extra_positional, **kwargs) -> None:
        if attn_type is not None and attn_type != AttentionType.DECODER:
            raise NotImplementedError(
                f"DeterministicAttention only supports decoder attention; got attn_type={attn_type!r}.")
        if kv_cache_dtype not in ("auto", "fp16", "bf16", "float16", "bfloat16"):
            raise NotImplementedError(
                f"DeterministicAttention does not support kv_cache_dtype={kv_cache_dtype!r}; "
                "supported: auto, fp16, bf16.")
        cfg = get_runtime_config()
        self.num_heads = num_heads
        self.head_size = head_size
        self.scale = scale
        self.num_kv_heads = num_kv_heads
        self.num_kv_groups = num_heads // num_kv_heads
        self.kv_cache_dtype = kv_cache_dtype
        self.logits_soft_cap = float(logits_soft_cap) if logits_soft_cap else 0.0
        self.window_size = int(sliding_window) if sliding_window else 0
        self.attn_type = attn_type or AttentionType.DECODER
        self.frac_bits = cfg.frac_bits
        self.fxp_int_bits = cfg.fxp_int_bits
        self.num_kv_splits = cfg.num_kv_splits
        if alibi_slopes is not None:
            slopes = torch.tensor(alibi_slopes, dtype=torch.float32) * RCP_LN2
            assert slopes.shape == (num_heads,), \
                f"alibi_slopes shape {tuple(slopes.shape)} != (num_heads={num_heads},)"
            self.alibi_slopes: torch.Tensor | None = slopes
        else:
            self.alibi_slopes = None

    def forward(self, layer: AttentionLayer, query: torch.Tensor, key: torch.Tensor,
                value: torch.Tensor, kv_cache: torch.Tensor, attn_metadata,
                output: torch.Tensor | None = None, output_scale: torch.Tensor | None = None,
                output_block_scale: torch.Tensor | None = None, **kwargs) -> torch.Tensor:
        if output_scale is not None or output_block_scale is not None:
            raise NotImplementedError("DeterministicAttention does not support fp8/quantized output scales.")
        num_tokens = query.shape[0]
        query = query.view(num_tokens, self.num_heads, self.head_size)
        if output is None:
            output = torch.empty(num_tokens, self.num_heads, self.head_size, dtype=query.dtype,
                                 device=query.device)
        else:
            output = output.view(num_tokens, self.num_heads, self.head_size)
        if attn_metadata is None:
            output.zero_()  # profiling run before metadata exists
            return output.view(num_tokens, self.num_heads * self.head_size)
        if self.alibi_slopes is not None and self.alibi_slopes.device != query.device:
            self.alibi_slopes = self.alibi_slopes.to(query.device)
        n = attn_metadata.num_actual_tokens
        args = dict(
            q=query[:n], kv_cache=kv_cache, o=output[:n],
            query_start_loc=attn_metadata.query_start_loc, seq_lens=attn_metadata.seq_lens,
            block_table=attn_metadata.block_table, max_query_len=int(attn_metadata.max_query_len),
            alibi_slopes=self.alibi_slopes, fxp_dtype=self.fxp_int_bits, is_causal=True,
            softmax_scale=self.scale, frac_bits=self.frac_bits,
            logits_soft_cap=self.logits_soft_cap, window_size=self.window_size,
            max_seq_len=int(attn_metadata.max_seq_len),
        )
        if getattr(attn_metadata, "use_cascade", False):
            shared_prefix_attention_fxp(common_prefix_len=int(attn_metadata.common_prefix_len), **args)
        else:
            unified_attention_fxp(num_kv_splits=self.num_kv_splits, **args)
        return output.view(num_tokens, self.num_heads * self.head_size)

    def do_kv_cache_update(self, layer: AttentionLayer, key: torch.Tensor, value: torch.Tensor,
                           kv_cache: torch.Tensor, slot_mapping: torch.Tensor) -> None:
        if self.attn_type in (AttentionType.ENCODER_ONLY, AttentionType.ENCODER):
            return
        from vllm._custom_ops import reshape_and_cache_flash

        key_cache, value_cache = kv_cache.unbind(1)
        reshape_and_cache_flash(key, value, key_cache, value_cache, slot_mapping,
                                self.kv_cache_dtype, layer._k_scale, layer._v_scale)

    def do_rope_and_kv_cache_update(self, layer: AttentionLayer, query: torch.Tensor, key: torch.Tensor,
                                    value: torch.Tensor, positions: torch.Tensor,
                                    cos_sin_cache: torch.Tensor, is_neox: bool, kv_cache: torch.Tensor,
                                    layer_slot_mapping: torch.Tensor) -> None:
        """Rotary position of query and key in place, key and value into the
        cache, for a caller that runs the layer itself: the engine does not
        call it (``fused_rope_kvcache_supported`` stays false)."""
        n = query.shape[0]
        q = query.view(n, self.num_heads, self.head_size)
        k, v = (x.view(n, self.num_kv_heads, self.head_size) for x in (key, value))
        rope_append_kv_fxp(q, k, v, kv_cache, layer_slot_mapping[:n], positions[:n], cos_sin_cache,
                           is_neox, q_out=q, k_out=k)
