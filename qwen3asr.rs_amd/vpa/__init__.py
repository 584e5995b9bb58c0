"""vpa — MI355X-native paged-KV hot path of the Qwen3-ASR decoder.

Hand-written HIP kernels for gfx950 behind the C ABI of ``include/vpa.h``
(``libvpa.so``), with the Candle-op-shaped tensor API of
``mistralrs_paged_attn`` (as re-exported by ``vasr-paged-attn``) on top.
"""

from ._lib import VpaError  # noqa: F401
from .ops import (  # noqa: F401
    BlockBuffers,
    DecodeTokenState,
    DeviceBlockAllocator,
    argmax_token_ids_from_logits,
    cache_geometry,
    gather_kv_cache,
    paged_attention,
    paged_attention_plan,
    paged_cache_read,
    paged_attention_varlen_prefill,
    paged_attention_workspace,
    reshape_and_cache,
    reshape_and_cache_paged_attention,
)
from .block_scaled import (  # noqa: F401
    block_scales,
    paged_attention_block_scaled,
    paged_attention_block_scaled_workspace,
    reshape_and_cache_block_scaled,
)
from .eviction import (  # noqa: F401
    evict_kv_cache,
    evict_kv_cache_workspace,
    paged_attention_weights,
    paged_attention_weights_workspace,
)
from .graph import DecodeGraphCache  # noqa: F401
from .logits import adjust_logits  # noqa: F401
from .pages import copy_blocks  # noqa: F401
from .rotary import rotary_frequencies, rotary_qk, rotary_reshape_and_cache  # noqa: F401
from .step import DeviceDecodeStep  # noqa: F401
from .verify import verify_draft_tokens, verify_draft_tokens_workspace  # noqa: F401

__all__ = [
    "DecodeGraphCache",
    "BlockBuffers",
    "DecodeTokenState",
    "DeviceBlockAllocator",
    "DeviceDecodeStep",
    "VpaError",
    "adjust_logits",
    "argmax_token_ids_from_logits",
    "block_scales",
    "cache_geometry",
    "copy_blocks",
    "evict_kv_cache",
    "evict_kv_cache_workspace",
    "gather_kv_cache",
    "paged_attention",
    "paged_attention_block_scaled",
    "paged_attention_block_scaled_workspace",
    "paged_attention_plan",
    "paged_attention_weights",
    "paged_attention_weights_workspace",
    "paged_cache_read",
    "paged_attention_varlen_prefill",
    "paged_attention_workspace",
    "reshape_and_cache",
    "reshape_and_cache_block_scaled",
    "reshape_and_cache_paged_attention",
    "rotary_frequencies",
    "rotary_qk",
    "rotary_reshape_and_cache",
    "verify_draft_tokens",
    "verify_draft_tokens_workspace",
]
