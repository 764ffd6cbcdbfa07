"""PyTorch frontend: the reference's ``stackkernels.torch`` attention API."""

from stackkernels_amd.torch.attention import (
    FlashAttention,
    FlashAttentionFunction,
    flash_attention,
    flash_attention_q8,
    flash_decode,
    flash_decode_q8,
)

from stackkernels_amd.torch.cache import kv_cache_update, kv_cache_update_q8, kv_page_plan

__all__ = ["flash_attention", "flash_decode", "FlashAttention", "FlashAttentionFunction",
           "flash_attention_q8", "flash_decode_q8", "kv_cache_update", "kv_cache_update_q8",
           "kv_page_plan"]
