"""Autograd layer and standalone functions (reference: ops/__init__.py,
ops/attention.py).  The reference's memory pool (ops/memory.py) is not part of
this build: torch's caching allocator owns all memory."""
from .attention import (  # noqa: F401
    EnhancedFlashAttentionV100Function,
    FlashAttentionV100Function,
    SUPPORTED_DTYPES,
    compare_with_pytorch_attention,
    compare_with_pytorch_attention_enhanced,
    flash_attention_backward,
    flash_attention_backward_enhanced,
    flash_attention_forward,
    flash_attention_forward_enhanced,
    gradient_checkpointing_mode,
    mixed_precision_mode,
)
from .paged import flash_attention_v100_paged  # noqa: F401
from .paged_cache import (  # noqa: F401
    paged_cache_accept_v100,
    paged_cache_compact_v100,
    paged_cache_fork_v100,
    paged_cache_write_v100,
)
from .rotary import rotary_embedding_v100, rotary_table_v100  # noqa: F401
from .scored import flash_attention_v100_scored  # noqa: F401
from .shared_prefix import flash_attention_v100_shared_prefix  # noqa: F401

__all__ = [
    "flash_attention_v100_scored",
    "flash_attention_v100_shared_prefix",
    "flash_attention_v100_paged",
    "paged_cache_write_v100",
    "paged_cache_accept_v100",
    "paged_cache_fork_v100",
    "paged_cache_compact_v100",
    "rotary_table_v100",
    "rotary_embedding_v100",
    "FlashAttentionV100Function",
    "EnhancedFlashAttentionV100Function",
    "flash_attention_forward",
    "flash_attention_backward",
    "compare_with_pytorch_attention",
    "flash_attention_forward_enhanced",
    "flash_attention_backward_enhanced",
    "compare_with_pytorch_attention_enhanced",
    "gradient_checkpointing_mode",
    "mixed_precision_mode",
]
