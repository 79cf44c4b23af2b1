"""B200-native ring flash attention behind the reference's ``ring_flash_attn`` operator."""
from .api import balanced, check, deterministic, ring_flash_attn, ring_flash_attn_with_lse  # noqa: F401
from .compat import (  # noqa: F401
    ring_flash_attn_func,
    ring_flash_attn_kvpacked_func,
    ring_flash_attn_qkvpacked_func,
)
from .kv4 import KV4Cache, kv4_append, kv4_attn, kv4_attn_with_lse, kv4_gather  # noqa: F401
from .schedule import shutdown  # noqa: F401
from .scored import DocumentMask, document_mask, scored_flash_attn, scored_flash_attn_with_lse  # noqa: F401

__all__ = [
    "ring_flash_attn",
    "ring_flash_attn_with_lse",
    "ring_flash_attn_func",
    "ring_flash_attn_kvpacked_func",
    "ring_flash_attn_qkvpacked_func",
    "scored_flash_attn",
    "scored_flash_attn_with_lse",
    "document_mask",
    "DocumentMask",
    "KV4Cache",
    "kv4_append",
    "kv4_gather",
    "kv4_attn",
    "kv4_attn_with_lse",
    "deterministic",
    "balanced",
    "check",
    "shutdown",
]
