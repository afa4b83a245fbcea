"""B200-native attention forward behind the TinyFA API (C ABI in include/tinyfa_b200.h)."""
from .api import (device_status, flash_attn_forward, flash_attn_scored_forward, flash_attn_varlen_forward, is_head_dim_compiled,
                  set_option)

from .cache import flash_attn_cache_forward, kv_cache_plan, kv_cache_store
from .host import flash_attn_forward_host

__all__ = ["flash_attn_forward", "flash_attn_forward_host", "flash_attn_scored_forward", "flash_attn_varlen_forward",
           "flash_attn_cache_forward", "kv_cache_plan", "kv_cache_store", "is_head_dim_compiled", "device_status", "set_option"]
