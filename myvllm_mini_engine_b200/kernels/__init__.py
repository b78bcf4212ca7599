"""Operator API of the paged-KV hot path (mirrors ``mini_engine/kernels``)."""

from .data import copy_blocks, write_kv_cache, write_kv_cache_batch, write_kv_cache_slots
from .fp8 import (paged_attention_fp8, paged_attention_fp8_with_append, paged_prefill_attention_fp8,
                  write_kv_cache_slots_fp8)
from .int4 import (int4_page_bytes, paged_attention_int4, paged_prefill_attention_int4, read_kv_cache_slots_int4,
                   write_kv_cache_batch_int4, write_kv_cache_slots_int4)
from .paged import paged_attention, paged_attention_with_append
from .prefill import paged_prefill_attention
from .sparse import (block_bounds_bytes, paged_attention_selected, read_block_bounds, select_blocks,
                     update_block_bounds)

__all__ = ["block_bounds_bytes", "copy_blocks", "int4_page_bytes", "paged_attention", "paged_attention_with_append", "paged_attention_fp8", "paged_attention_fp8_with_append", "paged_attention_int4", "paged_attention_selected", "paged_prefill_attention", "paged_prefill_attention_fp8", "paged_prefill_attention_int4", "read_block_bounds", "read_kv_cache_slots_int4", "select_blocks", "update_block_bounds", "write_kv_cache",
           "write_kv_cache_batch", "write_kv_cache_batch_int4", "write_kv_cache_slots", "write_kv_cache_slots_fp8", "write_kv_cache_slots_int4"]
