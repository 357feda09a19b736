"""B200 (sm_100a) fused multi-head attention forward: a drop-in for the operator of
kst179/fused-attention (``fused_attn.attention_forward``).

Public surface:
  attention_forward(head_dim, chunk_size, queries, keys, values, mask=None)   CUDA tensors
  attention_forward_host(...)                                                  host tensors
  bind_forward(...) -> (launch, out)                                           the same call, checked once, for loops
  shard_units / slice_tensor                                                   multi-GPU slicing
  KVCache / cache_create / cache_append / cache_select / cache_attention       a paged 8-bit key/value cache
  LatentCache / latent_cache_create / latent_append / latent_attention / latent_prompt   a paged cache of latent vectors
  PagePool / page_pool_create / pages_reserve / pages_fork / pages_compact / cache_copy   the pages of either
The compute path is the CUDA library ``lib/libfa_b200.so`` behind the C ABI of
``include/fa_b200.h``; there is no CPU path.
"""
from . import _lib
from .api import (attention_forward, attention_forward_host, bind_forward, cta_segments, describe_call, describe_schedule, plan_taken, query,
                  read_status, select_kernel, stream_has_scratch)
from .cache import KVCache, cache_append, cache_attention, cache_create, cache_select
from .latent import LatentCache, latent_append, latent_attention, latent_cache_create, latent_prompt, latent_status
from .pages import PagePool, cache_copy, page_pool_create, pages_compact, pages_fork, pages_reserve
from .sharding import (Shard, aggregate_throughput, attention_bytes, attention_flops, shard_units,
                       slice_tensor)

__all__ = [
    "attention_forward", "attention_forward_host", "bind_forward", "query", "read_status", "select_kernel",
    "describe_call", "describe_schedule", "cta_segments", "plan_taken", "stream_has_scratch",
    "KVCache", "cache_create", "cache_append", "cache_select", "cache_attention",
    "LatentCache", "latent_cache_create", "latent_append", "latent_attention", "latent_prompt", "latent_status",
    "PagePool", "page_pool_create", "pages_reserve", "pages_fork", "pages_compact", "cache_copy",
    "Shard", "shard_units", "slice_tensor", "attention_flops", "attention_bytes", "aggregate_throughput",
    "_lib",
]
