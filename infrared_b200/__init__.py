"""infrared_b200 — B200-native paged-decode attention for the infrared engine.

Three hand-written sm_100a CUDA paths behind a C ABI
(``include/infrared_b200.h``, ``libinfrared_b200.so``):

* ``cache_write`` — scatter of a step's K/V into the paged pool;
* ``paged_decode`` / ``paged_decode_write`` / ``paged_decode_rope_write`` —
  GQA decode attention over block tables (optionally fused with the cache
  write, and with the rotary embedding of q and the new K), split across all
  SMs in equal token shares with a log-sum-exp merge;
* ``kv_proj_rope_write`` — the K/V projections of a step's new tokens with
  bias, RoPE and the pool write in the epilogue (tcgen05 tensor cores), and
  ``paged_decode_rope`` — decode with RoPE on q, for such a step;
* ``paged_decode_lse`` + ``lse_merge`` — partials of a KV range and their
  combination, used to spread one long context over several GPUs;
* ``paged_prefill`` — causal attention of packed query rows (prefill with a
  cached prefix, mixed prefill + decode frames) on the tcgen05 tensor cores;
* ``cache_write_q8`` / ``cache_gather_q8`` / ``paged_decode_q8`` /
  ``paged_prefill_q8`` — the same over a cache of 8-bit codes (e4m3 or int8)
  with one scale per block and kv head, quantised as it is written;
* ``qk_norm_rope`` — RMS norm of every query and key head with the rotary
  embedding in the same pass.

``PagedKVPool``, ``PagedContext`` and ``paged_attention`` keep the
reference engine's interface (``PagedKVPoolQ8`` is the pool in 8 bits);
``shim.install()`` routes infrared's own decode calls here; ``dist`` shards
the work over the GPUs of one node.
"""

from ._lib import InfraredB200Error, UnsupportedShape
from .attention import paged_attention
from .ops import (DeviceError, cache_gather, cache_gather_q8, cache_write, cache_write_q8,
                  check_device_errors, derive_block_metadata, kv_proj_rope_write, lse_merge,
                  paged_decode, paged_decode_lse, paged_decode_q8, paged_decode_rope,
                  paged_decode_rope_write, paged_decode_write, paged_prefill, paged_prefill_q8,
                  qk_norm_rope)
from .paged_kv_cache import PagedContext, PagedKVPool, PagedKVPoolQ8

__all__ = [
    "DeviceError", "InfraredB200Error", "PagedContext", "PagedKVPool",
    "PagedKVPoolQ8", "UnsupportedShape",
    "cache_gather", "cache_gather_q8", "cache_write", "cache_write_q8", "check_device_errors",
    "derive_block_metadata", "kv_proj_rope_write", "lse_merge", "paged_attention",
    "paged_decode", "paged_decode_lse", "paged_decode_q8", "paged_decode_rope",
    "paged_decode_rope_write", "paged_decode_write", "paged_prefill", "paged_prefill_q8",
    "qk_norm_rope",
]
