"""MI355X (gfx950) split-KV MLA decode behind the reference's Python entry points.

The hot path is hand-written HIP (``csrc/mla_decode.hip``) reached through the C ABI of
``include/mla_decode_amd.h``; this package is the torch-side host code around it.  Around the decode: the serving step
(``serving``), trees of drafted tokens (``drafts``), norm and projections by 4-bit weights (``layer``).
"""
from .api import (Fp4KVCache, Fp8KVCache, TreePlan, flash_mla_with_kvcache, fp4_kv_cache, fp8_kv_cache,
                  get_mla_metadata, get_mla_metadata_host, kv_append, merge_partials, mla_decode_absorbed,
                  mla_decode_with_kvcache, num_parts_for, prepare_w_uv, quantize_kv_cache)
from .drafts import Accepted, kv_keep_path, tree_accept, tree_plan
from .layer import Fp4Weight, Fp8Rows, linear_fp4, pack_w_fp4, quantize_w_fp4, rms_norm
from .legacy import MlaKernel
from .serving import (PagePool, Reservation, Rope, apply_rope, kv_append_slots, kv_gather, page_pool,
                      release_pages, reserve_pages, rope_plan)

__all__ = [
    "Fp4KVCache",
    "Fp8KVCache",
    "flash_mla_with_kvcache",
    "fp4_kv_cache",
    "fp8_kv_cache",
    "get_mla_metadata",
    "get_mla_metadata_host",
    "kv_append",
    "merge_partials",
    "mla_decode_absorbed",
    "mla_decode_with_kvcache",
    "num_parts_for",
    "prepare_w_uv",
    "quantize_kv_cache",
    "TreePlan",
    "Accepted",
    "kv_keep_path",
    "tree_accept",
    "tree_plan",
    "Fp4Weight",
    "Fp8Rows",
    "linear_fp4",
    "pack_w_fp4",
    "quantize_w_fp4",
    "rms_norm",
    "MlaKernel",
    "PagePool",
    "Reservation",
    "Rope",
    "apply_rope",
    "kv_append_slots",
    "kv_gather",
    "page_pool",
    "release_pages",
    "reserve_pages",
    "rope_plan",
]
