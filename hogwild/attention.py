"""`hogwild.attention` as the reference ships it (python/hogwild/attention.py), served by the MI355X implementation.

The operator wrappers (`hogwild_fused` :19-23, `hogwild_sdpa` :26-35, `hogwild_rope` :70-74) keep their names, argument
order and defaults; loading this module loads `hogatt.abi3.so`, so `torch.ops.libhogatt.*` call sites work as well
(:12-16).  `CacheStructure`, `HogwildCache`, `merge_caches`, `AttentionModule` and `model_surgery` (:105-257, :263-354)
are the re-designed host-side objects of `inference_lib_amd.cache` / `.model`.  Not provided on purpose: the pure-torch
`hogwild_sdpa_pt` (:38-67) and a fallback to it when the library is missing -- without the built library this import
fails instead of degrading to an eager path.  Added: paged caches in 4 bits (`*_q4`, `q4_cache`), the pages of paged caches
(`fork_blocks`, `free_blocks`, `reserve_blocks`, `compact_blocks`, `copy_blocks`, `trim_blocks`, `PagedCache`), paged attention with a sliding
window (`*_window`), packed batches (`packed_slots`, `copy_to_slots`) and drafted tokens (`verify_drafts`).
"""
from inference_lib_amd.attention import (HAVE_TORCH_OPS, compact_blocks, copy_blocks, copy_to_blocks, copy_to_blocks_q4, copy_to_slots, fork_blocks,
                                         free_blocks, hogwild_fused, hogwild_paged_sdpa, hogwild_paged_sdpa_q4, hogwild_paged_sdpa_window,
                                         hogwild_rope, hogwild_sdpa, hogwild_varlen_paged_sdpa, hogwild_varlen_paged_sdpa_q4,
                                         hogwild_varlen_paged_sdpa_window, packed_slots, q4_cache, read_blocks_q4, reserve_blocks, trim_blocks,
                                         verify_drafts)
from inference_lib_amd.cache import CacheStructure, HogwildCache, PagedCache, SegmentCache, merge_caches
from inference_lib_amd.model import AttentionModule, decode_step, model_surgery

__all__ = ["hogwild_fused", "hogwild_sdpa", "hogwild_rope", "hogwild_paged_sdpa", "hogwild_varlen_paged_sdpa", "copy_to_blocks",
           "q4_cache", "copy_to_blocks_q4", "read_blocks_q4", "hogwild_paged_sdpa_q4", "hogwild_varlen_paged_sdpa_q4",
           "hogwild_paged_sdpa_window", "hogwild_varlen_paged_sdpa_window", "packed_slots", "copy_to_slots", "verify_drafts", "trim_blocks",
           "copy_blocks", "fork_blocks", "free_blocks", "reserve_blocks", "compact_blocks", "PagedCache",
           "CacheStructure", "HogwildCache", "SegmentCache", "merge_caches", "AttentionModule", "model_surgery", "decode_step",
           "HAVE_TORCH_OPS"]
