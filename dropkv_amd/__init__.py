"""MI355X (gfx950) implementation of DropKV's prefill-time KV eviction.

Public API (same names and semantics as the reference modules
``dropkv_triton`` / ``dropkv_cache``):

* :func:`dropkv_scores_triton` -- per-key eviction scores;
* :class:`DropKVCache`, :func:`prefill_chunked` -- the evicting cache;
* :mod:`dropkv_amd.ops` -- lower-level ops (scores, select, compact,
  compact2, EvictPlan for one-call layer eviction; tree_attention,
  tree_commit, norm_rope, token_logprobs and verify_drafts for drafted tokens;
  quant_cache, quant_append, quant_read and quant_attention for a cache in 8 bits);
* :class:`dropkv_amd.decode.CompressedDecoder` -- decoding on the compressed
  cache, in 16 or 8 bits, one token or a tree of drafted ones per forward.
"""

from .dropkv_cache import DropKVCache, prefill_chunked
from .dropkv_triton import dropkv_scores_triton

__all__ = ["dropkv_scores_triton", "DropKVCache", "prefill_chunked"]
