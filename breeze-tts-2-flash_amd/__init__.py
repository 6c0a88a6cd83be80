"""MI355X (gfx950) GQA flash-decoding attention for Breeze-TTS-2-flash's decode steps.

Public API:
  gqa_decode(q, k_cache, v_cache, seq_lens, scale, out=None, *, kv_start=None, mask=None, num_splits=0, ...)
  gqa_decode_masked(q, k_cache, v_cache, mask, scale, out=None, ...)
  gqa_decode_wave(q, k_cache, v_cache, seq_lens, scale, out=None, *, kv_start=None)   one wave per q head, short rows
  gqa_decode_fused(qkv, q_norm_weight, k_norm_weight, eps, cos, sin, k_cache, v_cache, cache_pos, scale, ...)
  gqa_decode_probs(q, k_cache, seq_lens, scale, probs=None, *, kv_start=None, mask=None)   softmax probabilities (dbg)
  attn_decode(query, kc, vc, mask, scaling, scores, cmax, part, counters, out, dbg=None)   (reference order)
  attn_decode_fused(qkv, qn_w, kn_w, eps, cos, sin, kc, vc, mask, cache_pos, scaling, ..., out, dbg=None)
  gemv_seg / gemv_resid / gemv_gateup / rmsnorm   backbone decode GEMVs (reference order; C ABI include/bz_gemv.h)
  gqa_window(q, k_cache, v_cache, seq_lens, scale, window, out=None, *, sinks=0, ...)   sliding window + sinks, 1..n tokens
  kv4_cache / kv4_store / kv4_load, gqa_decode_kv4(q, cache, seq_lens, scale, ...)   a KV cache in 4 bits and its attention
  gqa_decode_tracked(..., weights, ...), kv_select / kv_compact / kv_evict   eviction by accumulated attention weight
  rope_frequencies / rope(x, positions, freqs)   rotary positions: half or interleaved pairs, part of a head, long contexts
  paged_cache / rope_store / paged_store / paged_load   a KV cache in pages, bf16 or 8 bits, and a step's q, k, v on the way
  gqa_paged(q, cache, page_table, seq_lens, scale, q_start)   attention of each row's new tokens, 1..n, over its pages
  mask_interval(mask, capacity, ...)   the [kv_start, seq_lens) rows of an interval mask, once per decode step
  backbone.fused_decode_step(graph) / backbone.install(BackboneGraph)   the whole backbone decode step
  build() / load()   compile / open libbz_gqa_decode.so (C ABI: include/*.h)
  torch.ops.bz.*     the same entry points as torch operators (torch_ops.py), used while torch.compile traces
"""
from .attention import (default_splits, get_workspace, gqa_decode, gqa_decode_fused, gqa_decode_masked,
                        gqa_decode_probs, gqa_decode_wave, mask_interval, workspace_bytes)
from .compat import attn_decode, attn_decode_fused
from .gemv import gemv_gateup, gemv_resid, gemv_seg, rmsnorm
from .kernels import build, load
from .long_cache import (Kv4Cache, gqa_decode_kv4, gqa_decode_tracked, gqa_window, kv4_cache, kv4_load, kv4_store, kv_compact,
                         kv_evict, kv_select, long_workspace)
from .paged_cache import PagedCache, gqa_paged, paged_cache, paged_load, paged_store, paged_workspace, rope_store
from .rotary import Rope, rope, rope_frequencies
from . import backbone, hf_attention, torch_ops

__all__ = ["gqa_decode", "gqa_decode_masked", "gqa_decode_wave", "gqa_decode_fused", "gqa_decode_probs", "attn_decode",
           "attn_decode_fused", "gemv_seg", "gemv_resid", "gemv_gateup", "rmsnorm", "mask_interval", "backbone",
           "gqa_window", "Kv4Cache", "kv4_cache", "kv4_store", "kv4_load", "gqa_decode_kv4", "gqa_decode_tracked", "kv_select",
           "kv_compact", "kv_evict", "long_workspace",
           "Rope", "rope_frequencies", "rope", "PagedCache", "paged_cache", "paged_workspace", "paged_store", "rope_store",
           "paged_load", "gqa_paged",
           "workspace_bytes", "default_splits", "get_workspace", "build", "load"]
