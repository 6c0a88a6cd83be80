"""A KV cache in pages, as a server keeps it: rows grow page by page, pages are shared and given back, and a step's batch holds rows with
one new token next to chunks of prompts. rope_store and paged_store put a step's new keys and values into the pages (bf16, or
8 bits), paged_load reads them back, gqa_paged is the attention of the new tokens over them. Every call goes through the C ABI of
libbz_gqa_decode.so (include/bz_paged_cache.h), by way of the native binding (csrc/eager_paged.hpp).

The reference keeps one static cache row per batch row (third_party/breeze-tts/models/cudagraph/backbone_graph.py:73-75) and decodes one
token a row (flash/csrc/bb_attn.cu:416-429).

The batch's tokens. `page_table` int32 [B, pages a row], `seq_lens` int32 [B] (with the new tokens) and `q_start` int32 [B + 1] say where
the N tokens of a call belong: row b's are q_start[b] .. q_start[b + 1] - 1, the last positions of the row; position p lies in page
page_table[b, p / page_size]. q_start None: one token a row. Tokens behind q_start[B] are a batch's padding: nothing of theirs is
stored, and their rows of an output are left as they were (in one that the call allocates, whatever its memory held). Page numbers outside the cache (-1) hold nothing. All three are read on
the device, so a captured graph follows them.

Workspaces: gqa_paged makes one for each device and stream on first use, for calls of all sizes. A call made while its stream is being
captured into a HIP graph needs workspace=, made beforehand by paged_workspace. Errors raise RuntimeError.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from . import kernels
from .attention import _check
from .long_cache import _again
from .rotary import Rope, _flag


class PagedCache(NamedTuple):
    """Pages of K and V [pages, NKV, page_size, D], bf16, or float8_e4m3fn with scales uint8 [pages, NKV, page_size]
    (include/bz_paged_cache.h has the format)."""
    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor | None = None
    v_scale: torch.Tensor | None = None


def paged_cache(pages: int, num_kv_heads: int, page_size: int, head_dim: int, device, dtype=torch.bfloat16) -> PagedCache:
    """An empty cache (all zeros). dtype bfloat16, or float8_e4m3fn: one byte a value and one a (position, head). page_size: a power
    of two from 16 to 1024; head_dim 64 or 128."""
    _check(dtype in (torch.bfloat16, torch.float8_e4m3fn), f"dtype must be bfloat16 or float8_e4m3fn, got {dtype}")
    _check(head_dim in (64, 128), f"head_dim must be 64 or 128, got {head_dim}")
    _check(16 <= page_size <= 1024 and page_size & (page_size - 1) == 0,
           f"page_size must be a power of two from 16 to 1024, got {page_size}")
    _check(pages > 0 and num_kv_heads > 0, "pages and num_kv_heads must be positive")
    shape = (pages, num_kv_heads, page_size, head_dim)
    if dtype == torch.bfloat16:
        return PagedCache(*(torch.zeros(shape, dtype=dtype, device=device) for _ in range(2)))
    k, v = (torch.zeros(shape, dtype=torch.uint8, device=device).view(dtype) for _ in range(2))
    return PagedCache(k, v, *(torch.full(shape[:3], 127, dtype=torch.uint8, device=device) for _ in range(2)))


def paged_workspace(device: torch.device, head_dim: int, group: int, max_tokens: int = 0) -> torch.Tensor:
    """A new zero-filled workspace for gqa_paged, to be passed as workspace= (a captured graph keeps the one it was captured with, and
    graphs that share one must not run at the same time). group: q heads per kv head. max_tokens: what the calls pass, 1 for calls without
    q_start; up to 16 / group a ninth of the bytes is needed, up to 64 / group a quarter."""
    device = torch.device(device)
    idx = device.index if device.index is not None else torch.cuda.current_device()
    n = ctypes.c_size_t(0)
    kernels.run_on(torch.device("cuda", idx), lambda _: kernels.check(kernels.load().bz_paged_workspace_size(
        head_dim, group, max_tokens, ctypes.byref(n)), "bz_paged_workspace_size"))
    return torch.zeros(n.value, dtype=torch.uint8, device=torch.device("cuda", idx))


def paged_store(k: torch.Tensor, v: torch.Tensor, cache: PagedCache, page_table: torch.Tensor, seq_lens: torch.Tensor,
                q_start: torch.Tensor | None = None) -> PagedCache:
    """Stores the new tokens' keys and values as they are (bz_paged_store). k, v: bf16 [N, NKV, D]; a cache of 8 bits takes each
    vector's largest magnitude for its scale. Positions without a page are dropped. Returns cache."""
    if torch.compiler.is_compiling():
        torch.ops.bz.paged_store(k, v, *cache, page_table, seq_lens, q_start)
        return cache
    ck, cv, ks, vs = cache
    kernels.eager().paged_store(k, v, ck, cv, ks, vs, page_table, seq_lens, q_start)
    return cache


def rope_store(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cache: PagedCache, page_table: torch.Tensor,
               seq_lens: torch.Tensor, freqs: Rope, q_start: torch.Tensor | None = None, out: torch.Tensor | None = None, *,
               positions: torch.Tensor | None = None, q_norm_weight: torch.Tensor | None = None,
               k_norm_weight: torch.Tensor | None = None, eps: float = 1e-6) -> torch.Tensor:
    """What stands between a layer's q, k, v projections and gqa_paged, in one launch (bz_paged_store): q and k normed over each head
    (where weights bf16 [D] are given) and turned by their tokens' positions, k and v stored in the pages. q, k, v: bf16 [N, heads,
    D], as views of one projection's output or not. positions int32 or int64 [N]: to turn by, in place of the tokens' places in their
    rows (after an eviction, say). Everything is worked out in fp32 and rounded once. out may be q. Returns out, the turned q."""
    if torch.compiler.is_compiling():
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device) if out is None else out
        torch.ops.bz.rope_store(q, k, v, *cache, page_table, seq_lens, freqs[0], float(freqs[1]), _flag(freqs[2], "interleaved"), q_start,
                                out, positions, q_norm_weight, k_norm_weight, float(eps))
        return out
    ck, cv, ks, vs = cache
    return kernels.eager().rope_store(q, k, v, ck, cv, ks, vs, page_table, seq_lens, freqs[0], freqs[1], freqs[2], q_start, out,
                                      positions, q_norm_weight, k_norm_weight, eps)


def paged_load(cache: PagedCache, page_table: torch.Tensor, starts: torch.Tensor, tokens: int, k: torch.Tensor | None = None,
               v: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """The bf16 values of positions starts[b] .. starts[b] + tokens - 1 of each row (bz_paged_load), exactly as gqa_paged reads them;
    zeros where there is no page. starts: int32 [B]. k, v: optional outputs [B, NKV, tokens, D] bf16. Returns (k, v)."""
    if torch.compiler.is_compiling():
        _check((k is None) == (v is None), "paged_load takes both outputs or neither")
        if k is None:
            _, NKV, _, D = cache[0].shape
            k, v = (torch.empty(page_table.size(0), NKV, tokens, D, dtype=torch.bfloat16, device=cache[0].device) for _ in range(2))
        torch.ops.bz.paged_load(*cache, page_table, starts, int(tokens), k, v)
        return k, v
    ck, cv, ks, vs = cache
    return kernels.eager().paged_load(ck, cv, ks, vs, page_table, starts, tokens, k, v)


def gqa_paged(q: torch.Tensor, cache: PagedCache, page_table: torch.Tensor, seq_lens: torch.Tensor, scale: float,
              q_start: torch.Tensor | None = None, out: torch.Tensor | None = None, *, max_tokens: int = 0, max_seq_len: int = 0,
              workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Causal GQA attention of every row's new tokens over its pages (bz_gqa_paged): one token a row (a decode step), a few (a
    verified draft), a prompt's chunk, or all of these in one batch. q: bf16 [N, NH, D], NH / NKV of 1, 2, 4 or 8; a token at position
    p of its row attends [0, p]. max_tokens, max_seq_len: about the most new tokens and positions of a row, where known; they steer
    the launch, and with it the order of sums and whether softmax terms of rows of more than NKV 16 / NH tokens meet V as two bf16 terms or
    as one. A token that attends nothing gets zeros; nothing stored at positions a token does not attend reaches its
    output. Returns out [N, NH, D]."""
    if torch.compiler.is_compiling():
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device) if out is None else out
        torch.ops.bz.gqa_paged(q, *cache, page_table, seq_lens, float(scale), q_start, out, int(max_tokens), int(max_seq_len),
                               workspace)
        return out
    entry = kernels.eager().paged
    ck, cv, ks, vs = cache
    r = entry(q, ck, cv, ks, vs, page_table, seq_lens, scale, q_start, out, max_tokens, max_seq_len, workspace)
    return r if type(r) is not tuple else _again(r, entry, q, ck, cv, ks, vs, page_table, seq_lens, scale, q_start, out,
                                                 max_tokens, max_seq_len, workspace)
