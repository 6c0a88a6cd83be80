"""Keeping a long KV cache small, and reading it: attention with a sliding window and sinks (gqa_window), a cache held in 4
bits (kv4_cache, kv4_store, kv4_load, gqa_decode_kv4), and eviction by accumulated attention weight (gqa_decode_tracked,
kv_select, kv_compact, kv_evict). Every call goes through the C ABI of libbz_gqa_decode.so (include/bz_long_cache.h), by way
of the native binding (csrc/eager_long.hpp), which checks the tensors, picks the stream and workspace and calls the C entry.

The reference keeps every position of its static cache (third_party/breeze-tts/models/cudagraph/backbone_graph.py:73-75)
in bf16 and attends all of them (flash/csrc/bb_attn.cu:416-429); these operators bound what a decode step reads instead.

Workspaces: made on first use, for each device, stream and kind of call one for calls of up to 512 units (bz_long_cache.h),
one up to 1024, and so on. A call made while its stream is being captured into a HIP graph takes none of those, which graphs
would then share: it needs workspace=, made beforehand by long_workspace (one serves every call of a graph with as many units,
rounded up so; the calls that need none are captured without). Errors raise RuntimeError.
"""
from __future__ import annotations

import ctypes
import functools
from typing import NamedTuple

import torch

from . import attention, kernels
from .attention import _check

_WS: dict = {}  # (device index, raw stream handle, kind, sharing) -> workspace (csrc/eager_long.hpp: sharing_of)
_KINDS = {"window": kernels.LONG_WINDOW, "kv4": kernels.LONG_KV4, "tracked": kernels.LONG_TRACKED}


class Kv4Cache(NamedTuple):
    """A KV cache in 4 bits: codes k, v uint8 [B, NKV, capacity, D / 2] and scales k_scale, v_scale uint8 [B, NKV, capacity,
    D / 32] (include/bz_long_cache.h has the format)."""
    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor


def kv4_cache(batch: int, num_kv_heads: int, capacity: int, head_dim: int, device) -> Kv4Cache:
    """An empty 4-bit cache (all zeros): 4.25 bits a value where a bf16 cache has 16. head_dim 64 or 128."""
    _check(head_dim in (64, 128), f"head_dim must be 64 or 128, got {head_dim}")
    _check(batch > 0 and num_kv_heads > 0 and capacity > 0, "batch, num_kv_heads and capacity must be positive")
    make = lambda w: torch.zeros(batch, num_kv_heads, capacity, w, dtype=torch.uint8, device=device)  # noqa: E731
    return Kv4Cache(make(head_dim // 2), make(head_dim // 2), make(head_dim // 32), make(head_dim // 32))


# ------------------------------------------------------------------------------------------------- workspaces

@functools.lru_cache(maxsize=1024)
def _bytes(idx: int, kind: int, B: int, NH: int, NKV: int, D: int, cap: int, T: int, window: int, sinks: int, splits: int,
           longest: int) -> int:
    """bz_long_workspace_size with device idx current."""
    n = ctypes.c_size_t(0)
    kernels.run_on(torch.device("cuda", idx), lambda _: kernels.check(kernels.load().bz_long_workspace_size(
        kind, B, NH, NKV, D, cap, T, window, sinks, splits, longest, ctypes.byref(n)), "bz_long_workspace_size"))
    return int(n.value)


def _make_workspace(need) -> None:
    """Makes and registers the workspace that the native binding asked for: need = (device index, raw stream handle, kind,
    sharing, bytes). One serves calls of all sizes of up to 512 units, another those of up to 1024, and so on (bz_long_cache.h).
    Grown, never shrunk. A replaced one is kept: it was allocated on a stream of its own, and calls on this one may still be at
    work in it."""
    key, n = need[:4], need[4]
    with attention._WS_LOCK:
        ws = _WS.get(key)
        if ws is None or ws.numel() < n:
            new = attention._zeroed_outside_pools(n if ws is None else max(n, 2 * ws.numel()), key[0])
            _check(new.data_ptr() % 256 == 0, "workspace allocation is not 256-byte aligned")
            if ws is not None:
                attention._WS_RETIRED.append(ws)
            _WS[key] = ws = new
        kernels.eager().register_long_workspace(*key, ws)


def _again(need, entry, *args):
    """entry(*args) of the native binding once more, with the workspace it asked for (need, the tuple it returned)."""
    _make_workspace(need)
    return entry(*args)


def _call(entry, *args):
    """entry(*args) of the native binding, with the workspace it may ask for (for the torch operators)."""
    r = entry(*args)
    return r if type(r) is not tuple else _again(r, entry, *args)


def long_workspace(kind: str, device: torch.device, batch: int, num_q_heads: int, num_kv_heads: int, head_dim: int,
                   capacity: int, tokens: int = 1, *, window: int = 0, sinks: int = 0, num_splits: int = 0,
                   max_seq_len: int = 0) -> torch.Tensor:
    """A new zero-filled workspace for calls of gqa_window ("window"), gqa_decode_kv4 ("kv4") or gqa_decode_tracked
    ("tracked") with these sizes, to be passed as workspace= (a captured graph keeps the one it was captured with, and
    graphs that share one must not run at the same time). Empty where such calls need none."""
    _check(kind in _KINDS, f"kind must be one of {sorted(_KINDS)}, got {kind!r}")
    idx = device.index if device.index is not None else torch.cuda.current_device()
    n = _bytes(idx, _KINDS[kind], batch, num_q_heads, num_kv_heads, head_dim, capacity, tokens, window, sinks, num_splits,
               max_seq_len)
    return torch.zeros(n, dtype=torch.uint8, device=torch.device("cuda", idx))


# ---------------------------------------------------------------------------------------- window attention

def gqa_window(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, seq_lens: torch.Tensor, scale: float,
               window: int, out: torch.Tensor | None = None, *, sinks: int = 0, kv_start: torch.Tensor | None = None,
               num_splits: int = 0, max_seq_len: int = 0, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Causal GQA attention over a sliding window and the row's first positions (bz_gqa_window).

    q: [B, NH, D] or [B, NH, T, D] bf16, any T from one decode token to a whole prompt; row b's tokens are its last T
    positions, token t at position p = seq_lens[b] - T + t. It attends the last `window` positions up to its own (window
    0: all) and the row's first `sinks` positions, both from kv_start[b] on. k_cache, v_cache, seq_lens, kv_start, out
    and max_seq_len as in gqa_decode. A token that attends nothing gets zeros; nothing stored at positions a token does not
    attend reaches its output. Returns out."""
    if torch.compiler.is_compiling():
        out = attention._default_out(q) if out is None else out
        torch.ops.bz.gqa_window(q, k_cache, v_cache, seq_lens, float(scale), int(window), out, int(sinks), kv_start,
                                int(num_splits), int(max_seq_len), workspace)
        return out
    # (the binding called here, not through another function: 0.3 us of a 4.8 us call)
    entry = kernels.eager().window
    r = entry(q, k_cache, v_cache, seq_lens, scale, window, out, sinks, kv_start, num_splits, max_seq_len, workspace)
    return r if type(r) is not tuple else _again(r, entry, q, k_cache, v_cache, seq_lens, scale, window, out, sinks, kv_start,
                                                 num_splits, max_seq_len, workspace)


# --------------------------------------------------------------------------------------------- 4-bit cache

def kv4_store(k: torch.Tensor, v: torch.Tensor, cache: Kv4Cache, slots: torch.Tensor, *,
              counts: torch.Tensor | None = None) -> Kv4Cache:
    """Rounds new keys and values into a 4-bit cache (bz_kv4_store). k, v: [B, NKV, T, D] bf16 with equal strides; row b's
    tokens go to the slots slots[b] .. slots[b] + T - 1 (slots: int32 [B]); with counts (int32 [B]) only the first counts[b]
    tokens of row b, the rest being a batch's padding. Slots outside the cache are skipped. Returns cache."""
    if torch.compiler.is_compiling():
        torch.ops.bz.kv4_store(k, v, *cache, slots, counts)
        return cache
    kernels.eager().kv4_store(k, v, *cache, slots, counts)
    return cache


def kv4_load(cache: Kv4Cache, slots: torch.Tensor, tokens: int, k: torch.Tensor | None = None,
             v: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """The bf16 values of slots slots[b] .. slots[b] + tokens - 1 of a 4-bit cache (bz_kv4_load), exactly as gqa_decode_kv4
    reads them; zeros for slots outside the cache. k, v: optional outputs [B, NKV, tokens, D] bf16. Returns (k, v)."""
    if torch.compiler.is_compiling():
        _check((k is None) == (v is None), "kv4_load takes both outputs or neither")
        if k is None:
            B, NKV, _, half = cache[0].shape
            k, v = (torch.empty(B, NKV, tokens, 2 * half, dtype=torch.bfloat16, device=cache[0].device) for _ in range(2))
        torch.ops.bz.kv4_load(*cache, slots, int(tokens), k, v)
        return k, v
    return kernels.eager().kv4_load(*cache, slots, tokens, k, v)


def gqa_decode_kv4(q: torch.Tensor, cache: Kv4Cache, seq_lens: torch.Tensor, scale: float, out: torch.Tensor | None = None, *,
                   kv_start: torch.Tensor | None = None, window: int = 0, sinks: int = 0, num_splits: int = 0,
                   max_seq_len: int = 0, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """GQA decode attention over a 4-bit cache (bz_gqa_decode_kv4): gqa_window's ranges (window 0: the whole row) over the
    values the codes stand for, one to 16 query tokens per row (q: [B, NH, D] or [B, NH, T, D] bf16). A longer chunk goes
    through kv4_load and gqa_window. Returns out."""
    if torch.compiler.is_compiling():
        out = attention._default_out(q) if out is None else out
        torch.ops.bz.gqa_decode_kv4(q, *cache, seq_lens, float(scale), out, kv_start, int(window), int(sinks), int(num_splits),
                                    int(max_seq_len), workspace)
        return out
    entry = kernels.eager().kv4
    ck, cv, ks, vs = cache
    r = entry(q, ck, cv, ks, vs, seq_lens, scale, out, kv_start, window, sinks, num_splits, max_seq_len, workspace)
    return r if type(r) is not tuple else _again(r, entry, q, ck, cv, ks, vs, seq_lens, scale, out, kv_start, window, sinks,
                                                 num_splits, max_seq_len, workspace)


# ------------------------------------------------------------------------------------------------ eviction

def gqa_decode_tracked(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, seq_lens: torch.Tensor, scale: float,
                       weights: torch.Tensor, out: torch.Tensor | None = None, *, decay: float = 1.0,
                       weights_out: torch.Tensor | None = None, kv_start: torch.Tensor | None = None, num_splits: int = 0,
                       max_seq_len: int = 0, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """gqa_decode for one query token per row that also keeps account of the attention weights (bz_gqa_decode_tracked):
    weights_out[b, h, p] = decay * weights[b, h, p] + the softmax probabilities of position p summed over the q heads of kv
    head h, for p in [kv_start[b], seq_lens[b]); other positions are left as they were. weights: float32 [B, NKV,
    capacity]; weights_out None: in place. kv_select / kv_evict choose by them. Returns out."""
    weights_out = weights if weights_out is None else weights_out
    if torch.compiler.is_compiling():
        out = attention._default_out(q) if out is None else out
        torch.ops.bz.gqa_decode_tracked(q, k_cache, v_cache, seq_lens, float(scale), weights, out, float(decay),
                                        weights_out, kv_start, int(num_splits), int(max_seq_len), workspace)
        return out
    entry = kernels.eager().tracked
    r = entry(q, k_cache, v_cache, seq_lens, scale, weights, out, decay, weights_out, kv_start, num_splits, max_seq_len, workspace)
    return r if type(r) is not tuple else _again(r, entry, q, k_cache, v_cache, seq_lens, scale, weights, out, decay, weights_out,
                                                 kv_start, num_splits, max_seq_len, workspace)


def kv_select(weights: torch.Tensor, seq_lens: torch.Tensor, keep: int, *, sinks: int = 0, recent: int = 0,
              kv_start: torch.Tensor | None = None, index: torch.Tensor | None = None, lens: torch.Tensor | None = None,
              weights_out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Which positions of each (row, kv head) stay when at most `keep` may (bz_kv_select): all of a row that holds no more;
    else its first `sinks`, its last `recent`, and the heaviest of the others (of equal weights the lower position, NaN
    first). weights: float32 [B, NKV, capacity]. Returns index, int32 [B, NKV, keep]: the positions, ascending, then -1; and
    lens, int32 [B]: how many. index, lens: optional outputs (lens may be seq_lens). weights_out (may be weights): the kept
    weights from slot 0 on, zeros behind them up to the row's old end."""
    if torch.compiler.is_compiling():
        B, NKV, dev = weights.size(0), weights.size(1), weights.device
        index = torch.empty(B, NKV, keep, dtype=torch.int32, device=dev) if index is None else index
        lens = torch.empty(B, dtype=torch.int32, device=dev) if lens is None else lens
        torch.ops.bz.kv_select(weights, seq_lens, int(keep), int(sinks), int(recent), kv_start, index, lens, weights_out)
        return index, lens
    return kernels.eager().select(weights, seq_lens, keep, sinks, recent, kv_start, index, lens, weights_out)


def kv_compact(tensors, index: torch.Tensor, lens: torch.Tensor, outs=None):
    """Moves the chosen rows of a cache together (bz_kv_compact): for each tensor [B, NKV, capacity, X] (any dtype; (k, v), or
    a Kv4Cache), row d of each (row, kv head) becomes its row index[b, h, d], for d < lens[b]; other rows are left as they
    were. outs: tensors of the same shapes, or None for in place (index must ascend, as kv_select's does). Up to 4 tensors.
    Returns outs."""
    if torch.compiler.is_compiling():
        outs = tensors if outs is None else outs
        torch.ops.bz.kv_compact(list(tensors), index, lens, list(outs))
        return outs
    kernels.eager().compact(tensors, index, lens, outs)
    return tensors if outs is None else outs


def kv_evict(tensors, weights: torch.Tensor, seq_lens: torch.Tensor, keep: int, *, sinks: int = 0, recent: int = 0,
             kv_start: torch.Tensor | None = None, outs=None,
             weights_out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """kv_select, and the cache's tensors and weights compacted to what stays (in place unless outs / weights_out are given;
    the weights move with the selection, so weights_out shares no memory with the tensors).
    The kept positions of row b are then the slots [0, lens[b]) of every kv head, in their old order, so later calls take
    lens for seq_lens and no kv_start. Returns (index, lens)."""
    weights_out = weights if weights_out is None else weights_out
    if torch.compiler.is_compiling():
        index, lens = kv_select(weights, seq_lens, keep, sinks=sinks, recent=recent, kv_start=kv_start, weights_out=weights_out)
        kv_compact(tensors, index, lens, outs)
        return index, lens
    return kernels.eager().evict(weights, seq_lens, keep, sinks, recent, kv_start, None, None, weights_out, tensors, outs)
