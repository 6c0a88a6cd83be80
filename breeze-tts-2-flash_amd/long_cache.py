"""Keeping a long KV cache small, and reading it: attention with a sliding window and sinks (gqa_window), a cache held in 4
bits (kv4_cache, kv4_store, kv4_load, gqa_decode_kv4), and eviction by accumulated attention weight (gqa_decode_tracked,
kv_select, kv_compact, kv_evict). Every call goes through the C ABI of libbz_gqa_decode.so (include/bz_long_cache.h).

The reference keeps every position of its static cache (third_party/breeze-tts/models/cudagraph/backbone_graph.py:73-75)
in bf16 and attends all of them (flash/csrc/bb_attn.cu:416-429); these operators bound what a decode step reads instead.

Workspaces follow attention.py: one per device, stream and kind of call, made on first use, never while the stream is being
captured into a HIP graph (pass workspace=, made beforehand by long_workspace). Errors raise RuntimeError.
"""
from __future__ import annotations

import ctypes
import functools
from typing import NamedTuple

import torch

from . import attention, kernels
from .attention import _check, _int32_rows, _out_view, _q_view

_WS: dict = {}  # (device index, raw stream handle, kind, batch, NH, NKV, T) -> workspace
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


def _workspace(idx, stream, kind, B, NH, NKV, D, cap, T, window, sinks, splits, longest):
    """The cached workspace of these sizes on stream (None where the call needs none): grown, never shrunk, replaced ones
    kept for graphs that may hold them, as attention.get_workspace keeps its own."""
    n = _bytes(idx, kind, B, NH, NKV, D, cap, T, window, sinks, splits, longest)
    if n == 0:
        return None
    key = (idx, stream, kind, B, NH, NKV, T)
    ws = _WS.get(key)
    if ws is not None and ws.numel() >= n:
        return ws
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"no workspace of {n} bytes exists for the stream being captured, and nothing is allocated during "
                           "a capture: pass workspace= (long_workspace(...), made before the capture)")
    with attention._WS_LOCK:
        ws = _WS.get(key)
        if ws is None or ws.numel() < n:
            new = attention._zeroed_outside_pools(n if ws is None else max(n, 2 * ws.numel()), idx)
            _check(new.data_ptr() % 256 == 0, "workspace allocation is not 256-byte aligned")
            if ws is not None:
                attention._WS_RETIRED.append(ws)
            _WS[key] = ws = new
    return ws


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


def _launch(entry, args, a, kind, dev, workspace, window, sinks):
    """Calls entry(args) on dev's current stream; a: the bz_gqa_decode_args inside args."""
    fn = getattr(kernels.load(), entry)

    def launch(stream):
        ws = workspace
        if ws is None:
            ws = _workspace(dev.index, stream, kind, a.batch, a.num_q_heads, a.num_kv_heads, a.head_dim, a.capacity,
                            a.tokens_per_row, window, sinks, a.num_splits, a.max_seq_len)
        if ws is not None:
            a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel() * ws.element_size()
        kernels.check(fn(ctypes.byref(args), ctypes.c_void_p(stream)), entry)

    kernels.run_on(dev, launch)


def _check_workspace(workspace, dev) -> None:
    _check(workspace is None or (workspace.device == dev and workspace.is_contiguous()),
           "workspace must be a contiguous tensor on the query's device")


def _fill_q(a, q, seq_lens, kv_start, scale, out, num_splits, max_seq_len):
    """The query's, ranges' and output's part of a bz_gqa_decode_args; returns the output."""
    B, NH, T, D, q_sb, q_sh, q_st = _q_view(q)
    if out is None:
        out = attention._default_out(q)
    _check(out.device == q.device, "out must be on the query's device")
    o_sb, o_sh, o_st = _out_view(out, B, NH, T, D)
    a.q, a.q_stride_b, a.q_stride_h, a.q_stride_t = q.data_ptr(), q_sb, q_sh, q_st
    a.tokens_per_row = T
    a.seq_lens = _int32_rows(seq_lens, B, "seq_lens", q.device).data_ptr()
    a.kv_start = _int32_rows(kv_start, B, "kv_start", q.device).data_ptr() if kv_start is not None else None
    a.scale = float(scale)
    a.out, a.out_stride_b, a.out_stride_h, a.out_stride_t = out.data_ptr(), o_sb, o_sh, o_st
    a.batch, a.num_q_heads, a.head_dim = B, NH, D
    a.num_splits, a.max_seq_len = int(num_splits), int(max_seq_len)
    return out


def _fill_cache(a, q, k_cache, v_cache) -> None:
    _check(k_cache.dtype == torch.bfloat16 and v_cache.dtype == torch.bfloat16, "k_cache and v_cache must be bf16")
    _check(k_cache.device == q.device and v_cache.device == q.device, "all tensors must be on one device")
    _check(k_cache.dim() == 4 and v_cache.shape == k_cache.shape and v_cache.stride() == k_cache.stride(),
           "k_cache and v_cache must be [B, NKV, capacity, D] with equal shapes and strides")
    _check(k_cache.size(0) == q.size(0) and k_cache.size(3) == q.size(-1) and k_cache.stride(3) == 1,
           f"k_cache {tuple(k_cache.shape)} does not match query {tuple(q.shape)}")
    a.k_cache, a.v_cache = k_cache.data_ptr(), v_cache.data_ptr()
    a.kv_stride_b, a.kv_stride_h, a.kv_stride_s = k_cache.stride(0), k_cache.stride(1), k_cache.stride(2)
    a.num_kv_heads, a.capacity = k_cache.size(1), k_cache.size(2)


def _check_q(q) -> None:
    _check(q.is_cuda, "query must be a device tensor")
    _check(q.dtype == torch.bfloat16, "query must be bf16")
    _check(q.stride(-1) == 1, "query's head_dim must be contiguous")


def _check_reach(window, sinks) -> None:
    _check(0 <= int(window) <= 2**31 - 1 and 0 <= int(sinks) <= 2**31 - 1, "window and sinks must be int32 and not negative")


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
    return _gqa_window(q, k_cache, v_cache, seq_lens, scale, window, out, sinks, kv_start, num_splits, max_seq_len, workspace)


def _gqa_window(q, k_cache, v_cache, seq_lens, scale, window, out, sinks, kv_start, num_splits, max_seq_len, workspace):
    _check_q(q)
    _check_reach(window, sinks)
    _check_workspace(workspace, q.device)
    w = kernels.GqaWindowArgs()
    a = w.base
    out = _fill_q(a, q, seq_lens, kv_start, scale, out, num_splits, max_seq_len)
    _fill_cache(a, q, k_cache, v_cache)
    w.window, w.sinks = int(window), int(sinks)
    _launch("bz_gqa_window", w, a, kernels.LONG_WINDOW, q.device, workspace, w.window, w.sinks)
    return out


# --------------------------------------------------------------------------------------------- 4-bit cache

def _kv4_args(cache: Kv4Cache):
    """bz_kv4_cache of a checked cache."""
    k, v, ks, vs = cache
    _check(all(t.is_cuda and t.dtype == torch.uint8 and t.dim() == 4 and t.device == k.device for t in cache),
           "a 4-bit cache is four uint8 device tensors [B, NKV, capacity, ..] on one device")
    D = 2 * k.size(3)
    _check(v.shape == k.shape and v.stride() == k.stride() and k.stride(3) == 1,
           "codes k and v must have equal shapes and strides and a contiguous last dim")
    _check(ks.shape == vs.shape == (*k.shape[:3], D // 32) and ks.stride() == vs.stride(),
           f"scales must be [B, NKV, capacity, D / 32] = {(*k.shape[:3], D // 32)} with equal strides")
    _check(ks.stride(3) == 1 and ks.stride(2) == D // 32, "the last two dims of the scales must be contiguous")
    c = kernels.Kv4CacheArgs()
    c.k, c.v, c.k_scale, c.v_scale = k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr()
    c.stride_b, c.stride_h, c.stride_s = k.stride(0), k.stride(1), k.stride(2)
    c.scale_stride_b, c.scale_stride_h = ks.stride(0), ks.stride(1)
    c.batch, c.num_kv_heads, c.capacity, c.head_dim = k.size(0), k.size(1), k.size(2), D
    return c


def _check_kv(k, v, c, dev) -> None:
    _check(k.dtype == torch.bfloat16 and v.dtype == torch.bfloat16 and k.device == dev and v.device == dev,
           "k and v must be bf16 on the cache's device")
    _check(k.dim() == 4 and v.shape == k.shape and v.stride() == k.stride() and k.stride(3) == 1,
           "k and v must be [B, NKV, T, D] with equal shapes and strides and a contiguous last dim")
    _check((k.size(0), k.size(1), k.size(3)) == (c.batch, c.num_kv_heads, c.head_dim),
           f"k {tuple(k.shape)} does not match a cache of batch {c.batch}, {c.num_kv_heads} heads, head_dim {c.head_dim}")


def kv4_store(k: torch.Tensor, v: torch.Tensor, cache: Kv4Cache, slots: torch.Tensor, *,
              counts: torch.Tensor | None = None) -> Kv4Cache:
    """Rounds new keys and values into a 4-bit cache (bz_kv4_store). k, v: [B, NKV, T, D] bf16; row b's tokens go to the
    slots slots[b] .. slots[b] + T - 1 (slots: int32 [B]); with counts (int32 [B]) only the first counts[b] tokens of row b,
    the rest being a batch's padding. Slots outside the cache are skipped. Returns cache."""
    if torch.compiler.is_compiling():
        torch.ops.bz.kv4_store(k, v, *cache, slots, counts)
        return cache
    return _kv4_store(k, v, cache, slots, counts)


def _kv4_store(k, v, cache, slots, counts):
    c = _kv4_args(cache)
    dev = cache[0].device
    _check_kv(k, v, c, dev)
    _int32_rows(slots, c.batch, "slots", dev)
    if counts is not None:
        _int32_rows(counts, c.batch, "counts", dev)
    kernels.run_on(dev, lambda stream: kernels.check(kernels.load().bz_kv4_store(
        k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(1), k.stride(2), k.size(2), slots.data_ptr(),
        None if counts is None else counts.data_ptr(), ctypes.byref(c), stream), "bz_kv4_store"))
    return cache


def kv4_load(cache: Kv4Cache, slots: torch.Tensor, tokens: int, k: torch.Tensor | None = None,
             v: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """The bf16 values of slots slots[b] .. slots[b] + tokens - 1 of a 4-bit cache (bz_kv4_load), exactly as gqa_decode_kv4
    reads them; zeros for slots outside the cache. k, v: optional outputs [B, NKV, tokens, D] bf16. Returns (k, v)."""
    if k is None or v is None:
        _check(k is None and v is None, "kv4_load takes both outputs or neither")
        B, NKV, _, half = cache[0].shape
        k, v = (torch.empty(B, NKV, tokens, 2 * half, dtype=torch.bfloat16, device=cache[0].device) for _ in range(2))
    if torch.compiler.is_compiling():
        torch.ops.bz.kv4_load(*cache, slots, k, v)
        return k, v
    _check(k.dim() == 4 and k.size(2) == tokens, f"outputs must hold {tokens} tokens")
    return _kv4_load(cache, slots, k, v)


def _kv4_load(cache, slots, k, v):
    c = _kv4_args(cache)
    dev = cache[0].device
    _check_kv(k, v, c, dev)
    _int32_rows(slots, c.batch, "slots", dev)
    kernels.run_on(dev, lambda stream: kernels.check(kernels.load().bz_kv4_load(
        ctypes.byref(c), slots.data_ptr(), k.size(2), k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(1), k.stride(2),
        stream), "bz_kv4_load"))
    return k, v


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
    return _gqa_decode_kv4(q, cache, seq_lens, scale, out, kv_start, window, sinks, num_splits, max_seq_len, workspace)


def _gqa_decode_kv4(q, cache, seq_lens, scale, out, kv_start, window, sinks, num_splits, max_seq_len, workspace):
    _check_q(q)
    _check_reach(window, sinks)
    _check_workspace(workspace, q.device)
    ka = kernels.GqaKv4Args()
    c = ka.cache = _kv4_args(cache)
    a = ka.base
    out = _fill_q(a, q, seq_lens, kv_start, scale, out, num_splits, max_seq_len)
    _check(cache[0].device == q.device, "all tensors must be on one device")
    _check(c.batch == a.batch and c.head_dim == a.head_dim,
           f"a cache of batch {c.batch} and head_dim {c.head_dim} does not match query {tuple(q.shape)}")
    a.num_kv_heads, a.capacity = c.num_kv_heads, c.capacity
    ka.window, ka.sinks = int(window), int(sinks)
    _launch("bz_gqa_decode_kv4", ka, a, kernels.LONG_KV4, q.device, workspace, ka.window, ka.sinks)
    return out


# ------------------------------------------------------------------------------------------------ eviction

def _weights_view(t, B, NKV, cap, name, dev):
    _check(t.dtype == torch.float32 and t.device == dev and tuple(t.shape) == (B, NKV, cap) and t.stride(2) == 1,
           f"{name} must be float32 [B, NKV, capacity] = {(B, NKV, cap)} on the cache's device, its last dim contiguous")
    return t.stride(0), t.stride(1)


def _span(t):
    """[first, last + 1) byte addresses of t's elements."""
    last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()


def _apart(x, y) -> bool:
    """Whether two tensors [B, NKV, capacity, X] share no memory: their spans lie apart, or they interleave row by row (views
    of one tensor, such as a cache that holds K and V side by side)."""
    (a0, a1), (b0, b1) = _span(x), _span(y)
    if a1 <= b0 or b1 <= a0:
        return True
    nx, ny = x.element_size(), y.element_size()
    steps = [s * nx for n, s in zip(x.shape[:-1], x.stride()[:-1]) if n > 1]
    if steps != [s * ny for n, s in zip(y.shape[:-1], y.stride()[:-1]) if n > 1] or not steps:
        return False
    step = min(steps)
    if step <= 0 or any(s % step for s in steps):
        return False
    gap = (b0 - a0) % step
    return x.size(-1) * nx <= gap and gap + y.size(-1) * ny <= step


def _check_destination(src, dst, name) -> None:
    """dst is src itself (the same elements), or shares none of its memory; every element has a place of its own."""
    _check(all(s > 0 or n == 1 for n, s in zip(dst.shape, dst.stride())), f"{name} must not be a broadcast view")
    if dst.data_ptr() == src.data_ptr() and dst.stride() == src.stride():
        return
    (a0, a1), (b0, b1) = _span(src), _span(dst)
    _check(a1 <= b0 or b1 <= a0, f"{name} must be its source itself or not overlap it")


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
    return _gqa_decode_tracked(q, k_cache, v_cache, seq_lens, scale, weights, out, decay, weights_out, kv_start, num_splits,
                               max_seq_len, workspace)


def _gqa_decode_tracked(q, k_cache, v_cache, seq_lens, scale, weights, out, decay, weights_out, kv_start, num_splits,
                        max_seq_len, workspace):
    _check_q(q)
    _check(q.dim() == 3 or q.size(2) == 1, "gqa_decode_tracked takes one query token per row")
    _check_workspace(workspace, q.device)
    ta = kernels.GqaTrackedArgs()
    a = ta.base
    out = _fill_q(a, q, seq_lens, kv_start, scale, out, num_splits, max_seq_len)
    _fill_cache(a, q, k_cache, v_cache)
    ta.w_stride_b, ta.w_stride_h = _weights_view(weights, a.batch, a.num_kv_heads, a.capacity, "weights", q.device)
    ta.wo_stride_b, ta.wo_stride_h = _weights_view(weights_out, a.batch, a.num_kv_heads, a.capacity, "weights_out", q.device)
    _check_destination(weights, weights_out, "weights_out")
    ta.weights, ta.weights_out, ta.decay = weights.data_ptr(), weights_out.data_ptr(), float(decay)
    _launch("bz_gqa_decode_tracked", ta, a, kernels.LONG_TRACKED, q.device, workspace, 0, 0)
    return out


def kv_select(weights: torch.Tensor, seq_lens: torch.Tensor, keep: int, *, sinks: int = 0, recent: int = 0,
              kv_start: torch.Tensor | None = None, index: torch.Tensor | None = None, lens: torch.Tensor | None = None,
              weights_out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Which positions of each (row, kv head) stay when at most `keep` may (bz_kv_select): all of a row that holds no more;
    else its first `sinks`, its last `recent`, and the heaviest of the others (of equal weights the lower position, NaN
    first). weights: float32 [B, NKV, capacity]. Returns index, int32 [B, NKV, keep]: the positions, ascending, then -1; and
    lens, int32 [B]: how many. index, lens: optional outputs (lens may be seq_lens). weights_out (may be weights): the kept
    weights from slot 0 on, zeros behind them up to the row's old end."""
    B, NKV = weights.size(0), weights.size(1)
    if index is None:
        index = torch.empty(B, NKV, keep, dtype=torch.int32, device=weights.device)
    if lens is None:
        lens = torch.empty(B, dtype=torch.int32, device=weights.device)
    if torch.compiler.is_compiling():
        torch.ops.bz.kv_select(weights, seq_lens, int(keep), int(sinks), int(recent), kv_start, index, lens, weights_out)
        return index, lens
    return _kv_select(weights, seq_lens, keep, sinks, recent, kv_start, index, lens, weights_out)


def _kv_select(weights, seq_lens, keep, sinks, recent, kv_start, index, lens, weights_out):
    _check(weights.is_cuda and weights.dim() == 3, "weights must be a device tensor [B, NKV, capacity]")
    dev = weights.device
    B, NKV, cap = weights.shape
    a = kernels.KvSelectArgs()
    a.w_stride_b, a.w_stride_h = _weights_view(weights, B, NKV, cap, "weights", dev)
    a.weights = weights.data_ptr()
    a.seq_lens = _int32_rows(seq_lens, B, "seq_lens", dev).data_ptr()
    a.kv_start = _int32_rows(kv_start, B, "kv_start", dev).data_ptr() if kv_start is not None else None
    _check(index.dtype == torch.int32 and index.device == dev and tuple(index.shape) == (B, NKV, keep) and
           index.is_contiguous(), f"index must be a contiguous int32 [B, NKV, keep] = {(B, NKV, keep)} device tensor")
    a.index, a.lens = index.data_ptr(), _int32_rows(lens, B, "lens", dev).data_ptr()
    if weights_out is not None:
        a.wo_stride_b, a.wo_stride_h = _weights_view(weights_out, B, NKV, cap, "weights_out", dev)
        _check_destination(weights, weights_out, "weights_out")
        a.weights_out = weights_out.data_ptr()
    a.batch, a.num_kv_heads, a.capacity, a.keep, a.sinks, a.recent = B, NKV, cap, int(keep), int(sinks), int(recent)
    kernels.run_on(dev, lambda stream: kernels.check(kernels.load().bz_kv_select(
        ctypes.byref(a), ctypes.c_void_p(stream)), "bz_kv_select"))
    return index, lens


def kv_compact(tensors, index: torch.Tensor, lens: torch.Tensor, outs=None):
    """Moves the chosen rows of a cache together (bz_kv_compact): for each tensor [B, NKV, capacity, X] (any dtype; (k, v), or
    a Kv4Cache), row d of each (row, kv head) becomes its row index[b, h, d], for d < lens[b]; other rows are left as they
    were. outs: tensors of the same shapes, or None for in place (index must ascend, as kv_select's does). Up to 4 tensors.
    Returns outs."""
    outs = tensors if outs is None else outs
    if torch.compiler.is_compiling():
        torch.ops.bz.kv_compact(list(tensors), index, lens, list(outs))
        return outs
    _kv_compact(tensors, index, lens, outs)
    return outs


def _kv_compact(tensors, index, lens, outs):
    _check(0 < len(tensors) <= kernels.KV_TENSORS and len(outs) == len(tensors),
           f"kv_compact takes one to {kernels.KV_TENSORS} tensors and as many outputs")
    dev = tensors[0].device
    B, NKV, cap = tensors[0].shape[:3]
    _check(index.dtype == torch.int32 and index.device == dev and index.dim() == 3 and index.is_contiguous() and
           tuple(index.shape[:2]) == (B, NKV), "index must be a contiguous int32 [B, NKV, keep] device tensor")
    _int32_rows(lens, B, "lens", dev)
    arr = (kernels.KvTensor * len(tensors))()
    for i, (t, src, dst) in enumerate(zip(arr, tensors, outs)):
        _check(src.is_cuda and src.dim() == 4 and tuple(src.shape[:3]) == (B, NKV, cap) and src.device == dev and
               src.stride(3) == 1, "tensors must be [B, NKV, capacity, X] on one device with a contiguous last dim")
        _check(dst.shape == src.shape and dst.dtype == src.dtype and dst.device == dev and dst.stride(3) == 1,
               "an output must match its tensor")
        _check_destination(src, dst, "an output")
        for other in (*tensors[:i], *tensors[i + 1:], *outs[:i], *outs[i + 1:]):
            _check(_apart(other, dst), "an output must not overlap another tensor")
        n = src.element_size()
        t.src, t.dst, t.row_bytes = src.data_ptr(), dst.data_ptr(), src.size(3) * n
        t.src_stride_b, t.src_stride_h, t.src_stride_s = (n * s for s in src.stride()[:3])
        t.dst_stride_b, t.dst_stride_h, t.dst_stride_s = (n * s for s in dst.stride()[:3])
    kernels.run_on(dev, lambda stream: kernels.check(kernels.load().bz_kv_compact(
        arr, len(tensors), index.data_ptr(), lens.data_ptr(), B, NKV, cap, index.size(2), ctypes.c_void_p(stream)),
        "bz_kv_compact"))


def kv_evict(tensors, weights: torch.Tensor, seq_lens: torch.Tensor, keep: int, *, sinks: int = 0, recent: int = 0,
             kv_start: torch.Tensor | None = None, outs=None,
             weights_out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """kv_select, and the cache's tensors and weights compacted to what stays (in place unless outs / weights_out are given).
    The kept positions of row b are then the slots [0, lens[b]) of every kv head, in their old order, so later calls take
    lens for seq_lens and no kv_start. Returns (index, lens)."""
    index, lens = kv_select(weights, seq_lens, keep, sinks=sinks, recent=recent, kv_start=kv_start,
                            weights_out=weights if weights_out is None else weights_out)
    kv_compact(tensors, index, lens, outs)
    return index, lens
