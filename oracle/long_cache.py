"""Oracles of the long-cache operators (include/bz_long_cache.h) in float64: attention over a sliding window with sinks,
the 4-bit rounding of a block of 32 values, accumulated attention weights, and the selection of the positions that stay."""
import numpy as np

F4 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def attended(start, end, T, window, sinks):
    """For each of a row's T tokens (its last T positions) the positions it attends, ascending."""
    rows = []
    for t in range(T):
        e = max(start, end - (T - 1 - t))
        lo = max(start, e - window) if window > 0 else start
        rows.append([p for p in range(start, e) if p >= lo or p < start + sinks])
    return rows


def window_attention(q, k, v, lens, scale, window=0, sinks=0, kv_start=None):
    """(out, spread, reach): out [B, T, NH, D] of q [B, NH, T, D] over k, v [B, NKV, cap, D] (any float arrays), with the
    sums sum_p p |v| (spread, like out) and max_p sum_i |q_i k_i| (reach [B, T, NH]) that bound a rounded computation."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    B, NH, T, D = q.shape
    NKV, cap = k.shape[1], k.shape[2]
    G = NH // NKV
    out, spread, reach = np.zeros((B, T, NH, D)), np.zeros((B, T, NH, D)), np.zeros((B, T, NH))
    for b in range(B):
        e = min(max(int(lens[b]), 0), cap)
        s = min(max(int(kv_start[b]), 0), e) if kv_start is not None else 0
        for t, pos in enumerate(attended(s, e, T, window, sinks)):
            if not pos:
                continue
            for h in range(NKV):
                kk, vv = k[b, h, pos], v[b, h, pos]
                for g in range(G):
                    x = q[b, h * G + g, t]
                    w = kk @ x * scale
                    w = np.exp(w - w.max())
                    w /= w.sum()
                    out[b, t, h * G + g] = w @ vv
                    spread[b, t, h * G + g] = w @ np.abs(vv)
                    reach[b, t, h * G + g] = (np.abs(kk) @ np.abs(x)).max()
    return out, spread, reach


def attention_bound(out, spread, reach, scale, D, one_term=False):
    """How far a kernel's bf16 output may lie from out: half a bf16 step (2^-8 of the value), and the terms' own error times
    sum p |v|. A score is a sum of D products of bf16 values in fp32, D + 2 roundings of at most 2^-23 of sum |q_i k_i|
    each; it enters a term and the sum that divides it (twice), with the same again for the shift by the maximum; two bf16
    terms hold p to 2^-17, and the sums and exponentials add a few 2^-23. one_term: p is rounded to a single bf16 before it
    meets V (a chunk of many tokens), half a bf16 step of each term: 2^-8 of sum p |v| more."""
    ds = abs(scale) * reach * (D + 2) * 2.0 ** -23
    return 2.0 ** -8 * np.abs(out) + (4 * ds + 2.0 ** -15 + one_term * 2.0 ** -8)[..., None] * spread + 1e-30


def kv4_round(x):
    """(values, codes, scale bytes) of x [..., D]: every block of 32 under the smallest power of two 2^(E - 127), E >= 1, with
    max |x| <= 7 times it, every value at the nearest of F4 times it (ties to the even code, past 6 to 6); a block with
    NaN or an infinity is all NaN, code 0, E 255."""
    b = np.asarray(x, np.float64).reshape(*x.shape[:-1], -1, 32)
    bad = ~np.isfinite(b).all(-1)
    b = np.where(bad[..., None], 0.0, b)
    top = np.abs(b).max(-1)
    E = np.ones(top.shape, np.int64)
    while (grow := top > 7 * 2.0 ** (E - 127.0)).any():
        E += grow
    a = np.abs(b) / 2.0 ** (E - 127.0)[..., None]
    d = np.abs(a[..., None] - F4)
    near = d == d.min(-1, keepdims=True)
    even = near & (np.arange(8) % 2 == 0)
    pick = np.where(even.any(-1), even.argmax(-1), near.argmax(-1))
    code = pick | (np.signbit(b).astype(np.int64) << 3)
    values = np.copysign(F4[pick], b) * 2.0 ** (E - 127.0)[..., None]
    values = np.where(bad[..., None], np.nan, values).reshape(x.shape)
    E, code = np.where(bad, 255, E), np.where(bad[..., None], 0, code).reshape(x.shape)
    return values, (code[..., 0::2] | code[..., 1::2] << 4).astype(np.uint8), E.astype(np.uint8)


def select(weights, lens, keep, sinks=0, recent=0, kv_start=None):
    """(index [B, NKV, keep], kept lengths [B], the kept weights) as bz_kv_select defines them."""
    w = np.asarray(weights, np.float32)
    B, NKV, cap = w.shape
    index, kept = np.full((B, NKV, keep), -1, np.int32), np.zeros(B, np.int32)
    moved = np.array(w)
    for b in range(B):
        e = min(max(int(lens[b]), 0), cap)
        s = min(max(int(kv_start[b]), 0), e) if kv_start is not None else 0
        kept[b] = min(e - s, keep)
        for h in range(NKV):
            pos = list(range(s, e))
            if e - s > keep:
                middle = pos[sinks:len(pos) - recent]
                middle = sorted(middle, key=lambda p: (0, 0.0, p) if np.isnan(w[b, h, p]) else (1, -float(w[b, h, p]), p))
                pos = sorted(pos[:sinks] + middle[:keep - sinks - recent] + pos[len(pos) - recent:])
            index[b, h, :len(pos)] = pos
            moved[b, h, :e] = 0
            moved[b, h, :len(pos)] = w[b, h, pos]
    return index, kept, moved
