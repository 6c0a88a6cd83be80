"""Oracles of the paged cache's operators (include/bz_paged_cache.h) in float64: rotary positions, the 8-bit rounding of a head vector, where
a batch's tokens belong, and causal attention over pages."""
import numpy as np

from oracle.long_cache import attention_bound  # noqa: F401  (the tests' tolerance)


def turn(x, positions, inv_freq, factor=1.0, interleaved=False, inverse=False):
    """x [N, H, D] with pair i of its first 2 len(inv_freq) dims multiplied by factor e^(i position inv_freq[i])."""
    x, f = np.array(x, np.float64), np.asarray(inv_freq, np.float64)
    n, at = len(f), np.arange(len(f))
    a, b = (2 * at, 2 * at + 1) if interleaved else (at, at + n)
    z = factor * np.exp(1j * np.outer(np.asarray(positions, np.float64), f))[:, None]
    y = (x[..., a] + 1j * x[..., b]) * (1 / z if inverse else z)
    x[..., a], x[..., b] = y.real, y.imag
    return x


def turn_bound(x, y, inv_freq, factor=1.0, interleaved=False):
    """How far a bf16 result may lie from y = turn(x, ..): half a step of its rounding (2^-8 of the value), and the error of cos and sin, at
    most 2^-18 each (the hardware's functions on a reduced angle of 2^-25 turns), times the pair's values."""
    x, f = np.abs(np.asarray(x, np.float64)), np.asarray(inv_freq)
    n, at = len(f), np.arange(len(f))
    a, b = (2 * at, 2 * at + 1) if interleaved else (at, at + n)
    pair = np.zeros_like(x)
    pair[..., a] = pair[..., b] = x[..., a] + x[..., b]
    return 2.0 ** -8 * np.abs(y) + 2.0 ** -17 * abs(factor) * pair + 1e-38


def norm(x, w, eps):
    """x [.., D] normed over its last dim, times w."""
    x = np.asarray(x, np.float64)
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.asarray(w, np.float64)


# the e4m3 values of codes 0 .. 126: three mantissa bits, exponents from 2^-6 on, subnormals below
_E4M3 = np.array([(m / 8 if e == 0 else 1 + m / 8) * 2.0 ** (max(e, 1) - 7) for e in range(16) for m in range(8)])[:127]


def f8_round(x):
    """(values, codes, scale bytes) of x [..., D]: every vector under the smallest 2^(E - 127), E >= 10, with max |x| <= 448 times it, each
    value at the nearest e4m3 value times it, ties to the even code; a vector with NaN or an infinity is all NaN, code 0, E 255."""
    b = np.asarray(x, np.float64)
    bad = ~np.isfinite(b).all(-1)
    b = np.where(bad[..., None], 0.0, b)
    top = np.abs(b).max(-1)
    E = np.full(top.shape, 10, np.int64)
    while (grow := top > 448 * 2.0 ** (E - 127.0)).any():
        E += grow
    a = np.abs(b) / 2.0 ** (E - 127.0)[..., None]
    hi = np.clip(np.searchsorted(_E4M3, a), 1, 126)
    lo = hi - 1
    dl, dh = a - _E4M3[lo], _E4M3[hi] - a
    code = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    values = np.copysign(_E4M3[code], b) * 2.0 ** (E - 127.0)[..., None]
    code = code | (np.signbit(b).astype(np.int64) << 7)
    return (np.where(bad[..., None], np.nan, values), np.where(bad[..., None], 0, code).astype(np.uint8),
            np.where(bad, 255, E).astype(np.uint8))


def tokens_of(seq_lens, q_start):
    """[(row, position)] of the tokens q_start[0] .. q_start[-1] - 1, by token."""
    out = {}
    for b, n in enumerate(seq_lens):
        for t in range(q_start[b], q_start[b + 1]):
            out[t] = (b, int(n) - (q_start[b + 1] - t))
    return out


def place_of(table, page_size, pages, row, pos):
    """(page, place) of a position, None where there is none."""
    if pos < 0 or pos // page_size >= len(table[row]):
        return None
    page = int(table[row][pos // page_size])
    return (page, pos % page_size) if 0 <= page < pages else None


def paged_attention(q, k, v, table, seq_lens, q_start, scale):
    """(out, spread, reach) as window_attention's, by token: q [N, NH, D] over pages k, v [pages, NKV, page_size, D] (any float arrays).
    Tokens of no row stay zero."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    N, NH, D = q.shape
    pages, NKV, ps = k.shape[:3]
    G = NH // NKV
    out, spread, reach = np.zeros((N, NH, D)), np.zeros((N, NH, D)), np.zeros((N, NH))
    for b, n in enumerate(seq_lens):
        t0, t1 = q_start[b], q_start[b + 1]
        at = [(p, place_of(table, ps, pages, b, p)) for p in range(min(max(int(n), 0), len(table[b]) * ps))]
        pos = np.array([p for p, x in at if x is not None], np.int64)
        if t1 == t0 or len(pos) == 0:
            continue
        pg, pl = np.array([x for _, x in at if x is not None]).T
        own = int(n) - (t1 - np.arange(t0, t1))
        ok = pos[None] <= own[:, None]
        some = ok.any(1)
        for h in range(NKV):
            # what no token attends may be anything
            used = ok.any(0)
            kk, vv = (np.where(used[:, None], x[pg, h, pl], 0) for x in (k, v))
            for i in range(h * G, h * G + G):
                x = q[t0:t1, i]
                w = np.where(ok, x @ kk.T * scale, -np.inf)
                w = np.exp(w - np.where(some, w.max(1), 0)[:, None])
                w /= np.where(some, w.sum(1), 1)[:, None]
                out[t0:t1, i] = w @ vv
                spread[t0:t1, i] = w @ np.abs(vv)
                reach[t0:t1, i] = np.where(ok, np.abs(x) @ np.abs(kk).T, 0).max(1)
    return out, spread, reach
