"""The long-cache oracles against brute force and by their definitions (CPU)."""
import numpy as np
import pytest

from oracle.attention import decode_attention
from oracle.long_cache import F4, attended, kv4_round, select, window_attention


@pytest.mark.parametrize("start,end,T,window,sinks,want", [
    (0, 5, 1, 0, 0, [[0, 1, 2, 3, 4]]), (0, 5, 1, 2, 0, [[3, 4]]), (0, 5, 1, 2, 1, [[0, 3, 4]]),
    (2, 6, 2, 2, 1, [[2, 3, 4], [2, 4, 5]]), (0, 0, 1, 3, 2, [[]]), (3, 4, 3, 5, 1, [[], [], [3]]),
    (0, 3, 1, 9, 9, [[0, 1, 2]]),
])
def test_attended(start, end, T, window, sinks, want):
    assert attended(start, end, T, window, sinks) == want


def test_no_window_is_decode_attention():
    rng = np.random.default_rng(0)
    q, k, v = rng.standard_normal((2, 4, 1, 64)), rng.standard_normal((2, 2, 40, 64)), rng.standard_normal((2, 2, 40, 64))
    lens, start = [40, 17], [0, 3]
    out, _, _ = window_attention(q, k, v, lens, 0.125, kv_start=start)
    ref = decode_attention(q[:, :, 0].astype(np.float32), k.astype(np.float32), v.astype(np.float32), np.array(lens), 0.125,
                           kv_start=np.array(start))
    assert np.allclose(out[:, 0], ref, atol=1e-5)


def test_kv4_round_is_nearest_under_the_smallest_scale():
    rng = np.random.default_rng(1)
    x = rng.standard_normal((50, 64)) * np.exp2(rng.integers(-60, 60, (50, 1)))
    x[0] = 0
    values, codes, E = kv4_round(x)
    s = np.repeat(2.0 ** (E - 127.0), 32, -1)
    top = np.abs(x.reshape(50, 2, 32)).max(-1)
    assert (top <= 7 * 2.0 ** (E - 127.0)).all() and (E >= 1).all()
    assert ((E == 1) | (top > 7 * 2.0 ** (E - 128.0))).all()
    grid = np.concatenate([-F4[::-1], F4])
    assert np.array_equal(np.abs(values - x), np.abs(grid * s[..., None] - x[..., None]).min(-1))
    nib = np.stack([codes & 15, codes >> 4], -1).reshape(50, 64)
    assert np.array_equal(np.where(nib >= 8, -1, 1) * F4[nib & 7] * s, values)
    assert (E[0] == 1).all() and (values[0] == 0).all()
    ties = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.9] + [0.0] * 24)
    assert np.array_equal(kv4_round(ties)[0][:8], [0, 1, 1, 2, 2, 4, 4, 6])
    bad = np.ones((1, 64))
    bad[0, 40] = np.inf
    v, c, e = kv4_round(bad)
    assert np.isnan(v[0, 32:]).all() and np.isfinite(v[0, :32]).all() and e[0, 1] == 255 and (c[0, 16:] == 0).all()


def test_select():
    w = np.array([[[5, 1, 3, 3, np.nan, 3, 0, 9]]], np.float32)
    index, kept, moved = select(w, [8], 5, sinks=1, recent=1)
    assert index.tolist() == [[[0, 2, 3, 4, 7]]] and kept.tolist() == [5]
    assert np.array_equal(moved[0, 0], np.array([5, 3, 3, np.nan, 9, 0, 0, 0], np.float32), equal_nan=True)
    index, kept, _ = select(w, [4], 5, kv_start=[1])
    assert index.tolist() == [[[1, 2, 3, -1, -1]]] and kept.tolist() == [3]
