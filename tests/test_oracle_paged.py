"""The oracles of the paged cache's operators against other ways to the same: torch's float8 cast, complex numbers, a softmax by hand,
transformers' scaled frequencies."""
import numpy as np
import pytest
import torch

from oracle.paged import f8_round, paged_attention, place_of, tokens_of, turn


def test_f8_round_against_torch():
    rng = np.random.default_rng(0)
    x = rng.standard_normal((50, 64)).astype(np.float32) * np.exp2(rng.integers(-120, 120, (50, 1))).astype(np.float32)
    x[3], x[4, 7], x[5, 9] = 0, np.nan, np.inf
    x[6] = [448, 449, 464, -448, 1.0625, 1.1875, 2 ** -10, 3 * 2 ** -10] * 8  # the border of a scale, and ties
    x[7] = [448, 2 ** -10, 3 * 2 ** -10, 1.0625, 1.1875, -1.3125, 0.0, -0.0] * 8
    values, codes, E = f8_round(x)
    for i in range(50):
        if not np.isfinite(x[i]).all():
            assert E[i] == 255 and np.isnan(values[i]).all() and (codes[i] == 0).all()
            continue
        s = 2.0 ** (float(E[i]) - 127)
        top = np.abs(x[i].astype(np.float64)).max()
        assert top <= 448 * s and (E[i] == 10 or top > 224 * s)
        want = torch.from_numpy((x[i].astype(np.float64) / s).astype(np.float32)).to(torch.float8_e4m3fn)
        assert np.array_equal(want.view(torch.uint8).numpy(), codes[i])
        assert np.array_equal(want.double().numpy() * s, values[i])


@pytest.mark.parametrize("interleaved", [False, True])
def test_turn_by_hand(interleaved):
    x = np.random.default_rng(1).standard_normal((3, 2, 8))
    f, pos = np.array([1.0, 0.1]), [0, 3, 70000]
    y = turn(x, pos, f, 1.5, interleaved)
    for n in range(3):
        for i in range(2):
            a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + 2)
            c, s = np.cos(pos[n] * f[i]), np.sin(pos[n] * f[i])
            assert np.allclose(y[n, :, a], 1.5 * (x[n, :, a] * c - x[n, :, b] * s))
            assert np.allclose(y[n, :, b], 1.5 * (x[n, :, b] * c + x[n, :, a] * s))
    assert np.array_equal(y[..., 4:], x[..., 4:])
    assert np.allclose(turn(y, pos, f, 1.5, interleaved, inverse=True), x)


def test_paged_attention_by_hand():
    rng = np.random.default_rng(2)
    k, v = rng.standard_normal((2, 5, 1, 16, 64))
    q = rng.standard_normal((4, 2, 64))
    table, lens, q_start = [[4, 1, -1], [2, 9, 0]], [20, 40], [0, 1, 3]
    out, _, _ = paged_attention(q, k, v, table, lens, q_start, 0.2)
    assert tokens_of(lens, q_start) == {0: (0, 19), 1: (1, 38), 2: (1, 39)}
    assert place_of(table, 16, 5, 0, 19) == (1, 3) and place_of(table, 16, 5, 1, 16) is None
    assert place_of(table, 16, 5, 0, 40) is None and place_of(table, 16, 5, 0, 48) is None and place_of(table, 16, 5, 0, -1) is None
    for n, (b, p) in tokens_of(lens, q_start).items():
        at = [x for x in (place_of(table, 16, 5, b, i) for i in range(p + 1)) if x is not None]
        for h in range(2):
            w = np.array([np.exp(0.2 * (q[n, h] @ k[pg, 0, pl])) for pg, pl in at])
            assert np.allclose(out[n, h], sum(a * v[pg, 0, pl] for a, (pg, pl) in zip(w / w.sum(), at)))
    assert (out[3] == 0).all()


class _Config:  # what transformers' frequency functions ask of a model's configuration
    def __init__(self, dim, base, scaling):
        self.rope_theta, self.head_dim, self.hidden_size, self.num_attention_heads = base, dim, dim * 4, 4
        self.partial_rotary_factor, self.max_position_embeddings = 1.0, 4096
        self.rope_scaling = self.rope_parameters = dict(scaling, rope_theta=base)

    def standardize_rope_params(self):
        pass


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("kind,factor", [("linear", 4.0), ("yarn", 8.0), ("yarn", 1.0)])
def test_frequencies_against_transformers(pkg, dim, kind, factor):
    functions = pytest.importorskip("transformers.modeling_rope_utils").ROPE_INIT_FUNCTIONS
    scaling = dict(rope_type=kind, factor=factor)
    if kind == "yarn":
        scaling["original_max_position_embeddings"] = 4096
    f, scale = functions[kind](_Config(dim, 1e6, scaling), "cpu")
    ours = pkg.rope_frequencies(dim, 1e6, "cpu", scaling=kind, factor=factor, trained=4096)
    assert torch.allclose(ours.inv_freq.float(), f.float(), rtol=1e-5) and abs(ours.factor - scale) < 1e-6


def test_frequencies(pkg):
    f = pkg.rope_frequencies(64, 10000.0, "cpu").inv_freq
    assert f.dtype == torch.float64 and torch.allclose(f, 10000.0 ** (-torch.arange(32, dtype=torch.float64) / 32))
    g = pkg.rope_frequencies(64, 10000.0, "cpu", scaling="ntk", factor=4.0).inv_freq
    assert g[0] == f[0] and abs(g[-1] / f[-1] - 0.25) < 1e-12
    y = pkg.rope_frequencies(64, 10000.0, "cpu", scaling="yarn", factor=4.0, trained=8192, interleaved=True)
    assert y.interleaved and y.inv_freq[0] == f[0] and abs(y.inv_freq[-1] / f[-1] - 0.25) < 1e-12
    for bad in (dict(rotary_dim=24), dict(base=1.0), dict(base=float("inf")), dict(scaling="other"), dict(factor=2.0),
                dict(scaling="linear", factor=0.5), dict(scaling="yarn", factor=2.0), dict(rotary_dim=0)):
        with pytest.raises(RuntimeError):
            pkg.rope_frequencies(**{**dict(rotary_dim=64, base=10000.0, device="cpu"), **bad})
