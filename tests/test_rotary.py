"""Frequencies of rotary.rope_frequencies against their definitions, at the ends of their ranges."""
import math

import pytest
import torch


@pytest.mark.parametrize("dim,base,trained,fast,slow", [
    (64, 1e4, 6, 32.0, 1.0), (64, 1e4, 1, 32.0, 1.0), (128, 1e6, 4096, 2000.0, 652.0), (128, 1e6, 4096, 2000.0, 651.0),
    (64, 10.0, 1 << 24, 32.0, 1.0), (64, 1e4, 4096, 4.0, 4.0), (128, 1e6, 32768, 32.0, 1.0), (16, 1e4, 100, 1.0, 0.001)])
def test_yarn_keeps_and_interpolates_by_turns(pkg, dim, base, trained, fast, slow):
    """Pairs that turn at least beta_fast times within the trained positions keep their frequency, those that turn at most beta_slow times
    have it divided by factor, and between them it falls from the one to the other."""
    plain = pkg.rope_frequencies(dim, base, "cpu").inv_freq
    f = pkg.rope_frequencies(dim, base, "cpu", scaling="yarn", factor=8.0, trained=trained, beta_fast=fast, beta_slow=slow)
    part = (plain / f.inv_freq - 1) / 7  # 0: kept, 1: divided
    turns = trained * plain / (2 * math.pi)
    assert (part[turns >= fast] < 1e-12).all()
    assert (part[turns <= slow] > 1 - 1e-12).all()
    assert (part.diff() > -1e-12).all() and (part > -1e-12).all() and (part < 1 + 1e-12).all()
