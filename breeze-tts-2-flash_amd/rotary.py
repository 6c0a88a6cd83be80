"""Rotary positions: the frequencies of a model's heads (rope_frequencies) and turning heads by them (rope). The paged cache's
rope_store turns a step's q and k by the same on their way into the cache.

The reference turns whole heads of 128 dims, pairs of dims i and i + 64, inside its one-token prologue (flash/csrc/bb_attn.cu:78-100), by
cos and sin in bf16. Here a token carries its position, whatever the number of tokens, and angles are worked out from it in 64 bits.
"""
from __future__ import annotations

import math
from typing import NamedTuple

import torch

from . import kernels
from .attention import _check


class Rope(NamedTuple):
    """A rotation: pair i of the first 2 len(inv_freq) dims of a head is turned by position * inv_freq[i] (float64, on the tokens'
    device; their number a multiple of 8) and multiplied by factor. Pairs are dims i and i + len(inv_freq), or, interleaved, 2 i and
    2 i + 1; the dims behind them stay."""
    inv_freq: torch.Tensor
    factor: float = 1.0
    interleaved: bool = False


def rope_frequencies(rotary_dim: int, base: float, device, *, interleaved: bool = False, scaling: str | None = None,
                     factor: float = 1.0, trained: int = 0, beta_fast: float = 32.0, beta_slow: float = 1.0) -> Rope:
    """The rotation with inv_freq[i] = base^(-2 i / rotary_dim), stretched for contexts `factor` times as long as the model was
    trained for (factor >= 1):

      None      as trained
      "linear"  every angle divided by factor (positions interpolated)
      "ntk"     base times factor^(R / (R - 2)), R = rotary_dim: the lowest frequency is divided by factor, the highest kept
      "yarn"    pairs that turn at least beta_fast times within the `trained` positions kept, those that turn at most beta_slow
                times interpolated, between them (by pair number, from the floor of one bound to the ceiling of the other, within
                0 and R - 1) a mixture; cos and sin times 0.1 ln(factor) + 1 (Peng et al. 2023, sections 3.2 to 3.4)

    rotary_dim: a multiple of 16 up to the head's dims."""
    _check(rotary_dim > 0 and rotary_dim % 16 == 0, f"rotary_dim must be a positive multiple of 16, got {rotary_dim}")
    _check(math.isfinite(base) and base > 1, f"base must be finite and over 1, got {base}")
    _check(scaling in (None, "linear", "ntk", "yarn"), f"scaling must be None, 'linear', 'ntk' or 'yarn', got {scaling!r}")
    _check(math.isfinite(factor) and factor >= 1, f"factor must be finite and at least 1, got {factor}")
    _check(scaling is not None or factor == 1, "a factor other than 1 needs scaling=")
    if scaling == "ntk":
        base *= factor ** (rotary_dim / (rotary_dim - 2))
    f = base ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim)
    scale = 1.0
    if scaling == "linear":
        f = f / factor
    elif scaling == "yarn":
        _check(trained > 0, "yarn needs trained=, the positions the model was trained for")
        _check(beta_fast >= beta_slow > 0, "beta_fast must be at least beta_slow, and that over 0")
        # pair i turns trained / (2 pi) base^(-2 i / R) times within the trained positions: beta times at this i
        at = [rotary_dim * math.log(trained / (2 * math.pi * beta)) / (2 * math.log(base)) for beta in (beta_fast, beta_slow)]
        low, high = max(math.floor(at[0]), 0), min(math.ceil(at[1]), rotary_dim - 1)
        mix = ((torch.arange(rotary_dim // 2, dtype=torch.float64) - low) / max(high - low, 1e-3)).clamp(0, 1)
        if at[1] <= 0:  # not even pair 0 turns more than beta_slow times
            mix = torch.ones_like(f)
        f = f * (1 - mix) + f / factor * mix
        scale = 0.1 * math.log(factor) + 1
    return Rope(f.to(device), scale, interleaved)


def _flag(x, name: str) -> bool:
    """A flag of a traced call, refused where the binding refuses it."""
    _check(isinstance(x, (bool, int)) and x in (0, 1), f"{name} must be a bool")
    return bool(x)


def rope(x: torch.Tensor, positions: torch.Tensor, freqs: Rope, out: torch.Tensor | None = None, *,
         inverse: bool = False) -> torch.Tensor:
    """x turned by its tokens' positions (bz_rope_apply). x: bf16 [tokens, heads, head_dim], head_dim 64 or 128, any strides that are
    multiples of 8 (q and k as views of a projection's output); positions: int32 or int64 [tokens]. out may be x itself. inverse
    turns back: rope(rope(x, p, f), p, f, inverse=True) is x but for two roundings, and keys move from position p to p' by
    inverse and again. Angles are worked out and reduced to within half a turn in 64 bits (off by at most 2^-30 turns for positions up to 2^22), and
    rounded to 32 there (2^-26). Returns out."""
    if torch.compiler.is_compiling():
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device) if out is None else out
        torch.ops.bz.rope(x, positions, freqs[0], float(freqs[1]), _flag(freqs[2], "interleaved"), _flag(inverse, "inverse"), out)
        return out
    return kernels.eager().rope(x, positions, freqs[0], freqs[1], freqs[2], inverse, out)
