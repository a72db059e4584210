"""Rotary positions, as `PagedCache.append` turns queries and keys by them: pair j of
the first `rotary_dim` dims of a head is turned by position * frequency[j], and
multiplied by an amplitude.  Pairs are dims j and j + rotary_dim / 2 or, interleaved,
2j and 2j + 1.  Frequencies are base^(-2j / rotary_dim), changed for contexts longer
than a model was trained on by the usual methods, under the names that transformers'
configurations give them.  No counterpart in the reference, whose models turn their
own queries and keys.
"""
from __future__ import annotations

import math

import torch

SCALINGS = {"default": set(), "linear": {"factor"},
            "llama3": {"factor", "low_freq_factor", "high_freq_factor", "original_max_position_embeddings"},
            "yarn": {"factor", "original_max_position_embeddings"}}
OPTIONAL = {"yarn": {"attention_factor", "beta_fast", "beta_slow"}}


def _check(cond, what):
    if not cond:
        raise ValueError(what)


class Rotary:
    """`scaling` is None or a dict of a "rope_type" and its numbers:

    linear   every frequency divided by factor;
    llama3   frequencies of fewer than low_freq_factor turns within
             original_max_position_embeddings divided by factor, of more than
             high_freq_factor kept, between them blended;
    yarn     the pairs between those that make beta_slow (1) and beta_fast (32)
             turns blended from divided to kept, and the turned dims multiplied by
             attention_factor (0.1 ln(factor) + 1).

    Positions may be as large as they come: an angle is computed modulo a turn in
    64-bit integers.  `frequencies` (a float64 tensor on the host) and `amplitude` say
    what they came to."""

    def __init__(self, head_dim, *, base=10000.0, rotary_dim=None, interleaved=False, scaling=None, device="cuda"):
        self.head_dim = int(head_dim)
        self.rotary_dim = self.head_dim if rotary_dim is None else int(rotary_dim)
        _check(16 <= self.rotary_dim <= self.head_dim and self.rotary_dim % 16 == 0,
               "rotary_dim must be a multiple of 16, up to head_dim")
        base = float(base)
        _check(base > 0 and math.isfinite(base), "a positive base required")
        self.base, self.interleaved = base, bool(interleaved)
        pairs = range(self.rotary_dim // 2)
        try:
            frequencies, self.amplitude = _scaled([base ** (-2.0 * j / self.rotary_dim) for j in pairs], scaling, base,
                                                  self.rotary_dim)
        except OverflowError:
            raise ValueError("a base and scaling of which float64 holds the numbers required") from None
        _check(all(math.isfinite(f) for f in frequencies), "frequencies that are finite required")
        _check(math.isfinite(self.amplitude) and abs(self.amplitude) <= torch.finfo(torch.float32).max,
               "an attention factor that is finite in float32 required")
        self.frequencies = torch.tensor(frequencies, dtype=torch.float64, device="cpu")
        # the part of a turn at position 1, in units of 2^-64 (as the bits of an int64)
        turns = [round(math.fmod(f / (2 * math.pi), 1.0) * 2.0 ** 64) % 2 ** 64 for f in frequencies]
        self.turns = torch.tensor([t - 2 ** 64 if t >= 2 ** 63 else t for t in turns], dtype=torch.int64,
                                  device=torch.device(device))
        self.device = self.turns.device


def _scaled(freq, scaling, base, dim):
    """The frequencies and the amplitude under a scaling."""
    if scaling is None:
        return freq, 1.0
    kind = scaling.get("rope_type", "default")
    _check(kind in SCALINGS, f"rope_type must be one of {sorted(SCALINGS)}")
    given = set(scaling) - {"rope_type"}
    _check(SCALINGS[kind] <= given, f"{kind} scaling needs {sorted(SCALINGS[kind] - given)}")
    unknown = given - SCALINGS[kind] - OPTIONAL.get(kind, set())
    _check(not unknown, f"{kind} scaling does not know {sorted(unknown)}")
    if kind == "default":
        return freq, 1.0
    factor = float(scaling["factor"])
    _check(factor > 0 and math.isfinite(factor), "a positive factor required")
    if kind == "linear":
        return [f / factor for f in freq], 1.0
    original = float(scaling["original_max_position_embeddings"])
    _check(original > 0, "a positive original_max_position_embeddings required")
    if kind == "llama3":
        low, high = float(scaling["low_freq_factor"]), float(scaling["high_freq_factor"])
        _check(0 < low < high, "low_freq_factor below high_freq_factor required")
        kept = [min(max((original * f / (2 * math.pi) - low) / (high - low), 0.0), 1.0) for f in freq]
        return [f * (x + (1 - x) / factor) for f, x in zip(freq, kept)], 1.0
    fast, slow = float(scaling.get("beta_fast") or 32), float(scaling.get("beta_slow") or 1)
    _check(0 < slow <= fast and base > 1, "beta_slow up to beta_fast, and a base above 1, required")

    def pair_of(turns):
        return dim * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))

    first, last = max(math.floor(pair_of(fast)), 0), min(math.ceil(pair_of(slow)), dim - 1)
    kept = [1 - min(max((j - first) / max(last - first, 0.001), 0.0), 1.0) for j in range(dim // 2)]
    amplitude = scaling.get("attention_factor")
    amplitude = (0.1 * math.log(factor) + 1 if factor > 1 else 1.0) if amplitude is None else float(amplitude)
    return [f * (x + (1 - x) / factor) for f, x in zip(freq, kept)], amplitude
