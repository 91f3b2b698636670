"""Inverse frequencies of rotary positions and their forms for long contexts, for the operators
``rope`` and ``rope_cache`` (which take any table: row at position p turns pair i by p * inv_freq[i]).

Unscaled, pair i of rot / 2 has f_i = base^(-2i / rot). With a factor s > 1 on the context:

* ``linear``: f_i / s (positions are interpolated);
* ``ntk``: base * s^(rot / (rot - 2)) in place of base: pair 0 is kept, the last one divided by s;
* ``yarn``: pairs that turn more than ``beta_fast`` times over the original length keep f_i, those
  that turn less than ``beta_slow`` times get f_i / s, linear in i between (ends rounded outwards to
  whole pairs); cosines and sines are multiplied by 0.1 ln(s) + 1 (the operators' ``scale``);
* ``wavelength``: by the number of turns over the original length, f_i / s below ``low_turns``, f_i
  above ``high_turns``, and between a mixture linear in the turns.

Formed in fp64 and rounded once to fp32.
"""

from __future__ import annotations

import math

import torch

KINDS = ("none", "linear", "ntk", "yarn", "wavelength")


def inverse_frequencies(rot: int, base: float = 10000.0, kind: str = "none", factor: float = 1.0,
                        original_length: int = 8192, beta_fast: float = 32.0,
                        beta_slow: float = 1.0, low_turns: float = 1.0, high_turns: float = 4.0,
                        device=None) -> tuple[torch.Tensor, float]:
    """(inv_freq fp32 [rot / 2], scale on cosines and sines)."""
    if rot < 2 or rot % 2 or not base > 1 or kind not in KINDS or not factor > 0:
        raise ValueError(f"rot={rot}, base={base}, kind={kind!r} of {KINDS}, factor={factor}")
    if kind == "ntk" and rot == 2:
        raise ValueError("ntk needs more than one pair")
    pair = torch.arange(rot // 2, dtype=torch.float64)
    if kind == "ntk":
        base = base * factor ** (rot / (rot - 2))
    f = base ** (-2.0 * pair / rot)
    scale = 1.0
    if kind == "linear":
        f = f / factor
    elif kind == "yarn":
        def pair_of(turns):  # the (real-valued) pair that turns so often over the original length
            return rot / 2 * math.log(original_length / (2 * math.pi * turns)) / math.log(base)

        first = max(math.floor(pair_of(beta_fast)), 0)
        last = min(math.ceil(pair_of(beta_slow)), rot - 1)
        stretched = ((pair - first) / max(last - first, 1e-3)).clamp(0, 1)
        f = f * (1 - stretched) + f / factor * stretched
        scale = 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0
    elif kind == "wavelength":
        if not high_turns > low_turns:
            raise ValueError(f"high_turns={high_turns} must be above low_turns={low_turns}")
        turns = original_length * f / (2 * math.pi)
        kept = ((turns - low_turns) / (high_turns - low_turns)).clamp(0, 1)
        f = f * kept + f / factor * (1 - kept)
    return f.float().to(device), scale
