"""Inverse frequencies and their forms for long contexts, from their definitions, on the host."""

from __future__ import annotations

import importlib
import math

import pytest
import torch


@pytest.fixture(scope="module")
def freq(built):
    return importlib.import_module("mi50_vllm_lab_b200.positions").inverse_frequencies


def exact(rot, base):
    return [base ** (-2.0 * i / rot) for i in range(rot // 2)]


def close(got, want):
    """One rounding to fp32 of an fp64 value whose own few roundings are 2^-50 of it."""
    want = torch.tensor(want, dtype=torch.float64)
    assert got.dtype == torch.float32
    assert bool(((got.double() - want).abs() <= 2.0 ** -24 * (1 + 1e-6) * want).all())


@pytest.mark.parametrize("rot,base", [(2, 10000.0), (64, 1e6), (128, 5e5), (80, 10000.0)])
def test_plain_and_linear(freq, rot, base):
    f, s = freq(rot, base)
    close(f, exact(rot, base))
    assert s == 1.0
    f, s = freq(rot, base, "linear", factor=4.0)
    close(f, [x / 4 for x in exact(rot, base)])
    assert s == 1.0


def test_ntk_keeps_the_first_pair_and_divides_the_last(freq):
    f, s = freq(64, 1e4, "ntk", factor=8.0)
    e = exact(64, 1e4)
    close(f[:1], e[:1])
    close(f[-1:], [e[-1] / 8])
    assert s == 1.0 and bool((f[1:] < f[:-1]).all())


def test_yarn(freq):
    rot, base, n, factor = 128, 1e6, 32768, 4.0
    f, s = freq(rot, base, "yarn", factor=factor, original_length=n)
    e = exact(rot, base)
    assert s == 0.1 * math.log(4.0) + 1.0
    turns = [n * x / (2 * math.pi) for x in e]
    first = max(i for i in range(rot // 2) if turns[i] >= 32)  # the last pair that turns enough
    last = min(i for i in range(rot // 2) if turns[i] <= 1)
    ramp = [min(max((i - first) / (last - first), 0.0), 1.0) for i in range(rot // 2)]
    close(f, [x * (1 - r) + x / factor * r for x, r in zip(e, ramp)])
    assert freq(rot, base, "yarn", factor=1.0)[1] == 1.0


def test_wavelength(freq):
    rot, base, n, factor = 128, 5e5, 8192, 8.0
    f, s = freq(rot, base, "wavelength", factor=factor, original_length=n, low_turns=1.0,
                high_turns=4.0)
    want = []
    for x in exact(rot, base):
        turns = n * x / (2 * math.pi)
        mix = (turns - 1.0) / 3.0
        want.append(x if turns >= 4 else x / factor if turns <= 1 else (1 - mix) * x / factor + mix * x)
    close(f, want)
    assert s == 1.0


@pytest.mark.parametrize("kw", [dict(rot=0), dict(rot=3), dict(base=1.0), dict(kind="other"),
                                dict(factor=0.0), dict(kind="ntk", rot=2),
                                dict(kind="wavelength", low_turns=4.0, high_turns=4.0)])
def test_refusals(freq, kw):
    with pytest.raises(ValueError):
        freq(**{"rot": 64, **kw})
