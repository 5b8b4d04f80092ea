"""More of rotary positions without a GPU: numbers near the ends of their ranges, frequencies in turns."""
from __future__ import annotations

import math
import random
from fractions import Fraction

import pytest

torch = pytest.importorskip("torch")

from jacq_amd import rotary  # noqa: E402
from jacq_amd.kivi import KiviCheckError  # noqa: E402
from jacq_amd.rotary import Rotary, Scaling  # noqa: E402


@pytest.mark.parametrize("amplitude", [1e39, -1e39])
def test_amplitudes_beyond_fp32_are_refused(amplitude):
    with pytest.raises(KiviCheckError, match="amplitude"):
        Rotary(64, amplitude=amplitude)
    with pytest.raises(KiviCheckError, match="amplitude"):
        Rotary(64, scaling=Scaling("turns", 8.0, amplitude=abs(amplitude)))
    assert Rotary(64, amplitude=torch.finfo(torch.float32).max).amplitude > 3e38


@pytest.mark.parametrize("dim,base,factor", [(4, 10000.0, 1e200), (64, 1e300, 1e100)])
def test_a_base_that_its_scaling_takes_beyond_a_double_is_refused(dim, base, factor):
    with pytest.raises(KiviCheckError, match="base"):
        Rotary(dim, base=base, scaling=Scaling("base", factor))


@pytest.mark.parametrize("seed", range(4))
def test_turns_are_those_of_exact_fractions(seed):
    """A frequency in 2^-64 turns, rounded to the nearest, ties to even, modulo a turn."""
    rng = random.Random(seed)
    two_pi = 2 * (Fraction(3.141592653589793) + Fraction(1.2246467991473532e-16))
    values = [0.0, 1.0, -1.0, 5e-324, -5e-324, 2 * math.pi, 1e300, -1e300, 2.0 ** -62, float(two_pi) / 2 ** 65]
    values += [rng.choice((-1, 1)) * 10.0 ** rng.uniform(-25, 25) for _ in range(200)]
    for f in values:
        assert rotary._turns(f) == round(Fraction(f) / two_pi * 2 ** 64) % 2 ** 64, f


def test_making_a_rotary_takes_no_fractions(monkeypatch):
    """They took 1.3 ms for 128 pairs."""
    def refuse(*_):
        raise AssertionError("a fraction")
    monkeypatch.setattr(Fraction, "__truediv__", refuse)
    monkeypatch.setattr(Fraction, "__mul__", refuse)
    assert len(Rotary(256).speeds) == 128
