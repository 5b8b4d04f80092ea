"""More refusals of rotary positions, without a GPU: numbers near the ends of their ranges."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

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
