"""The tolerance of tests/kivi_attend_bounds.py sees one token's mistake in a long sequence, on the CPU: the
mistake is made in the definition."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from tests import kivi_attend_ref as ref  # noqa: E402
from tests.kivi_attend_bounds import tight_tolerance  # noqa: E402


@pytest.mark.parametrize("at,by", [(10000, 10001), (77, 5000), (19960, 19959)])
def test_another_tokens_value_is_beyond_it(at, by):
    gen = torch.Generator().manual_seed(0)
    nh, nkv, hd, m, n = 32, 2, 128, 21, 20000
    k, v = torch.randn((2, nkv, n, hd), generator=gen, dtype=torch.float64)
    k[..., 3] *= 5
    q = torch.randn((m, nh, hd), generator=gen, dtype=torch.float64)
    r = ref.attend(q, k, v)
    wrong = v.clone()
    wrong[:, at] = v[:, by]
    off = (ref.attend(q, k, wrong)["o"] - r["o"]).abs()
    assert bool((off > tight_tolerance(r, hd, torch.float16)).any())
