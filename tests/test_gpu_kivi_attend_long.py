"""Long sequences through both kernels of the int4 cache's attention, under a tolerance that sees one token's
mistake."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from tests import kivi_attend_ref as ref  # noqa: E402
from tests.kivi_attend_bounds import tight_tolerance  # noqa: E402
from tests.test_gpu_kivi_attend import ints, kivi  # noqa: E402,F401
from tests.test_gpu_kivi_attend_edges import SIZES, call  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("page", [16, 32])
@pytest.mark.parametrize("heads,m,prompt", SIZES)
def test_every_token_counts(kivi, heads, m, prompt, page):  # noqa: F811
    nh, nkv, hd = heads
    lens = [20000, 700, 9000, 40]
    cache, tables, seq, q, cu, most = call(kivi, *heads, page, lens, m, prompt, seed=21, residual=128)
    for dtype, out in ((torch.float16, torch.float16), (torch.float16, torch.float32),
                       (torch.bfloat16, torch.float32)):
        x = q.to(dtype)
        for causal, window, sinks in ((True, None, 0), (True, 5000, 100), (False, None, 0)):
            o = torch.empty(q.shape, dtype=out, device="cuda")
            if causal:
                cache.prefill(x, ints(*cu), most, seq, tables, window=window, sinks=sinks, out=o)
            else:
                cache.cross(x, ints(*cu), most, seq, tables, out=o)
            for b, n in enumerate(lens):
                rows = slice(cu[b] + (max(0, m - n) if causal else 0), cu[b + 1])
                r = ref.attend(x[rows], *ref.held_values(cache, tables, b, n), window, sinks, causal)
                ref.assert_within(o[rows], r["o"], tight_tolerance(r, hd, out),
                                  f"sequence {b} of {n}, {dtype} to {out}, causal {causal}, window {window}")
