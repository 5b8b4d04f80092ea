"""What outputs of the int4 cache's attention may be off by, without the slack that
tests/kivi_attend_ref.py leaves long sequences."""
from __future__ import annotations

import torch

from tests import kivi_attend_ref as ref
from tests.q8_ref import HALF_STEP


def tight_tolerance(r, hd, dtype):
    """Of an output against ref.held_values.

    A weight 2^(t - m) is rounded to fp16: by half a step, 2^-11 of it, or below 2^-14 by 2^-25.  m is at
    least 7 below a row's largest t, in every wavefront and slice, so the weights' sum is at least 2^7, and
    the n roundings below 2^-14 are at most n 2^-25 / 2^7 of the largest |v|.  Those of the fp32 sums:
    products are exact, a step of the matrix cores adds 16 of them or more to a sum, so there are n / 16
    steps, 16 additions within one, at most 64 where wavefronts and slices are joined, and one more each
    time that m moves (by 8 at least, over a range of 2 size log2(e)), each off by at most a last place,
    2^-23; a lane's sum of weights has n / 2 additions at most, by half of one.  Then the scores' error, and
    the output's own rounding (below fp16's normal numbers 2^-25)."""
    n, half, own = r["n"], HALF_STEP[torch.float16], HALF_STEP[dtype]
    moves = 2 * 1.4427 * r["size"][..., None] / 8 + 1
    sums = (n / 16 + 16 + 64 + moves) * 2.0 ** -23
    weights = (n / 2 + 64 + moves) * 2.0 ** -24
    return (own * r["o"].abs() + (half + sums + ref.score_error(r, hd)[..., None]) * r["abs"] * (1 + own)
            + weights * r["o"].abs() + n * 2.0 ** -32 * r["vmax"] + 2.0 ** -25)
