"""Edges of the 8-bit cache's host side, without a GPU."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from jacq_amd import kivi, q8  # noqa: E402,F401
from tests.test_q8 import EINVAL, Record, error  # noqa: E402


def test_a_call_of_no_queries_with_weights_is_checked():
    for kw in (dict(total_q=0), dict(max_q=0)):
        error(Record().attend(WEIGHTS=0x60000, SEQ_LENS=0, **kw), EINVAL, "null")
        error(Record().attend(WEIGHTS=0x60002, Q=0, O=0, **kw), EINVAL, "4-byte")
        assert Record().attend(Q=0, O=0, SEQ_LENS=0, **kw) == 0
