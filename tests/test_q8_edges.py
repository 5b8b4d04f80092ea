"""Edges of the 8-bit cache's host side, without a GPU."""
from __future__ import annotations

import copy
import pickle

import pytest

torch = pytest.importorskip("torch")

from jacq_amd import kivi, q8  # noqa: E402,F401
from tests.test_q8 import EINVAL, GOOD, Record, error  # noqa: E402


def test_a_call_of_no_queries_with_weights_is_checked():
    for kw in (dict(total_q=0), dict(max_q=0)):
        error(Record().attend(WEIGHTS=0x60000, SEQ_LENS=0, **kw), EINVAL, "null")
        error(Record().attend(WEIGHTS=0x60002, Q=0, O=0, **kw), EINVAL, "4-byte")
        assert Record().attend(Q=0, O=0, SEQ_LENS=0, **kw) == 0


@pytest.fixture
def cache():
    return q8.PagedQ8Cache(q8.Q8Geometry(**GOOD), 3, device="cpu")


def held(c):
    """The addresses that a call of this cache passes."""
    return tuple(getattr(c._record, n) for n in q8.POOL)


def test_calls_take_the_tensors_that_a_cache_holds_now(cache):
    for name in q8.POOL:
        new = getattr(cache, name).clone()
        setattr(cache, name, new)
        assert getattr(cache, name) is new
        assert held(cache) == tuple(t.data_ptr() for t in cache.pool())
        for bad in (new[:, :1], new.to(torch.float64)):
            with pytest.raises(kivi.KiviCheckError, match=name):
                setattr(cache, name, bad)
        assert getattr(cache, name) is new  # as it was
        assert held(cache) == tuple(t.data_ptr() for t in cache.pool())
    with pytest.raises(kivi.KiviCheckError, match="k_code"):
        cache.geo = q8.Q8Geometry(**{**GOOD, "num_pages": 17})
    cache.geo = q8.Q8Geometry(**{**GOOD, "max_pages_per_seq": 9})
    assert cache._table_shape == (3, 9)


def test_copies_and_pickles_hold_tensors_of_their_own(cache):
    cache.k_code.random_(0, 255)
    for make, shared in ((copy.copy, True), (copy.deepcopy, False),
                         (lambda c: pickle.loads(pickle.dumps(c)), False)):
        other = make(cache)
        assert other.geo == cache.geo and other.batch == 3
        assert all(torch.equal(a, b) for a, b in zip(other.pool(), cache.pool()))
        assert held(other) == tuple(t.data_ptr() for t in other.pool())
        assert (held(other) == held(cache)) == shared
    view = copy.deepcopy(cache.sequence_view(1))
    assert view.batch == 1 and held(view)[0] != held(cache)[0]


def test_a_view_of_no_sequence_is_refused(cache):
    for b in (-1, 3, 1 << 40):
        with pytest.raises(kivi.KiviCheckError, match="sequence must be in"):
            cache.sequence_view(b)
    t = dict(zip(q8.POOL, cache.pool()))
    with pytest.raises(kivi.KiviCheckError, match="batch"):
        q8.PagedQ8Cache.from_tensors(cache.geo, {**t, "k_tail": t["k_tail"][:0],
                                                 "v_tail": t["v_tail"][:0]})


def workspace(batch, total, max_q, weighted=0, **geo):
    g = q8.Q8Geometry(**{**dict(num_heads=40, num_kv_heads=8, head_dim=128, page_size=32,
                                max_pages_per_seq=512, num_pages=512), **geo})
    return q8.lib().jacq_q8_attend_workspace_size(g.ref, batch, total, max_q, weighted)


@pytest.mark.parametrize("heads", [(40, 8, 128), (14, 2, 64)])
def test_a_call_is_planned_by_its_queries_not_by_the_caches_sequences(heads):
    geo = dict(zip(("num_heads", "num_kv_heads", "head_dim"), heads))
    # queries of one sequence: as many slices of its tokens in a cache of one sequence and of many
    for queries in (200, 512, 2000):
        alone = workspace(1, queries, queries, **geo)
        assert alone > 0
        for batch in (2, 64, 1000):
            assert workspace(batch, queries, queries, **geo) == alone
    # so few that the decode's kernel has them alone, whose workspace is the smaller by what block
    # weights take: their sums of 1024 groups of 16 tokens and rows, and the rows' own
    queries = 20
    g = heads[0] // heads[1]
    blocks = -(-queries * g // 32)
    for batch in (1, 64):
        sums = batch * heads[1] * blocks * 1024 * 32 * 4
        rows = -(-queries * heads[0] * 4 // 256) * 256
        assert (workspace(batch, queries, queries, 1, **geo)
                - workspace(batch, queries, queries, **geo)) == sums + rows


def test_more_row_tiles_than_a_launch_has_are_refused():
    r = Record(max_pages_per_seq=4)
    error(r.attend(batch=100, total_q=2 ** 31 - 1, max_q=100), EINVAL, "too many query rows")
