"""Edges of the 8-bit paged cache's calls, through both attention kernels: the decode's takes few
rows or few heads, the prompts' the rest, so each size here says which one it is for."""
from __future__ import annotations

import dataclasses
import random

import pytest

torch = pytest.importorskip("torch")

from tests import q8_ref as ref  # noqa: E402
from tests.test_gpu_q8 import I32, check_attention, ints, make, q8, randn, spoil  # noqa: E402,F401

pytestmark = pytest.mark.gpu


def offsets(m):
    cu = [0]
    for x in m:
        cu.append(cu[-1] + x)
    return cu


def runs_prefill(q8, cache, total, max_q):  # noqa: F811
    """Whether a call without block weights goes to the prompts' kernel: the other one's workspace
    is as much smaller without them as what they take (under a table so wide that its calls are
    cut; the choice does not go by the table)."""
    g = dataclasses.replace(cache.geo, max_pages_per_seq=16384)
    rows = max_q * g.gqa
    block = 16 if rows <= 16 else 32
    weights = (cache.batch * g.num_kv_heads * -(-rows // block) * g.max_pages_per_seq
               * (g.page_size // 16) * min(rows, block), total * g.num_heads)
    size = [q8.lib().jacq_q8_attend_workspace_size(g.ref, cache.batch, total, max_q, w)
            for w in (0, 1)]
    return size[1] - size[0] != sum(-(-4 * n // 256) * 256 for n in weights)


@pytest.mark.parametrize("codes", ["int8", "e4m3"])
@pytest.mark.parametrize("page", [16, 32])
@pytest.mark.parametrize("heads,m,prompt", [((4, 2, 64), 40, False), ((4, 1, 128), 45, False),
                                            ((32, 8, 128), 40, True), ((14, 2, 64), 60, True)])
def test_a_page_outside_the_pool_reaches_no_query_before_it(q8, codes, page, heads, m, prompt):  # noqa: F811
    """The codes read in its place are page 0's, which may be memory that was never written."""
    nh, nkv, hd = heads
    lens = [160 + page + 3, 224 + page + 5, 200]
    cache, tables, seq = make(q8, nh, nkv, hd, page, codes, lens, seed=page + m)
    assert runs_prefill(q8, cache, 3 * m, m) == prompt
    spare = (set(range(cache.geo.num_pages)) - set(tables[tables >= 0].tolist())).pop()
    for x in (cache.k_code, cache.v_code, cache.k_scale, cache.v_scale):
        x[spare] = x[0]
    tables[tables == 0] = spare
    gen = torch.Generator("cuda").manual_seed(m)
    q = randn(gen, 3 * m, nh, hd)
    cu = offsets([m] * 3)
    clean = cache.prefill(q, ints(*cu), m, seq, tables)
    check_attention(cache, tables, lens, q, cu, clean)
    cache.k_code[0], cache.v_code[0] = 0x7F, 0xFF
    cache.k_scale[0], cache.v_scale[0] = float("inf"), float("nan")
    # pages in the midst of 64-token tiles, with queries before them in the same tile
    bad = tables.clone()
    bad[0, 160 // page], bad[1, 224 // page] = 1 << 30, -7
    got = cache.prefill(q, ints(*cu), m, seq, bad)
    for b, first in ((0, 160), (1, 224), (2, lens[2])):
        sees = torch.arange(lens[b] - m, lens[b], device="cuda") >= first
        assert b == 2 or 0 < int(sees.sum()) < m
        rows = slice(cu[b], cu[b + 1])
        assert bool(got[rows][sees].isnan().all())
        assert torch.equal(got[rows][~sees], clean[rows][~sees]), b


@pytest.mark.parametrize("heads,batch,m", [((4, 1, 64), 512, 1), ((10, 1, 128), 512, 3),
                                           ((32, 2, 64), 20, 9), ((8, 1, 128), 20, 17)])
def test_many_light_tokens_weigh_beside_a_heavy_one(q8, heads, batch, m):  # noqa: F811
    """A first token of 96 % of the weight, in a block of 32 times the others' V scale, and 65536
    tokens of 2^-20.5 of its weight each: next to the heaviest they are 2^-25.5, and 4 % together.
    As many sequences of the same pages as leave each to few wavefronts."""
    nh, nkv, hd = heads
    page, n = 32, 65536 + 32
    k = torch.zeros((n, nkv, hd), dtype=torch.float16, device="cuda")
    k[0, :, 0] = 1.0
    v = torch.ones((n, nkv, hd), dtype=torch.float16, device="cuda")
    v[:page] = 0.0
    v[0, :, 3] = 32.0
    width = n // page
    tables = torch.arange(width, **I32).repeat(batch, 1)
    cache = q8.PagedQ8Cache(q8.Q8Geometry(nh, nkv, hd, page, width, width), batch)
    cache.sequence_view(0).append(k, v, tables[:1], ints(0), cu_new=ints(0, n))
    assert runs_prefill(q8, cache, m * batch, m) == (m > 3)
    q = torch.zeros((m * batch, nh, hd), dtype=torch.float16, device="cuda")
    q[:, :, 0] = 20.5 * 0.6931471805599453 * hd ** 0.5
    o = torch.empty((m * batch, nh, hd), device="cuda")
    lse = torch.empty((m * batch, nh), device="cuda")
    cache.prefill(q, ints(*offsets([m] * batch)), m, ints(*[n] * batch), tables, out=o, lse=lse)
    r = ref.attend(q[:m], *ref.held_values(cache, tables, 0, n), n)
    assert 0.035 < float(r["o"][0, 0, 0]) < 0.05
    err = ref.score_error(r, hd)
    # half a step of the weights, relative; 2^-32 of the heaviest's block each; the scores' error
    tol = (2.0 ** -24 * r["o"].abs() + (2.0 ** -11 + err[..., None]) * r["abs"]
           + n * 2.0 ** -32 * r["vmax"])
    for b in range(batch):
        rows = slice(b * m, b * m + m)
        ref.assert_within(o[rows], r["o"], tol)
        ref.assert_within(lse[rows], r["lse"], err + 2.0 ** -22 * (1 + r["lse"].abs()))


@pytest.mark.parametrize("heads,most", [((10, 2, 128), 3), ((8, 2, 64), 20), ((32, 8, 128), 70),
                                        ((14, 2, 64), 80)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (50, 3)])
def test_queries_past_max_q_leave_the_others_where_they_stand(q8, heads, most, window, sinks):  # noqa: F811
    nh, nkv, hd = heads
    lens, ms = [300, 40, 1000], [most + 50, 1, most]
    cache, tables, seq = make(q8, nh, nkv, hd, 32, "e4m3", lens, seed=most)
    spoil(cache, tables, lens)
    gen = torch.Generator("cuda").manual_seed(most + 1)
    cu = offsets(ms)
    q = randn(gen, cu[-1], nh, hd)
    out = torch.full_like(q, 7.0)
    lse = torch.full((cu[-1], nh), 7.0, device="cuda")
    names = dict(window=window, sinks=sinks)
    assert runs_prefill(q8, cache, cu[-1], most) == (most >= 70)
    cache.prefill(q, ints(*cu), most, seq, tables, out=out, lse=lse, **names)
    want = cache.prefill(q, ints(*cu), max(ms), seq, tables, **names)
    check_attention(cache, tables, lens, q, cu, want, **names)
    assert bool((out[most:cu[1]] == 7).all()) and bool((lse[most:cu[1]] == 7).all())
    out[most:cu[1]] = want[most:cu[1]]
    k, v = ref.held_values(cache, tables, 0, 300)
    lse[most:cu[1]] = ref.attend(q[:cu[1]], k, v, 300, window, sinks)["lse"][most:].float()
    check_attention(cache, tables, lens, q, cu, out, lse, **names)
    if most <= 64:
        w = torch.empty((3, cache.geo.max_pages_per_seq), device="cuda")
        cache.prefill(q, ints(*cu), most, seq, tables, weights=w, decay=0.0, **names)
        r = ref.attend(q[:cu[1]], k, v, 300, window, sinks)
        sums = r["p"][:, :most].sum((0, 1, 2))
        sums = torch.cat((sums, sums.new_zeros(20))).view(-1, 32).sum(1)
        ref.assert_within(w[0, :10], sums, (float(ref.score_error(r, hd).max()) + 2.0 ** -14) * sums
                          + 2.0 ** -100)


@pytest.mark.parametrize("decay", [0.0, 0.5, 1.0])
def test_weights_decay_in_a_call_of_no_queries(q8, decay):  # noqa: F811
    """As those of a sequence without queries do beside one that has some."""
    cache, tables, seq = make(q8, 10, 2, 64, 32, "int8", [300, 40], seed=3)
    gen = torch.Generator("cuda").manual_seed(4)
    held = torch.rand((2, cache.geo.max_pages_per_seq), generator=gen, device="cuda")
    q = randn(gen, 2, 10, 64)
    want = held.clone()
    cache.prefill(q, ints(0, 0, 2), 2, seq, tables, weights=want, decay=decay)
    want[1] = decay * held[1]
    for rows, most in ((q[:0], 5), (q[:0], 0), (q, 0)):
        w = held.clone()
        if decay == 0.0:
            w[0, 0] = float("nan")
        out = torch.full((rows.shape[0], 10, 64), 7.0, dtype=torch.float16, device="cuda")
        cache.prefill(rows, ints(0, 0, rows.shape[0]), most, seq, tables, weights=w, decay=decay,
                      out=out)
        assert torch.equal(w, want) and bool((out == 7).all())


def test_a_tensor_put_in_the_place_of_another_is_the_one_used(q8):  # noqa: F811
    cache, tables, seq = make(q8, 4, 2, 64, 16, "int8", [37, 20], seed=8)
    gen = torch.Generator("cuda").manual_seed(9)
    k, v, q = randn(gen, 2, 2, 64), randn(gen, 2, 2, 64), randn(gen, 2, 4, 64)
    before = cache.decode(q, seq, tables)
    for name in ("k_tail", "v_tail", "k_code"):
        old = getattr(cache, name)
        keep = old.clone()
        setattr(cache, name, keep)
        old.fill_(1)  # nothing reads it any more
    assert torch.equal(cache.decode(q, seq, tables), before)
    cache.append(k, v, tables, seq)
    assert torch.equal(cache.k_tail[0, :, 5], k[0]) and torch.equal(cache.v_tail[1, :, 4], v[1])
    got = cache.decode(q, seq + 1, tables)
    check_attention(cache, tables, [38, 21], q, [0, 1, 2], got)


@pytest.mark.parametrize("heads,batch", [((32, 8, 128), 64), ((14, 2, 64), 65), ((16, 1, 64), 300),
                                         ((8, 1, 128), 5000)])
def test_prompts_of_few_among_many_sequences(q8, heads, batch):  # noqa: F811
    """Most sequences have no query, some one, few as many as a prompt has; one is long, so that
    its row tiles are cut and merged.  Rows before, between and behind them stay."""
    rng = random.Random(batch)
    nh, nkv, hd = heads
    lens = [rng.choice((0, 1, 17, 64, 200)) for _ in range(batch)]
    ms = [rng.choice((0, 0, 0, 0, 0, 0, 0, 0, 0, 1)) if n else 0 for n in lens]
    for b, n, m in ((0, 300, 40), (batch // 3, 9000, 130), (batch // 3 + 1, 40, 40),
                    (batch // 2, 700, 33), (batch - 1, 150, 150)):
        lens[b], ms[b] = n, m
    cache, tables, seq = make(q8, nh, nkv, hd, 32, "int8", lens, seed=batch)
    spoil(cache, tables, lens)
    cu = [3 + x for x in offsets(ms)]
    total, most = cu[-1] + 50, 150
    assert runs_prefill(q8, cache, total, most)
    size = q8.lib().jacq_q8_attend_workspace_size(cache.geo.ref, batch, total, most, 0)
    assert size >= 2 * total * nh * (hd + 2) * 4  # slices
    gen = torch.Generator("cuda").manual_seed(batch)
    q = randn(gen, total, nh, hd)
    some = [b for b in range(batch) if ms[b] > 1] + rng.sample([b for b in range(batch) if ms[b] == 1],
                                                               min(20, ms.count(1)))
    for window, sinks in ((None, 0), (100, 3)):
        names = dict(window=window, sinks=sinks)
        out, lse = torch.full_like(q, 7.0), torch.full((total, nh), 7.0, device="cuda")
        cache.prefill(q, ints(*cu), most, seq, tables, out=out, lse=lse, **names)
        for b in some:
            rows = slice(cu[b], cu[b + 1])
            check_attention(cache.sequence_view(b), tables[b:b + 1], lens[b:b + 1], q[rows],
                            [0, ms[b]], out[rows], lse[rows], **names)
        assert not bool((lse[3:cu[-1]] == 7).any())  # every row has been written
        for x in (out, lse):
            assert bool((x[:3] == 7).all()) and bool((x[cu[-1]:] == 7).all())
