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


# The decode's kernel takes up to 64 rows (queries x heads of a kv head) or 2048 (query, head) rows of
# a call: a few heads stay in it, 70 queries of 32/8 heads do not.
BOTH = pytest.mark.parametrize("heads,m,prompt", [((4, 2, 64), 40, False), ((10, 2, 128), 12, False),
                                                  ((32, 8, 128), 70, True), ((28, 4, 64), 90, True)])


@BOTH
@pytest.mark.parametrize("codes", ["int8", "e4m3"])
@pytest.mark.parametrize("where", ["block", "tail"])
def test_a_nan_key_reaches_the_queries_that_see_it(q8, heads, m, prompt, codes, where):  # noqa: F811
    """One kv head of one token, in K or V; windows that end before it."""
    nh, nkv, hd = heads
    g, page, n = nh // nkv, 16, 16 * 20 + 9
    gen = torch.Generator("cuda").manual_seed(m)
    k, v = randn(gen, n, nkv, hd), randn(gen, n, nkv, hd)
    at = n - 9 - max(page, m // 2) if where == "block" else n - 4
    (k if codes == "int8" else v)[at, 1, 7] = float("nan")
    cache = q8.PagedQ8Cache(q8.Q8Geometry(nh, nkv, hd, page, 32, 32, codes), 1)
    tables = torch.randperm(32, generator=gen, device="cuda").to(torch.int32).view(1, 32)
    cache.append(k, v, tables, ints(0), cu_new=ints(0, n))
    assert runs_prefill(q8, cache, m, m) == prompt
    q = randn(gen, m, nh, hd)
    pos = torch.arange(n - m, n, device="cuda")
    first = at // page * page if where == "block" else at  # a block quantised with it is NaN whole
    last = (at // page + 1) * page - 1 if where == "block" else at
    for window, sinks in ((None, 0), (7, 0), (5, 3)):
        lse = torch.empty((m, nh), device="cuda")
        got = cache.prefill(q, ints(0, m), m, ints(n), tables, window=window, sinks=sinks, lse=lse)
        sees = pos >= first
        if window is not None:
            sees &= pos - window < last
        assert 0 < int(sees.sum()) <= m - (m > 40 or where == "tail")
        head = torch.arange(nh, device="cuda") // g == 1
        want = sees[:, None] & head[None]
        assert torch.equal(got.isnan().all(-1), want) and torch.equal(got.isnan().any(-1), want)
        assert torch.equal(lse.isnan(), want)
        check = [h for h in range(nh) if h // g != 1]
        kk, vv = ref.held_values(cache, tables, 0, n)
        r = ref.attend(q, kk.nan_to_num(0), vv, n, window, sinks)
        tol = ref.tolerance(r, hd, torch.float16)
        ref.assert_within(got[:, check], r["o"][:, check], tol[:, check])
        ref.assert_within(got[~sees], r["o"][~sees], tol[~sees])


@BOTH
def test_queries_of_any_size_through_both_kernels(q8, heads, m, prompt):  # noqa: F811
    """bf16 queries past fp16's range and below it, a row of zeros, NaN and infinity, beside keys of
    a zero block; causal, so that tiles are masked in part."""
    nh, nkv, hd = heads
    page, n = 32, 300
    gen = torch.Generator("cuda").manual_seed(m)
    k = randn(gen, n, nkv, hd)
    v = randn(gen, n, nkv, hd)
    k[256:288] = 0  # its scale of K is 2^-24 / 127
    cache = q8.PagedQ8Cache(q8.Q8Geometry(nh, nkv, hd, page, 10, 10, "int8"), 1)
    tables = torch.arange(10, **I32).flip(0).contiguous().view(1, 10)
    cache.append(k, v, tables, ints(0), cu_new=ints(0, n))
    assert runs_prefill(q8, cache, m, m) == prompt
    q = randn(gen, m, nh, hd, dtype=torch.bfloat16)
    sizes = torch.tensor([1e8, 1e-8, 1.0, 1e-30, 0.0, 1e5, 1e-36], device="cuda")
    f = sizes[torch.arange(m * nh, device="cuda") % 7].view(m, nh, 1)
    q = (q.float() * f).bfloat16()
    for scale in (1e-7, 0.1):
        rows = torch.ones((m, nh), dtype=torch.bool, device="cuda")
        if scale == 0.1:
            # scores of 1e6 and more are one key's alone: their error is past any weight's
            rows = f[..., 0] < 1e4
        o = torch.empty((m, nh, hd), device="cuda")
        lse = torch.empty((m, nh), device="cuda")
        cache.prefill(q, ints(0, m), m, ints(n), tables, scale=scale, out=o, lse=lse)
        r = ref.attend(q, *ref.held_values(cache, tables, 0, n), n, scale=scale)
        tol = ref.tolerance(r, hd, torch.float32)
        ref.assert_within(o[rows], r["o"][rows], tol[rows])
        err = ref.score_error(r, hd) + 2.0 ** -22 * (1 + r["lse"].abs())
        ref.assert_within(lse[rows], r["lse"][rows], err[rows])
    clean = cache.prefill(q, ints(0, m), m, ints(n), tables, scale=1e-7)
    q[m - 3, 1, 5], q[m // 2, nh - 1, 9] = float("nan"), float("inf")
    got = cache.prefill(q, ints(0, m), m, ints(n), tables, scale=1e-7)
    bad = torch.zeros((m, nh), dtype=torch.bool, device="cuda")
    bad[m - 3, 1] = bad[m // 2, nh - 1] = True
    assert bool(got[bad].isnan().all()) and torch.equal(got[~bad], clean[~bad])


@BOTH
@pytest.mark.parametrize("codes", ["int8", "e4m3"])
def test_blocks_whose_scales_differ_by_far_through_both_kernels(q8, heads, m, prompt, codes):  # noqa: F811
    """V of the blocks differs by factors of up to 2^20; the blocks of the largest are as good as
    unseen, so what O is made of is small beside them."""
    nh, nkv, hd = heads
    page, n = 16, 16 * 12 + 7
    gen = torch.Generator("cuda").manual_seed(m)
    k, v = randn(gen, n, nkv, hd, scale=0.1), randn(gen, n, nkv, hd)
    f = torch.tensor([1.0, 2.0 ** -10, 2.0 ** 10, 2.0 ** -14, 0.0, 3.0], device="cuda").repeat(3)
    v = (v * f.repeat_interleave(page)[:n].view(n, 1, 1)).half()
    for block in (2, 8):
        k[block * page:(block + 1) * page] = -8.0
    cache = q8.PagedQ8Cache(q8.Q8Geometry(nh, nkv, hd, page, 13, 13, codes), 1)
    tables = torch.arange(13, **I32).view(1, 13)
    cache.append(k, v, tables, ints(0), cu_new=ints(0, n))
    assert runs_prefill(q8, cache, m, m) == prompt
    q = torch.full((m, nh, hd), 0.7, dtype=torch.float16, device="cuda")
    q += randn(gen, m, nh, hd, scale=0.05)
    o = torch.empty((m, nh, hd), device="cuda")
    cache.prefill(q, ints(0, m), m, ints(n), tables, out=o)
    kk, vv = ref.held_values(cache, tables, 0, n)
    r = ref.attend(q, kk, vv, n)
    # what fp16 weights lose, 2^-32 of the heaviest's block a token, is of what weighs anything
    seen = r["p"].amax((0, 1, 2)) > 2.0 ** -30
    assert not bool(seen[32:48].any()) and bool(seen[16:32].all())
    r["vmax"] = vv[:, seen].abs().amax()
    ref.assert_within(o, r["o"], ref.tolerance(r, hd, torch.float32))


@pytest.mark.parametrize("heads", [(32, 8, 128), (14, 2, 64), (16, 1, 64)])
@pytest.mark.parametrize("step", [-1, 0, 1])
def test_either_side_of_the_rule_between_the_kernels(q8, heads, step):  # noqa: F811
    """64 rows of a kv head, and 2048 (query, head) rows of a call: the last of the one kernel, the
    first of the other, and all of both batches against the definition."""
    nh, nkv, hd = heads
    for batch, m in ((2048 // (64 // (nh // nkv) * nh) + 3, 64 // (nh // nkv) + step),
                     (1, 2048 // nh + step)):
        if m < 1:
            continue
        lens = [m + 70 * b + 5 for b in range(batch)]
        cache, tables, seq = make(q8, nh, nkv, hd, 32, "int8", lens, seed=m + batch)
        spoil(cache, tables, lens)
        cu = offsets([m] * batch)
        gen = torch.Generator("cuda").manual_seed(m)
        q = randn(gen, cu[-1], nh, hd, dtype=torch.bfloat16)
        assert (runs_prefill(q8, cache, cu[-1], m)
                == (m * (nh // nkv) > 64 and cu[-1] * nh > 2048))
        lse = torch.empty((cu[-1], nh), device="cuda")
        got = cache.prefill(q, ints(*cu), m, seq, tables, lse=lse)
        check_attention(cache, tables, lens, q, cu, got, lse)


@pytest.mark.parametrize("heads", [(32, 8, 128), (12, 6, 64), (30, 10, 64), (5, 5, 128)])
@pytest.mark.parametrize("m", [1, 7])
def test_block_weights_of_more_kv_heads_than_wavefronts(q8, heads, m):  # noqa: F811
    nh, nkv, hd = heads
    lens = [m, 100, 1003]
    cache, tables, seq = make(q8, nh, nkv, hd, 32, "int8", lens, seed=nkv)
    spoil(cache, tables, lens)
    gen = torch.Generator("cuda").manual_seed(nkv + 1)
    cu = offsets([m] * 3)
    q = randn(gen, cu[-1], nh, hd)
    w = torch.full((3, cache.geo.max_pages_per_seq), float("nan"), device="cuda")
    for window, sinks in ((None, 0), (50, 3)):
        names = dict(window=window, sinks=sinks, weights=w, decay=0.0)
        got = (cache.decode(q, seq, tables, **names) if m == 1 else
               cache.prefill(q, ints(*cu), m, seq, tables, **names))
        check_attention(cache, tables, lens, q, cu, got, weights=w, window=window, sinks=sinks)


@pytest.mark.parametrize("why", ["key", "page"])
def test_weights_of_a_poisoned_sequence_evict_as_nan(q8, why):  # noqa: F811
    """Its weights are NaN, which is lightest: all alike, so the earlier blocks stay.  The others'
    weights are as if it were not there."""
    page, nh, nkv, hd = 16, 16, 8, 64
    lens = [160 + 5, 160 + 5]
    gen = torch.Generator("cuda").manual_seed(11)
    k, v = randn(gen, 2 * 165, nkv, hd), randn(gen, 2 * 165, nkv, hd)
    tables = torch.randperm(22, generator=gen, device="cuda").to(torch.int32).view(2, 11)
    cache = q8.PagedQ8Cache(q8.Q8Geometry(nh, nkv, hd, page, 11, 22, "e4m3"), 2)
    if why == "key":
        k[40, 5, 3] = float("nan")
    cache.append(k, v, tables, ints(0, 0), cu_new=ints(0, 165, 330))
    seen = tables.clone()
    if why == "page":
        seen[0, 2] = -1
    q = randn(gen, 2, nh, hd)
    w = torch.empty((2, 11), device="cuda")
    got = cache.decode(q, ints(*lens), seen, weights=w, decay=0.0)
    assert bool(w[0].isnan().all()) and not bool(w[1].isnan().any())
    check_attention(cache.sequence_view(1), tables[1:], lens[1:], q[1:], [0, 1], got[1:],
                    weights=w[1:])
    names = dict(sink_pages=0, recent_pages=1)
    out = cache.evict(w, ints(*lens), tables, 4, **names)
    want = ref.evict(w.cpu(), lens, tables.cpu(), page, 4, 0, 1)
    for a, b in zip(out, want):
        assert torch.equal(a.cpu().nan_to_num(-5.0) if a.is_floating_point() else a.cpu(),
                           b.nan_to_num(-5.0) if b.is_floating_point() else b)
    assert out[0][0, :4].tolist() == [*tables[0, :3].tolist(), int(tables[0, 9])]
