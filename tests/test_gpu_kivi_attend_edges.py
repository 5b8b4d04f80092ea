"""Edges of the int4 cache's attention of chunks, through both of its kernels: the one for few queries
takes few rows or little work, the prompts' the rest, so each size here says which one it is for."""
from __future__ import annotations

import ctypes
import random

import pytest

torch = pytest.importorskip("torch")

from tests import kivi_attend_ref as ref  # noqa: E402
from tests.test_gpu_kivi_attend import (I32, check, ints, is_prompt, kivi, make,  # noqa: E402,F401
                                        offsets, randn)

pytestmark = pytest.mark.gpu
WIDE = 262080  # tokens of a table that makes prompts of calls of 320 rows and more (kPromptWork)
# (heads, queries of a sequence, whether that is a prompt under a wide table)
SIZES = [((10, 2, 128), 3, False), ((14, 2, 64), 2, False), ((32, 2, 128), 21, True),
         ((14, 2, 64), 47, True)]


def call(kivi, nh, nkv, hd, page, lens, m, prompt, seed=0, residual=64, **kw):  # noqa: F811
    """A cache, queries and offsets of a call that is, or is not, a prompt's."""
    cache, tables, seq = make(kivi, nh, nkv, hd, page, residual, lens, seed=seed,
                              width=(WIDE + 64 - residual) // page if prompt else None, **kw)
    cu = offsets([m] * len(lens) if isinstance(m, int) else m)
    most = max(b - a for a, b in zip(cu, cu[1:]))
    assert is_prompt(kivi, cache, cu[-1], most) == prompt
    gen = torch.Generator("cuda").manual_seed(seed + 1)
    return cache, tables, seq, randn(gen, cu[-1], nh, hd), cu, most


def same(a, b):
    """Equal, NaN where the other is."""
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(), b.nan_to_num())


@pytest.mark.parametrize("page", [16, 32])
@pytest.mark.parametrize("heads,m,prompt", SIZES)
def test_a_page_outside_the_pool_is_nan_to_those_who_see_it(kivi, heads, m, prompt, page):  # noqa: F811
    lens = [500, 333, 64 + 37]
    cache, tables, seq, q, cu, most = call(kivi, *heads, page, lens, m, prompt, seed=m)
    clean = cache.prefill(q, ints(*cu), most, seq, tables)
    check(cache, tables, lens, q, cu, clean)
    # a page in the midst of the first sequence, the second page of a group, one the last queries' windows
    # begin behind
    tables[0, 160 // page] = -1
    tables[1, (32 + 31) // page] = cache.geo.num_pages
    tables[2, 0] = 2 ** 31 - 1
    # what is read in their place may be anything
    cache.k_scale[0], cache.k_zero[0] = float("inf"), float("nan")
    cache.v_scale[0], cache.v_zero[0] = float("nan"), float("inf")
    for window, sinks in ((None, 0), (64, 0), (64, 40), (300, 7)):
        got = cache.prefill(q, ints(*cu), most, seq, tables, window=window, sinks=sinks)
        check(cache, tables, lens, q, cu, got, window=window, sinks=sinks)
    got = cache.cross(q, ints(*cu), most, seq, tables)
    check(cache, tables, lens, q, cu, got, causal=False)
    k, v = cache.read(seq * 0, seq, tables, sum(lens))
    at = 0
    for b, n in enumerate(lens):
        *want, there = ref.exact_values(cache, tables, b, n)
        for x, w in zip((k, v), want):
            part = x[at:at + n]
            assert bool(part[~there].isnan().all())
            part, w = part[there], ref.to_half(w.transpose(0, 1)[there])
            assert same(part, w)
        at += n


@pytest.mark.parametrize("heads,m,prompt", SIZES)
def test_values_that_are_not_finite_reach_no_query_before_them(kivi, heads, m, prompt):  # noqa: F811
    nh, nkv, hd = heads
    lens = [400, 300, 97, 160]
    cache, tables, seq, q, cu, most = call(kivi, *heads, 16, lens, m, prompt, seed=3)
    inf, nan = float("inf"), float("nan")
    # fp16 tokens among the last queries' own, one channel each
    for b, n in enumerate(lens):
        left = n - ref.old_tokens(cache.geo, n)
        cache.v_scr[b, 0, left - 1, 5] = (nan, inf, -inf, nan)[b]
        cache.k_scr[b, nkv - 1, left - 2, 7] = nan
        cache.v_scr[b, nkv - 1, left // 2, hd - 1] = -inf
    # int4 tokens: scales and zeros of V of a token, of K of a group; the largest that stay finite
    page = tables[0, 20 // 16].long()
    cache.v_scale[page, 0, 20 % 16, 0] = inf
    cache.v_zero[tables[1, 100 // 16].long(), 0, 100 % 16, hd // 32 - 1] = nan
    cache.k_scale[tables[1, 160 // 16].long(), 0, 9] = nan
    p3 = tables[3, 2].long()
    cache.v_scale[p3, 0], cache.v_zero[p3, 0] = 8730.0, -65504.0
    cache.v_scale[p3, nkv - 1], cache.v_zero[p3, nkv - 1] = 8800.0, -30000.0  # up to 102000
    for window, sinks in ((None, 0), (30, 0), (30, 21), (200, 2)):
        got = cache.prefill(q, ints(*cu), most, seq, tables, window=window, sinks=sinks,
                            out=torch.empty(cu[-1], nh, hd, device="cuda"))
        for b, n in enumerate(lens):
            rows = slice(cu[b], cu[b + 1])
            k, v = ref.held_values(cache, tables, b, n)
            if b == 3:  # by scale and zero alone, whether a code is large enough or not
                k[nkv - 1, 32:48], v[nkv - 1, 32:48] = nan, 0.0
            r = ref.attend(q[rows], k, v, window, sinks)
            ref.assert_within(got[rows], r["o"], ref.tolerance(r, hd, got.dtype),
                              f"sequence {b}, window {window}, sinks {sinks}")


@pytest.mark.parametrize("heads,m,prompt", SIZES)
def test_queries_that_are_not_finite_are_nan_alone(kivi, heads, m, prompt):  # noqa: F811
    lens = [150, 260, 90]
    cache, tables, seq, q, cu, most = call(kivi, *heads, 16, lens, m, prompt, seed=4)
    for dtype in (torch.float16, torch.bfloat16):
        x = q.to(dtype)
        x[1, 1, 3], x[m, 0, 0], x[2 * m + 1, 2, 9] = float("nan"), float("inf"), float("-inf")
        got = cache.prefill(x, ints(*cu), most, seq, tables)
        bad = torch.zeros(cu[-1], heads[0], dtype=torch.bool, device="cuda")
        bad[1, 1] = bad[m, 0] = bad[2 * m + 1, 2] = True
        assert torch.equal(got.isnan().any(-1), bad) and torch.equal(got.isnan().all(-1), bad)


@pytest.mark.parametrize("heads,m,prompt", SIZES)
def test_large_scores_and_far_scales(kivi, heads, m, prompt):  # noqa: F811
    """Softmax of a token or two; bf16 beyond fp16's range; maxima that keep rising."""
    nh, nkv, hd = heads
    lens = [600, 222]
    cache, tables, seq, q, cu, most = call(kivi, *heads, 16, lens, m, prompt, seed=5)
    got = cache.prefill(q * 30, ints(*cu), most, seq, tables)
    check(cache, tables, lens, q * 30, cu, got)
    for factor in (2.0 ** 60, 2.0 ** -60):
        big = q.to(torch.bfloat16) * factor
        got = cache.prefill(big, ints(*cu), most, seq, tables, scale=hd ** -0.5 / factor)
        check(cache, tables, lens, big, cu, got, scale=hd ** -0.5 / factor)
    # rising: the keys of later groups are multiples of earlier ones
    for b, n in enumerate(lens):
        for t in range(0, ref.old_tokens(cache.geo, n), 16):
            cache.k_scale[tables[b, t // 16].long()] *= 1 + t // 32 / 8
    got = cache.prefill(q, ints(*cu), most, seq, tables)
    check(cache, tables, lens, q, cu, got)


@pytest.mark.parametrize("heads,m,prompt", SIZES)
def test_rows_outside_and_past_max_q_are_left(kivi, heads, m, prompt):  # noqa: F811
    nh, nkv, hd = heads
    lens = [300, 140, 75]
    cache, tables, seq, q, cu, most = call(kivi, *heads, 32, lens, m, prompt, seed=6)
    gen = torch.Generator("cuda").manual_seed(8)
    wide = randn(gen, 3 * m + 9, nh * hd + 24)
    x = wide[:, 16:16 + nh * hd].unflatten(1, (nh, hd))  # rows that lie apart
    where = ints(4, 4 + m, 4 + 2 * m, 4 + 3 * m)
    most = m - 1
    if prompt:
        assert is_prompt(kivi, cache, x.shape[0], most)
    out = torch.full((x.shape[0], nh, hd), 7.0, device="cuda", dtype=torch.float16)
    lse = torch.full((x.shape[0], nh), 7.0, device="cuda")
    for causal in (True, False):
        out.fill_(7.0)
        lse.fill_(7.0)
        (cache.prefill if causal else cache.cross)(x, where, most, seq, tables, out=out, lse=lse)
        for b, n in enumerate(lens):
            at = 4 + b * m
            r = ref.attend(x[at:at + m], *ref.held_values(cache, tables, b, n), causal=causal)
            tol = ref.tolerance(r, hd, out.dtype)
            ref.assert_within(out[at:at + most], r["o"][:most], tol[:most], f"sequence {b}")
            assert bool((out[at + most:at + m] == 7.0).all()) and bool((lse[at + most:at + m] == 7).all())
        assert bool((out[:4] == 7.0).all()) and bool((out[4 + 3 * m:] == 7.0).all())
        assert bool((lse[:4] == 7.0).all()) and bool((lse[4 + 3 * m:] == 7.0).all())
    # offsets outside the tensor and going back: rows that the others do not name are as they should be
    out.fill_(7.0)
    cache.prefill(x, ints(-5, m, 2, 2), most, seq, tables, out=out)
    r = ref.attend(x[:m], *ref.held_values(cache, tables, 0, lens[0]))
    ref.assert_within(out[:most], r["o"][:most], ref.tolerance(r, hd, out.dtype)[:most], "the first")
    assert bool((out[most:] == 7.0).all())


@pytest.mark.parametrize("batch", [64, 65, 200, 1100])
def test_many_sequences(kivi, batch):  # noqa: F811
    """Cuts planned by every workgroup, by a kernel; sequences without queries between the others."""
    rng = random.Random(batch)
    nh, nkv, hd = 8, 2, 64
    lens = [rng.choice((0, 1, 40, 97, 130)) for _ in range(batch)]
    for b in (0, batch // 2, batch - 1):
        lens[b] = 1500
    cache, tables, seq = make(kivi, nh, nkv, hd, 16, 32, lens, seed=batch)
    gen = torch.Generator("cuda").manual_seed(batch)
    for m in ([1] * batch, [rng.choice((0, 0, 1, 3)) for _ in range(batch)],
              [rng.choice((0, 0, 5, 90)) if n else 0 for n in lens]):
        cu = offsets(m)
        q = randn(gen, cu[-1], nh, hd)
        got = cache.prefill(q, ints(*cu), max(m), seq, tables, window=700, sinks=5)
        check(cache, tables, lens, q, cu, got, window=700, sinks=5)
        got = cache.cross(q, ints(*cu), max(m), seq, tables)
        check(cache, tables, lens, q, cu, got, causal=False)


@pytest.mark.parametrize("batch", [6, 40, 90])
@pytest.mark.parametrize("heads", [(40, 8, 128), (14, 2, 64), (16, 1, 64)])
def test_steps_beside_prompts(kivi, heads, batch):  # noqa: F811
    """A call of sequences for both kernels: none, one, a few queries, as many as the one takes and one
    more, some hundreds."""
    rng = random.Random(batch)
    nh, nkv, hd = heads
    split = 32 // (nh // nkv)
    lens = [rng.choice((1, 100, 333, 900, 1600)) for _ in range(batch)]
    lens[1], lens[2] = 2000, 1200
    m = [rng.choice((0, 1, 1, 2, split, split + 1)) for _ in lens]
    m[1], m[2] = 400, split + 1
    cache, tables, seq = make(kivi, nh, nkv, hd, 16, 64, lens, seed=batch,
                              width=(WIDE if batch < 9 else 20000) // 16)
    cu = offsets(m)
    assert 2 * cu[-1] <= batch * 400 and is_prompt(kivi, cache, cu[-1], 400)
    gen = torch.Generator("cuda").manual_seed(batch)
    q = randn(gen, cu[-1], nh, hd, dtype=torch.bfloat16)
    for window, sinks in ((None, 0), (500, 40)):
        lse = torch.empty(cu[-1], nh, device="cuda")
        got = cache.prefill(q, ints(*cu), 400, seq, tables, window=window, sinks=sinks, lse=lse)
        check(cache, tables, lens, q, cu, got, lse, window, sinks)
    got = cache.cross(q, ints(*cu), 400, seq, tables)
    check(cache, tables, lens, q, cu, got, causal=False)


def test_steps_beside_a_prompt_captured(kivi):  # noqa: F811
    """With other queries, offsets (so other sequences for each kernel) and lengths copied in."""
    nh, nkv, hd, batch = 16, 2, 128, 12
    lens = [700 + 31 * b for b in range(batch)]
    cache, tables, seq = make(kivi, nh, nkv, hd, 32, 32, lens, seed=1, width=WIDE // 32)
    gen = torch.Generator("cuda").manual_seed(3)
    q, where = randn(gen, 420, nh, hd), torch.zeros(batch + 1, **I32)
    assert is_prompt(kivi, cache, 420, 300)
    out = torch.empty_like(q)

    def call():
        cache.prefill(q, where, 300, seq, tables, window=400, sinks=2, out=out)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    rng = random.Random(4)
    for i in range(4):
        m = [rng.choice((0, 1, 4, 5)) for _ in lens]
        m[rng.randrange(batch)] = 300
        m[rng.randrange(batch)] = 40
        q.copy_(randn(gen, *q.shape))
        where.copy_(ints(*offsets(m)))
        out.fill_(7.0)
        graph.replay()
        check(cache, tables, lens, q, offsets(m), out, window=400, sinks=2)
        assert bool((out[sum(m):] == 7.0).all())
        got = out.clone()
        out.fill_(7.0)
        call()
        assert torch.equal(got, out)


@pytest.mark.parametrize("heads,m,prompt", SIZES)
def test_lengths_are_clamped(kivi, heads, m, prompt):  # noqa: F811
    nh, nkv, hd = heads
    lens = [0, 200, 64 + 320]
    cache, tables, seq, q, cu, most = call(kivi, *heads, 16, lens, m, prompt, seed=8)
    cap = cache.geo.max_pages_per_seq * 16 // 32 * 32 + 64
    wild = ints(-2 ** 31, 200, 2 ** 31 - 1 if not prompt else 384)
    if not prompt:
        assert lens[2] == cap
    assert torch.equal(cache.prefill(q, ints(*cu), most, wild, tables),
                       cache.prefill(q, ints(*cu), most, seq, tables))
    assert torch.equal(cache.cross(q, ints(*cu), most, wild, tables),
                       cache.cross(q, ints(*cu), most, seq, tables))
    for a, b in zip(cache.read(ints(5, -9, 100), wild, tables, 484),
                    cache.read(ints(0, 0, 100), seq, tables, 484)):
        assert torch.equal(a, b) and bool(a.isfinite().all())


@pytest.mark.parametrize("heads,m,prompt", SIZES)
def test_the_output_may_be_the_queries(kivi, heads, m, prompt):  # noqa: F811
    cache, tables, seq, q, cu, most = call(kivi, *heads, 32, [2000, 300, 77], m, prompt, seed=2)
    want = cache.prefill(q, ints(*cu), most, seq, tables)
    assert cache.prefill(q, ints(*cu), most, seq, tables, out=q) is q
    assert torch.equal(q, want)


@pytest.mark.parametrize("batch,longest,prompt", [(7, 200, False), (7, 2100, True), (70, 200, True)])
@pytest.mark.parametrize("hd", [64, 128])
def test_prompts_in_passes(kivi, batch, longest, prompt, hd):  # noqa: F811
    """Tiles laid a few at a time, sequences that begin in one pass and end behind it."""
    rng = random.Random(batch)
    lens = [rng.choice((0, 65, 300, 1000)) for _ in range(batch)]
    lens[3] = 2100
    cache, tables, seq = make(kivi, 16, 2, hd, 32, 32, lens, seed=batch, width=2100 // 32 + 1)
    m = [min(n, rng.choice((0, 1, 130, 200))) for n in lens]
    m[3] = longest
    cu = offsets(m)
    gen = torch.Generator("cuda").manual_seed(1)
    q = randn(gen, cu[-1], 16, hd)
    assert is_prompt(kivi, cache, cu[-1], longest) == prompt
    once = cache.prefill(q, ints(*cu), longest, seq, tables)
    check(cache, tables, lens, q, cu, once)
    images = min(batch, cu[-1]) * ((66 * 32 + 32 + 63) // 64)
    pass_bytes = kivi.lib().jacq_kivi_test_pass_bytes
    pass_bytes.argtypes, pass_bytes.restype = [ctypes.c_int64], None
    for passes in (2, 5, 40, 60):  # of 7 sequences 60 are rounded up to 80, too many: the other kernel
        pass_bytes(images * 4 * 64 * hd * 2 // passes)
        try:
            # with a geometry of its own: sizes are kept by it
            other = kivi.PagedKiviCache.from_tensors(
                kivi.KiviGeometry(16, 2, hd, 32, 32, 32, tables.shape[1], cache.geo.num_pages),
                dict(zip(("k_code", "k_scale", "k_zero", "v_code", "v_scale", "v_zero", "k_scr", "v_scr"),
                         cache.pool())))
            got = other.prefill(q, ints(*cu), longest, seq, tables)
            check(cache, tables, lens, q, cu, got)
            many = is_prompt(kivi, other, cu[-1], longest)
            assert many == (prompt and (passes < 60 or batch > 7))
            if many:
                assert torch.equal(got, once)
        finally:
            pass_bytes(0)


@pytest.mark.parametrize("heads,m,prompt", SIZES)
def test_long_sequences_in_slices(kivi, heads, m, prompt):  # noqa: F811
    lens = [20000, 700, 9000]
    cache, tables, seq, q, cu, most = call(kivi, *heads, 16, lens, m, prompt, seed=7, residual=128)
    for window, sinks in ((None, 0), (5000, 100)):
        lse = torch.empty(cu[-1], heads[0], device="cuda")
        got = cache.prefill(q, ints(*cu), most, seq, tables, window=window, sinks=sinks, lse=lse)
        check(cache, tables, lens, q, cu, got, lse, window, sinks)
        again = cache.prefill(q, ints(*cu), most, seq, tables, window=window, sinks=sinks, lse=lse)
        assert torch.equal(got, again)  # the same bits


@pytest.mark.parametrize("heads,m,prompt", SIZES)
def test_captured_and_replayed(kivi, heads, m, prompt):  # noqa: F811
    """With new queries, lengths and tables copied in, eager calls between, on a stream of its own."""
    nh, nkv, hd = heads
    lens = [900, 333, 70]
    cache, tables, seq, q, cu, most = call(kivi, *heads, 16, lens, m, prompt, seed=9)
    where = ints(*cu)
    held = (q.clone(), seq.clone(), tables.clone())
    out, xout = torch.empty_like(q), torch.empty_like(q)
    starts = torch.zeros_like(seq)

    def calls():
        cache.prefill(q, where, most, seq, tables, window=200, sinks=3, out=out)
        cache.cross(q, where, most, seq, tables, out=xout)
        return cache.read(starts, seq, tables, sum(lens))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        calls()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        read = calls()
    gen = torch.Generator("cuda").manual_seed(2)
    for i in (0, 1, 2, 3, 0, 0):
        q.copy_(randn(gen, *q.shape))
        now = [n - i * 60 if n > 300 else n for n in lens]
        seq.copy_(ints(*now))
        # shorter sequences: the residual window of each is whatever the scratch holds, NaN among it
        want = (cache.prefill(q, where, most, seq, tables, window=200, sinks=3),
                cache.cross(q, where, most, seq, tables),
                *cache.read(starts, seq, tables, sum(now)))
        out.fill_(0)
        xout.fill_(0)
        graph.replay()
        torch.cuda.synchronize()
        for got, w in zip((out, xout, *read), want):
            assert same(got[:w.shape[0]], w) and (i > 0 or bool(w.isfinite().all()))
    del held


def test_calls_on_two_streams_at_once(kivi):  # noqa: F811
    jobs = [call(kivi, *SIZES[i][0], 16, [3000, 900, 333], SIZES[i][1], SIZES[i][2], seed=i)
            for i in (0, 2)]
    want = [c.prefill(q, ints(*cu), most, seq, t) for c, t, seq, q, cu, most in jobs]
    streams = [torch.cuda.Stream() for _ in jobs]
    where = [ints(*cu) for *_, cu, _ in jobs]
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for (c, t, seq, q, cu, most), s, w in zip(jobs, streams, where):
            with torch.cuda.stream(s):
                got.append(c.prefill(q, w, most, seq, t))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_a_given_workspace_is_enough_and_may_hold_anything(kivi):  # noqa: F811
    for heads, m, prompt in SIZES:
        cache, tables, seq, q, cu, most = call(kivi, *heads, 16, [3000, 900, 333], m, prompt, seed=m)
        want = cache.prefill(q, ints(*cu), most, seq, tables)
        size = kivi.lib().jacq_kivi_attend_workspace_size(cache.geo.ref, 3, cu[-1], most)
        ws = torch.full((size + 4096,), 0xFF, dtype=torch.uint8, device="cuda")
        got = cache.prefill(q, ints(*cu), most, seq, tables, workspace=ws[:size])
        assert torch.equal(got, want) and bool((ws[size:] == 0xFF).all())
        if size:
            with pytest.raises(kivi.KiviLaunchError, match="workspace"):
                cache.prefill(q, ints(*cu), most, seq, tables, workspace=ws[:size - 1])


def test_offsets_that_go_back_stay_in_the_workspace(kivi):  # noqa: F811
    """More sequences have queries than there are queries: tiles for whose keys there is no room."""
    nh, nkv, hd, total, most, batch = 128, 8, 64, 330, 320, 1000
    geo = kivi.KiviGeometry(nh, nkv, hd, 16, 32, 32, 75, 75)
    cache = kivi.PagedKiviCache(geo, batch)
    for x in cache.pool():
        x.zero_()
    assert is_prompt(kivi, cache, total, most)
    tables = torch.arange(75, **I32).repeat(batch, 1)
    seq = torch.full((batch,), 1200, **I32)
    q = torch.ones(total, nh, hd, dtype=torch.float16, device="cuda")
    size = kivi.lib().jacq_kivi_attend_workspace_size(geo.ref, batch, total, most)
    ws = torch.full((size + (1 << 24),), 0xFF, dtype=torch.uint8, device="cuda")
    for cu in (torch.arange(batch + 1) % (total + 1), torch.arange(batch, -1, -1) % 320,
               (torch.arange(batch + 1) % 2) * total):
        got = cache.prefill(q, cu.to(**I32), most, seq, tables, workspace=ws[:size])
        torch.cuda.synchronize()
        assert bool((ws[size:] == 0xFF).all()), "written behind the workspace"
    del got


def test_pools_past_32_bits(kivi):  # noqa: F811
    """Pages whose codes lie behind the first 4 GiB."""
    nh, nkv, hd, pages = 40, 8, 128, 600_000
    geo = kivi.KiviGeometry(nh, nkv, hd, 16, 32, 32, 64, pages)
    shapes = {"k_code": (pages, nkv, 16, 64), "v_code": (pages, nkv, 16, 64),
              "k_scale": (pages, nkv, 128), "k_zero": (pages, nkv, 128),
              "v_scale": (pages, nkv, 16, 4), "v_zero": (pages, nkv, 16, 4),
              "k_scr": (2, nkv, 64, 128), "v_scr": (2, nkv, 64, 128)}
    cache = kivi.PagedKiviCache.from_tensors(geo, {
        n: torch.empty(s, dtype=torch.uint8 if "code" in n else torch.float16, device="cuda")
        for n, s in shapes.items()})
    assert cache.k_code.numel() > 2 ** 32
    gen = torch.Generator("cuda").manual_seed(0)
    lens = [333, 700]
    tables = torch.stack([pages - 1 - torch.arange(64), pages - 100 - torch.arange(64)]).to(**I32)
    for b, n in enumerate(lens):
        k, v = randn(gen, 2, 1, n, nkv, hd)
        cache.sequence_view(b).append(k, v, tables[b:b + 1], torch.zeros(1, **I32))
    for m, prompt in ((2, False), (70, True)):
        cu = offsets([m, m])
        q = randn(gen, cu[-1], nh, hd)
        if prompt:  # under a wider table
            wide = torch.zeros((2, WIDE // 16), **I32)
            wide[:, :64] = tables
            cache.geo = kivi.KiviGeometry(nh, nkv, hd, 16, 32, 32, WIDE // 16, pages)
            tables = wide
        assert is_prompt(kivi, cache, cu[-1], m) == prompt
        got = cache.prefill(q, ints(*cu), m, ints(*lens), tables)
        check(cache, tables, lens, q, cu, got)
    got = cache.read(ints(0, 0), ints(*lens), tables, sum(lens))
    want = [ref.exact_values(cache, tables, b, n) for b, n in enumerate(lens)]
    for i in range(2):
        assert torch.equal(got[i], ref.to_half(torch.cat([w[i] for w in want], 1).transpose(0, 1)))


def test_no_pages_at_all(kivi):  # noqa: F811
    """A table of no width: everything is in the residual window."""
    geo = kivi.KiviGeometry(8, 2, 64, 16, 32, 96, 0, 1)
    cache = kivi.PagedKiviCache(geo, 2)
    gen = torch.Generator("cuda").manual_seed(0)
    cache.k_scr.copy_(randn(gen, *cache.k_scr.shape))
    cache.v_scr.copy_(randn(gen, *cache.v_scr.shape))
    tables, lens = torch.zeros((2, 0), **I32), [96, 17]
    q = randn(gen, 7, 8, 64)
    got = cache.prefill(q, ints(0, 3, 7), 4, ints(*lens), tables)
    check(cache, tables, lens, q, [0, 3, 7], got)
    k, v = cache.read(ints(0, 0), ints(*lens), tables, sum(lens))
    assert torch.equal(k, torch.cat([cache.k_scr[b, :, :n].transpose(0, 1) for b, n in enumerate(lens)]))


def test_random_calls(kivi):  # noqa: F811
    rng = random.Random(20)
    for i in range(25):
        nh, nkv, hd = rng.choice([(14, 2, 64), (40, 8, 128), (5, 5, 128), (16, 1, 64), (24, 2, 64)])
        page, residual = rng.choice((16, 32)), rng.choice((32, 64, 128, 256))
        batch = rng.randint(1, 9)
        lens = [rng.choice((0, 1, 31, 64, rng.randint(1, 400), rng.randint(1, 3000)))
                for _ in range(batch)]
        m = [rng.choice((0, 1, rng.randint(1, 9), rng.randint(1, 400))) for _ in lens]
        wide = rng.random() < 0.5
        cache, tables, seq = make(kivi, nh, nkv, hd, page, residual, lens, seed=i,
                                  width=(WIDE + 64 - residual) // page if wide else None)
        cu = offsets(m)
        gen = torch.Generator("cuda").manual_seed(i)
        q = randn(gen, cu[-1], nh, hd, dtype=rng.choice((torch.float16, torch.bfloat16)))
        window, sinks = rng.choice(((None, 0), (rng.randint(1, 2000), rng.choice((0, 1, 70, 500)))))
        print(i, nh, nkv, hd, page, residual, lens, m, wide, window, sinks, flush=True)
        lse = torch.empty(cu[-1], nh, device="cuda") if rng.random() < 0.5 else None
        got = cache.prefill(q, ints(*cu), max(m), seq, tables, window=window, sinks=sinks, lse=lse)
        check(cache, tables, lens, q, cu, got, lse, window, sinks)
        got = cache.cross(q, ints(*cu), max(m), seq, tables, lse=lse)
        check(cache, tables, lens, q, cu, got, lse, causal=False)
