"""The 8-bit paged cache on the GPU against its definition in 64 bits (tests/q8_ref.py)."""
from __future__ import annotations

import random

import pytest

torch = pytest.importorskip("torch")

from tests import q8_ref as ref  # noqa: E402

pytestmark = pytest.mark.gpu
I32 = {"dtype": torch.int32, "device": "cuda"}


@pytest.fixture(scope="module")
def q8():
    from jacq_amd import q8 as m
    assert torch.cuda.is_available(), "GPU tests need a GPU"
    m.lib()
    return m


def ints(*x):
    return torch.tensor(x, **I32)


def randn(gen, *shape, dtype=torch.float16, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


def make(q8, nh, nkv, hd, page, codes, lens, seed=0, spare=3, dtype=torch.float16, width=None):
    """A cache whose sequences hold `lens` random tokens, appended in one call, in shuffled
    pages; returns (cache, tables, seq_lens)."""
    gen = torch.Generator("cuda").manual_seed(seed)
    need = [-(-n // page) for n in lens]
    width = max([1, *need]) if width is None else width
    pages = sum(need) + spare
    perm = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    tables = torch.full((len(lens), width), -1, **I32)
    at = 0
    for b, k in enumerate(need):
        tables[b, :k] = perm[at:at + k]
        at += k
    geo = q8.Q8Geometry(nh, nkv, hd, page, width, pages, codes)
    cache = q8.PagedQ8Cache(geo, len(lens))
    total = sum(lens)
    k = randn(gen, total, nkv, hd, dtype=dtype)
    k[:, :, 3] *= 5
    v = randn(gen, total, nkv, hd, dtype=dtype)
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    cache.append(k, v, tables, torch.zeros(len(lens), **I32), cu_new=ints(*cu),
                 max_new=max(lens))
    return cache, tables, ints(*lens)


def spoil(cache, tables, lens):
    """NaN, infinities and stray codes wherever no token of a sequence is."""
    used = torch.zeros(cache.geo.num_pages, dtype=torch.bool, device="cuda")
    for b, n in enumerate(lens):
        used[tables[b, :n // cache.geo.page_size].long()] = True
        left = n % cache.geo.page_size
        cache.k_tail[b, :, left:] = float("nan")
        cache.v_tail[b, :, left:] = float("inf")
    cache.k_code[~used] = 0x7F
    cache.v_code[~used] = 0xFF
    cache.k_scale[~used] = float("nan")
    cache.v_scale[~used] = float("inf")


def check_attention(cache, tables, lens, q, cu, got, lse=None, weights=None, window=None, sinks=0,
                    scale=None, held=None, decay=0.0):
    """Every sequence's rows of `got` against the reference over what the cache holds."""
    g = cache.geo
    for b, n in enumerate(lens):
        rows = slice(cu[b], cu[b + 1])
        m = cu[b + 1] - cu[b]
        if m == 0 and weights is None:
            continue
        k, v = ref.held_values(cache, tables, b, n)
        qb = q[rows]
        # queries before the sequence's first token see nothing
        lack = max(0, m - n)
        assert not got[rows][:lack].any()
        r = ref.attend(qb[lack:], k, v, n, window, sinks, scale)
        what = f"sequence {b} of {n} tokens, {m} queries, window {window}, sinks {sinks}"
        ref.assert_within(got[rows][lack:], r["o"], ref.tolerance(r, g.head_dim, got.dtype), what)
        err = ref.score_error(r, g.head_dim)
        if lse is not None:
            assert bool((lse[rows][:lack] == -torch.inf).all())
            ref.assert_within(lse[rows][lack:], r["lse"],
                              err + 2.0 ** -22 * (1 + r["lse"].abs().nan_to_num(posinf=0)), what)
        if weights is not None:
            w = torch.zeros(g.max_pages_per_seq * g.page_size, dtype=torch.float64, device="cuda")
            w[:n] = r["p"].sum((0, 1, 2))
            w = w.view(-1, g.page_size).sum(1)
            if held is not None:
                w = w + decay * held[b].double()
            # a group's sum passes through a base-2 logarithm of up to 2^8 in fp32
            rel = float(err.max() if err.numel() else 0) + 2.0 ** -15 + 2.0 ** -16
            ref.assert_within(weights[b], w, rel * w + 2.0 ** -100, what + " weights")


HEADS = [(4, 4, 64), (14, 2, 64), (10, 2, 128), (8, 1, 128), (16, 1, 128), (32, 2, 64)]


# ---------------------------------------------------------------- append and read

@pytest.mark.parametrize("codes", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("page", [16, 32, 64])
@pytest.mark.parametrize("hd", [64, 128])
def test_append_in_any_pieces_gives_the_definitions_bits(q8, codes, dtype, page, hd):
    rng = random.Random(page * hd)
    gen = torch.Generator("cuda").manual_seed(page + hd)
    nkv, lens = 3, [0, 1, page - 1, page, page + 1, 3 * page + 5, 200]
    width = max(lens) // page + 1
    pages = len(lens) * width
    tables = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32).view(-1, width)
    tables = tables.contiguous()
    k = [randn(gen, n, nkv, hd, dtype=dtype, scale=3.0) for n in lens]
    v = [randn(gen, n, nkv, hd, dtype=dtype, scale=0.02) for n in lens]
    geo = q8.Q8Geometry(6, nkv, hd, page, width, pages, codes)
    cache = q8.PagedQ8Cache(geo, len(lens))
    at = [0] * len(lens)
    while at != lens:  # pieces of any length, some of none
        step = [min(n - a, rng.choice((0, 1, 1, 7, page, 150))) for a, n in zip(at, lens)]
        cu = [0]
        for s in step:
            cu.append(cu[-1] + s)
        # new tokens as a slice of a wider projection: rows lie apart
        wide = torch.zeros((cu[-1], 2 * nkv + 1, hd), dtype=dtype, device="cuda")
        nk, nv = wide[:, :nkv], wide[:, nkv:2 * nkv]
        for b, s in enumerate(step):
            nk[cu[b]:cu[b + 1]] = k[b][at[b]:at[b] + s]
            nv[cu[b]:cu[b + 1]] = v[b][at[b]:at[b] + s]
        cache.append(nk, nv, tables, ints(*at), cu_new=ints(*cu),
                     max_new=max(step) if rng.random() < 0.5 else None)
        at = [a + s for a, s in zip(at, step)]
    for b, n in enumerate(lens):
        full = n // page
        for x, code, scale, tail in ((k[b], cache.k_code, cache.k_scale, cache.k_tail),
                                     (v[b], cache.v_code, cache.v_scale, cache.v_tail)):
            h = ref.as_half(x)
            y, s = ref.quantise(h[:full * page].view(full, page, nkv, hd).transpose(1, 2), codes)
            to = tables[b, :full].long()
            want = ref.code_bytes(y, codes)
            got = code[to].transpose(2, 3) if code is cache.v_code else code[to]
            if codes == "e4m3":  # -0 is as good as 0
                assert torch.equal(ref.byte_values(got, codes), ref.byte_values(want, codes))
            else:
                assert torch.equal(got, want)
            assert torch.equal(scale[to], s.float())  # a / top, rounded once
            assert torch.equal(tail[b, :, :n - full * page],
                               h[full * page:].transpose(0, 1))
    # read back: everything, and a part of every sequence
    for starts in ([0] * len(lens), [n // 3 for n in lens]):
        total = sum(n - s for n, s in zip(lens, starts))
        for out in (torch.float16, torch.bfloat16, torch.float32):
            gk, gv = cache.read(ints(*starts), ints(*lens), tables, total, dtype=out)
            at0 = 0
            for b, n in enumerate(lens):
                wk, wv = ref.held_values(cache, tables, b, n)
                for got, want in ((gk, wk), (gv, wv)):
                    part = want[:, starts[b]:].transpose(0, 1)
                    ref.assert_within(got[at0:at0 + n - starts[b]], part,
                                      2.0 ** -24 * part.abs() * 2 + ref.HALF_STEP[out]
                                      * part.abs() * (1 + 2.0 ** -23) + 2.0 ** -25)
                at0 += n - starts[b]


@pytest.mark.parametrize("codes,values", [
    ("int8", [254.0] + [float(i) for i in range(-253, 254, 2)]),      # 127 x / 254 = x / 2
    ("e4m3", [448.0] + [float(i) for i in range(17, 32, 2)]            # between multiples of 2
     + [float(i) for i in range(-34, -63, -4)] + [i * 2.0 ** -10 for i in (1, 3, 5, 7, 9, -11)])])
def test_halves_go_to_the_even_code(q8, codes, values):
    page, hd = 16, 64
    x = torch.zeros(page * hd, dtype=torch.float16, device="cuda")
    x[:len(values)] = torch.tensor(values, device="cuda")
    x = x.view(page, 1, hd)
    cache = q8.PagedQ8Cache(q8.Q8Geometry(1, 1, hd, page, 1, 1, codes), 1)
    cache.append(x, x.flip(0).contiguous(), ints(0).view(1, 1), ints(0), cu_new=ints(0, page))
    y, _ = ref.quantise(x.view(1, 1, page, hd), codes)
    got = ref.byte_values(cache.k_code, codes)
    assert torch.equal(got, y)
    assert torch.equal(ref.byte_values(cache.v_code, codes).transpose(2, 3), y.flip(2))


@pytest.mark.parametrize("codes", ["int8", "e4m3"])
def test_append_extremes(q8, codes):
    """Zero blocks, infinities, values past fp16 and below it; NaN in K or V of a token."""
    page, hd, nkv = 16, 64, 4
    gen = torch.Generator("cuda").manual_seed(5)
    k = randn(gen, 2 * page, nkv, hd, dtype=torch.bfloat16)
    v = randn(gen, 2 * page, nkv, hd, dtype=torch.bfloat16)
    k[:, 0] = 0
    v[:, 0] = 0
    k[3, 1, 5], v[4, 1, 6] = float("inf"), -float("inf")
    k[:page, 2] *= 1e30
    v[:page, 2] *= 1e-30
    k[5, 3, 7], v[page + 2, 3, 9] = float("nan"), float("nan")
    cache = q8.PagedQ8Cache(q8.Q8Geometry(4, nkv, hd, page, 2, 2, codes), 1)
    tables = ints(1, 0).view(1, 2)
    cache.append(k, v, tables, ints(0), cu_new=ints(0, 2 * page))
    hk, hv = ref.couple_nan(ref.as_half(k), ref.as_half(v))
    for x, code, scale in ((hk, cache.k_code, cache.k_scale), (hv, cache.v_code, cache.v_scale)):
        y, s = ref.quantise(x.view(2, page, nkv, hd).transpose(1, 2), codes)
        got = code[tables[0].long()]
        got = got.transpose(2, 3) if code is cache.v_code else got
        assert torch.equal(ref.byte_values(got, codes), y)
        got = scale[tables[0].long()]
        assert torch.equal(got.isnan(), s.isnan())
        assert torch.equal(got.nan_to_num(0), s.float().nan_to_num(0))
    # and in the tail
    cache = q8.PagedQ8Cache(q8.Q8Geometry(4, nkv, hd, 64, 1, 1, codes), 1)
    cache.append(k, v, ints(0).view(1, 1), ints(0), cu_new=ints(0, 2 * page))
    assert torch.equal(cache.k_tail[0, :, :2 * page].nan_to_num(7.0),
                       hk.transpose(0, 1).nan_to_num(7.0))
    assert torch.equal(cache.v_tail[0, :, :2 * page], hv.transpose(0, 1))


def test_append_drops_what_the_table_does_not_hold(q8):
    """Pages outside the pool, tokens past the table, offsets that do not fit: nothing else is
    touched."""
    page, hd = 16, 64
    gen = torch.Generator("cuda").manual_seed(6)
    cache = q8.PagedQ8Cache(q8.Q8Geometry(2, 2, hd, page, 2, 3, "int8"), 3)
    k, v = randn(gen, 90, 2, hd), randn(gen, 90, 2, hd)
    tables = torch.tensor([[2, 7], [-1, 1], [0, 0]], **I32)
    for t in cache.pool():
        t.zero_()
    cache.append(k, v, tables, ints(0, 0, -3), cu_new=ints(0, 40, 80, 90))  # 40 > 2 x 16
    y, s = ref.quantise(torch.stack((k[:page], k[40 + page:40 + 2 * page])).transpose(1, 2), "int8")
    assert torch.equal(cache.k_code[2], ref.code_bytes(y[0], "int8"))
    assert torch.equal(cache.k_code[1], ref.code_bytes(y[1], "int8"))
    assert not cache.k_code[0].any() and not cache.k_scale[0].any()
    assert not cache.k_tail.any()
    cache.append(k[:3], v[:3], tables, ints(32, 40, 100))  # full sequences: nothing to do
    assert not cache.k_tail.any()
    cache.append(k[:9], v[:9], tables, ints(0, 0, 0), cu_new=ints(0, 1000, -5, 9))
    assert torch.equal(cache.k_tail[0, :, :9], k[:9].transpose(0, 1))


# ---------------------------------------------------------------- decode

@pytest.mark.parametrize("codes", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("page", [16, 32, 64])
def test_decode(q8, codes, dtype, heads, page):
    nh, nkv, hd = heads
    lens = [0, 1, 15, 16, 17, 63, 64, 65, 127, 129, 500, 1021]
    cache, tables, seq = make(q8, nh, nkv, hd, page, codes, lens, seed=nh + page)
    spoil(cache, tables, lens)
    gen = torch.Generator("cuda").manual_seed(1)
    q = randn(gen, len(lens), nh, hd, dtype=dtype, scale=1.5)
    lse = torch.empty((len(lens), nh), device="cuda")
    cu = list(range(len(lens) + 1))
    got = cache.decode(q, seq, tables, lse=lse)
    check_attention(cache, tables, lens, q, cu, got, lse)
    out = torch.empty((len(lens), nh, hd), device="cuda")
    assert cache.decode(q, seq, tables, out=out, scale=0.05) is out
    check_attention(cache, tables, lens, q, cu, out, scale=0.05)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (5, 3), (16, 0), (63, 4), (64, 64),
                                          (100, 200), (129, 17), (1000, 0), (5000, 5000)])
@pytest.mark.parametrize("page", [16, 64])
def test_decode_window_and_sinks(q8, window, sinks, page):
    lens = [0, 1, 2, 17, 64, 100, 130, 700, 1500]
    cache, tables, seq = make(q8, 10, 2, 128, page, "int8", lens, seed=window)
    spoil(cache, tables, lens)
    gen = torch.Generator("cuda").manual_seed(2)
    q = randn(gen, len(lens), 10, 128)
    lse = torch.empty((len(lens), 10), device="cuda")
    got = cache.decode(q, seq, tables, window=window, sinks=sinks, lse=lse)
    check_attention(cache, tables, lens, q, list(range(len(lens) + 1)), got, lse, window=window,
                    sinks=sinks)


@pytest.mark.parametrize("given_back", [False, True])
@pytest.mark.parametrize("m", [1, 3, 50])
@pytest.mark.parametrize("page", [16, 32])
def test_pages_before_the_window_may_hold_anything(q8, page, m, given_back):
    # and their entries may name no page
    lens, window, sinks = [333, 700, 1000, 65], 100, 10
    cache, tables, n = make(q8, 40, 8, 128, page, "e4m3", lens, seed=page)
    gen = torch.Generator("cuda").manual_seed(m)
    q = randn(gen, len(lens) * m, 40, 128)
    cu = [b * m for b in range(len(lens) + 1)]
    names = dict(window=window, sinks=sinks)

    def attend(t):
        if m == 1:
            return cache.decode(q, n, t, **names)
        return cache.prefill(q, ints(*cu), m, n, t, **names)

    want = attend(tables)
    seen = torch.zeros(cache.geo.num_pages, dtype=torch.bool, device="cuda")
    bare = torch.full_like(tables, -1)
    for b, k in enumerate(lens):
        for p in range(k // page):
            if p * page < sinks or (p + 1) * page > k - m + 1 - window:
                seen[int(tables[b, p])] = True
                bare[b, p] = tables[b, p]
    assert int((~seen).sum()) > 4
    cache.k_code[~seen], cache.v_code[~seen] = 0x7F, 0xFF
    cache.k_scale[~seen], cache.v_scale[~seen] = float("inf"), float("nan")
    if given_back:
        # such an entry is read as page 0's codes, which are spoiled too
        spare = int((~seen).nonzero()[-1])
        for x in (cache.k_code, cache.v_code, cache.k_scale, cache.v_scale):
            x[spare] = x[0]
        for x in (cache.k_code, cache.v_code):
            x[0] = 0x7F
        bare[bare == 0] = spare
    assert torch.equal(attend(bare if given_back else tables), want)
    if not given_back:
        check_attention(cache, tables, lens, q, cu, want, **names)


@pytest.mark.parametrize("lens", [[20001], [3, 9000, 1, 0, 12345], [700] * 70 + [5000]])
@pytest.mark.parametrize("codes", ["int8", "e4m3"])
def test_decode_split_over_workgroups(q8, lens, codes):
    cache, tables, seq = make(q8, 8, 2, 128, 32, codes, lens, seed=9)
    gen = torch.Generator("cuda").manual_seed(3)
    q = randn(gen, len(lens), 8, 128, dtype=torch.bfloat16, scale=2)
    got = cache.decode(q, seq, tables)
    check_attention(cache, tables, lens, q, list(range(len(lens) + 1)), got)
    again = cache.decode(q, seq, tables)
    assert torch.equal(got, again)


def test_scales_that_differ_by_far(q8):
    """Blocks whose V (and K) differ by factors of 2^20: no weight is lost next to a large scale."""
    page, hd, n = 16, 64, 16 * 12
    gen = torch.Generator("cuda").manual_seed(4)
    k, v = randn(gen, n, 1, hd, scale=0.1), randn(gen, n, 1, hd)
    f = torch.tensor([1.0, 2.0 ** -10, 2.0 ** 12, 2.0 ** -14, 0.0, 3.0], device="cuda")
    v = (v.view(12, page, 1, hd) * f.repeat(2).view(12, 1, 1, 1)).half().view(n, 1, hd)
    k.view(12, page, 1, hd)[2] = -8.0  # the block of the largest V is as good as unseen
    k.view(12, page, 1, hd)[8] = -8.0
    cache = q8.PagedQ8Cache(q8.Q8Geometry(4, 1, hd, page, 12, 12, "int8"), 1)
    tables = torch.arange(12, **I32).view(1, 12)
    cache.append(k, v, tables, ints(0), cu_new=ints(0, n))
    q = torch.full((1, 4, hd), 0.7, dtype=torch.float16, device="cuda")
    got = cache.decode(q, ints(n), tables, out=torch.empty((1, 4, hd), device="cuda"))
    kk, vv = ref.held_values(cache, tables, 0, n)
    r = ref.attend(q, kk, vv, n)
    # the subnormal weights' part of the tolerance, against the values that weigh anything
    seen = (r["p"].amax((0, 1, 2)) > 2.0 ** -30)
    r["vmax"] = vv[:, seen].abs().amax()
    ref.assert_within(got, r["o"], ref.tolerance(r, hd, torch.float32))


def test_queries_out_of_fp16s_range(q8):
    """bf16 queries past fp16's largest and below its least; a row of zeros; NaN and infinity
    stay in their row."""
    lens = [300]
    cache, tables, seq = make(q8, 8, 2, 64, 32, "int8", lens, seed=12)
    gen = torch.Generator("cuda").manual_seed(8)
    q = randn(gen, 1, 8, 64, dtype=torch.bfloat16)
    factor = torch.tensor([1e8, 1e-8, 1.0, 1e-30, 0.0, 1e5, 1.0, 1.0], device="cuda")
    q = (q.float() * factor.view(1, 8, 1)).bfloat16()
    scale = torch.ones(8)
    got = cache.decode(q, seq, tables, scale=1e-7)
    check_attention(cache, tables, lens, q, [0, 1], got, scale=1e-7)
    clean = cache.decode(q, seq, tables, scale=1e-7)
    q[0, 2, 5] = float("nan")
    q[0, 6, 9] = float("inf")
    got = cache.decode(q, seq, tables, scale=1e-7)
    bad = got.isnan().any(-1)[0]
    assert bad.tolist() == [False, False, True, False, False, False, True, False]
    assert torch.equal(got[0, ~bad], clean[0, ~bad])
    del scale


@pytest.mark.parametrize("where", ["block", "tail"])
def test_nan_reaches_those_who_see_it(q8, where):
    page, hd = 16, 64
    n = 16 * 20 + 9
    gen = torch.Generator("cuda").manual_seed(21)
    k, v = randn(gen, n, 2, hd), randn(gen, n, 2, hd)
    at = 100 if where == "block" else n - 3
    v[at, 1, 7] = float("nan")
    cache = q8.PagedQ8Cache(q8.Q8Geometry(4, 2, hd, page, 32, 32, "e4m3"), 1)
    tables = torch.randperm(32, generator=gen, device="cuda").to(torch.int32).view(1, 32)
    cache.append(k, v, tables, ints(0), cu_new=ints(0, n))
    m = 40
    q = randn(gen, m, 4, hd)
    for call in (lambda **kw: cache.prefill(q, ints(0, m), m, ints(n), tables, **kw),
                 lambda **kw: cache.prefill(q[-12:], ints(0, 12), 12, ints(n), tables, **kw)):
        got = call()
        first = got.shape[0] - m
        pos = torch.arange(n - got.shape[0], n, device="cuda")
        sees = pos >= at if where == "tail" else torch.ones_like(pos, dtype=torch.bool)
        assert torch.equal(got[:, 2:].isnan().all(-1).all(-1), sees)
        assert not got[:, :2].isnan().any()
        if where == "block":  # behind the window: the block is not seen
            got = call(window=150, sinks=4)
            assert not got.isnan().any()
        del first


def test_pages_outside_the_pool_read_as_nan(q8):
    lens = [200, 200, 200]
    cache, tables, seq = make(q8, 4, 2, 64, 32, "int8", lens, seed=30)
    gen = torch.Generator("cuda").manual_seed(31)
    q = randn(gen, 3, 4, 64)
    clean = cache.decode(q, seq, tables)
    bad = tables.clone()
    bad[0, 2], bad[1, 5] = 1 << 30, -7
    got = cache.decode(q, seq, bad)
    assert got[:2].isnan().all() and torch.equal(got[2], clean[2])
    qq = randn(gen, 3 * 70, 4, 64)
    got = cache.prefill(qq, ints(0, 70, 140, 210), 70, seq, bad)
    # the second sequence's entry holds tokens 160 to 191: its queries from 130 to 159 see none
    assert got[:70].isnan().all() and not got[70:100].isnan().any()
    assert got[100:140].isnan().all() and not got[140:].isnan().any()
    k, _ = cache.read(ints(0, 0, 0), seq, bad, 600)
    assert k[64:96].isnan().all() and not k[400:].isnan().any()
    # behind the length they are not looked at
    short = cache.decode(q, ints(64, 160, 200), bad)
    assert not short.isnan().any()


# ---------------------------------------------------------------- prompts

@pytest.mark.parametrize("codes,dtype", [("int8", torch.float16), ("e4m3", torch.bfloat16)])
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("page", [16, 32, 64])
def test_prefill(q8, codes, dtype, heads, page):
    """Ragged prompts: some whole, some the ends of longer sequences, one without queries, one
    with more queries than tokens."""
    nh, nkv, hd = heads
    lens = [1, 0, 64, 130, 333, 700, 90, 5]
    m = [1, 0, 64, 130, 333, 41, 0, 9]
    cache, tables, seq = make(q8, nh, nkv, hd, page, codes, lens, seed=40)
    spoil(cache, tables, lens)
    cu = [0]
    for x in m:
        cu.append(cu[-1] + x)
    gen = torch.Generator("cuda").manual_seed(41)
    # Q as a slice of a wider projection, rows behind the last sequence
    wide = randn(gen, cu[-1] + 5, nh + 2, hd, dtype=dtype)
    q = wide[:, :nh]
    out = torch.full((cu[-1] + 5, nh, hd), 7.0, dtype=dtype, device="cuda")
    lse = torch.full((cu[-1] + 5, nh), 7.0, device="cuda")
    cache.prefill(q, ints(*cu), max(m), seq, tables, out=out, lse=lse)
    check_attention(cache, tables, lens, q, cu, out, lse)
    assert bool((out[cu[-1]:] == 7).all()) and bool((lse[cu[-1]:] == 7).all())


@pytest.mark.parametrize("window,sinks", [(1, 0), (7, 2), (64, 1), (100, 70), (333, 4), (9999, 3)])
@pytest.mark.parametrize("few", [False, True])
def test_prefill_window_and_sinks(q8, window, sinks, few):
    lens = [40, 1100, 450]
    m = [9, 9, 9] if few else [40, 300, 450]
    cache, tables, seq = make(q8, 12, 2, 64, 32, "int8", lens, seed=50)
    spoil(cache, tables, lens)
    cu = [0, m[0], m[0] + m[1], sum(m)]
    gen = torch.Generator("cuda").manual_seed(51)
    q = randn(gen, cu[-1], 12, 64)
    got = cache.prefill(q, ints(*cu), max(m), seq, tables, window=window, sinks=sinks)
    check_attention(cache, tables, lens, q, cu, got, window=window, sinks=sinks)


@pytest.mark.parametrize("codes", ["int8", "e4m3"])
@pytest.mark.parametrize("heads,m,n", [((40, 8, 128), 60, 9000), ((14, 2, 64), 300, 5003),
                                       ((8, 8, 128), 700, 2049), ((16, 1, 64), 70, 20001)])
def test_prefill_in_slices(q8, codes, heads, m, n):
    """Few row tiles over long contexts: several workgroups share a tile's tokens."""
    nh, nkv, hd = heads
    lens, ms = [n, 40, n // 3], [m, 40, 0]
    cache, tables, seq = make(q8, nh, nkv, hd, 32, codes, lens, seed=45)
    spoil(cache, tables, lens)
    size = q8.lib().jacq_q8_attend_workspace_size(cache.geo.ref, 3, m + 40, m, 0)
    assert size >= 2 * (m + 40) * nh * (hd + 2) * 4  # in slices indeed
    gen = torch.Generator("cuda").manual_seed(46)
    cu = [0, m, m + 40, m + 40]
    q = randn(gen, cu[-1] + 2, nh, hd, dtype=torch.bfloat16)
    for window, sinks in ((None, 0), (500, 3)):
        out = torch.full((cu[-1] + 2, nh, hd), 7.0, dtype=torch.bfloat16, device="cuda")
        lse = torch.full((cu[-1] + 2, nh), 7.0, device="cuda")
        cache.prefill(q, ints(*cu), m, seq, tables, window=window, sinks=sinks, out=out, lse=lse)
        check_attention(cache, tables, lens, q, cu, out, lse, window=window, sinks=sinks)
        assert bool((out[cu[-1]:] == 7).all()) and bool((lse[cu[-1]:] == 7).all())


@pytest.mark.parametrize("heads", [(4, 4, 64), (10, 2, 128), (16, 1, 64)])
@pytest.mark.parametrize("m", [2, 3, 4, 8, 13])
def test_few_queries(q8, heads, m):
    """The sizes at which the rows of a sequence fill one, two or more blocks of the decode
    kernel, or pass on to the prompts' kernel."""
    nh, nkv, hd = heads
    lens = [m, 40, 2000, 777, m + 1]
    cache, tables, seq = make(q8, nh, nkv, hd, 32, "e4m3", lens, seed=60 + m)
    spoil(cache, tables, lens)
    gen = torch.Generator("cuda").manual_seed(61)
    cu = [m * i for i in range(len(lens) + 1)]
    q = randn(gen, cu[-1], nh, hd)
    lse = torch.empty((cu[-1], nh), device="cuda")
    got = cache.prefill(q, ints(*cu), m, seq, tables, lse=lse)
    check_attention(cache, tables, lens, q, cu, got, lse)


def test_a_prompts_last_token_is_its_decode(q8):
    lens = [513, 1000]
    cache, tables, seq = make(q8, 8, 2, 128, 32, "int8", lens, seed=70)
    gen = torch.Generator("cuda").manual_seed(71)
    q = randn(gen, 1513, 8, 128)
    full = cache.prefill(q, ints(0, 513, 1513), 1000, seq, tables)
    one = cache.decode(q[[512, 1512]].contiguous(), seq, tables)
    # either is within its tolerance of the exact one
    for i, b in ((512, 0), (1512, 1)):
        k, v = ref.held_values(cache, tables, b, lens[b])
        r = ref.attend(q[i:i + 1], k, v, lens[b])
        ref.assert_within(full[i:i + 1] - one[b:b + 1].double(), torch.zeros_like(r["o"]),
                          2 * ref.tolerance(r, 128, torch.float16))


# ---------------------------------------------------------------- weights and eviction

@pytest.mark.parametrize("page", [16, 32, 64])
@pytest.mark.parametrize("m,window,sinks", [(1, None, 0), (1, 100, 5), (5, None, 0), (64, 200, 20)])
def test_block_weights(q8, page, m, window, sinks):
    lens = [m, 64, 100, 1003, 2500]
    cache, tables, seq = make(q8, 10, 2, 128, page, "int8", lens, seed=80)
    spoil(cache, tables, lens)
    gen = torch.Generator("cuda").manual_seed(81)
    cu = [m * i for i in range(len(lens) + 1)]
    q = randn(gen, cu[-1], 10, 128)
    w = torch.full((len(lens), cache.geo.max_pages_per_seq), float("nan"), device="cuda")

    def call(decay):
        if m == 1:
            return cache.decode(q, seq, tables, window=window, sinks=sinks, weights=w, decay=decay)
        return cache.prefill(q, ints(*cu), m, seq, tables, window=window, sinks=sinks, weights=w,
                             decay=decay)

    got = call(0.0)
    check_attention(cache, tables, lens, q, cu, got, weights=w, window=window, sinks=sinks)
    held = w.clone()
    call(0.5)
    check_attention(cache, tables, lens, q, cu, got, weights=w, window=window, sinks=sinks,
                    held=held, decay=0.5)
    w.copy_(held)
    call(1.0)
    assert torch.equal(w, held + held)


@pytest.mark.parametrize("page,width", [(16, 1), (16, 40), (32, 1500), (16, 5000), (64, 16384)])
@pytest.mark.parametrize("place", ["new", "same"])
def test_evict(q8, page, width, place):
    rng = random.Random(width)
    gen = torch.Generator("cuda").manual_seed(90)
    cap = page * width
    lens = [0, cap, cap - 1, cap // 2 + 1, max(0, cap - page), rng.randint(0, cap)]
    geo = q8.Q8Geometry(8, 2, 64, page, width, 4, "int8")
    cache = q8.PagedQ8Cache(geo, len(lens))
    w = torch.randn((len(lens), width), generator=gen, device="cuda").abs()
    w[torch.rand(w.shape, generator=gen, device="cuda") < 0.3] = 0.0
    w[1] = (w[1] * 4).round()  # many equal ones
    w[2, ::3] = float("nan")
    w[3] *= -1
    tables = torch.randint(0, 1 << 30, (len(lens), width), generator=gen, **I32)
    seq = ints(*lens)
    for keep, sink, recent in {(0, 0, 0), (1, 0, 1), (width // 2, 0, 0), (width // 2 + 1, 1, 0),
                               (max(2, width // 3), 1, 1), (width, 1, 0), (2 ** 31 - 1, 3, 9)}:
        want = ref.evict(w.cpu(), lens, tables.cpu(), page, keep, sink, recent)
        t, s, x = tables.clone(), seq.clone(), w.clone()
        out = None if place == "new" else (t, s, x, torch.empty_like(s))
        got = cache.evict(x, s, t, keep, sink_pages=sink, recent_pages=recent, out=out)
        for name, a, b in zip(("tables", "lengths", "weights", "evicted"), got, want):
            assert torch.equal(a.cpu().nan_to_num(-5.0) if a.is_floating_point() else a.cpu(),
                               b.nan_to_num(-5.0) if b.is_floating_point() else b), (name, keep)
        if place == "new":
            assert torch.equal(t, tables) and torch.equal(s, seq)


def test_serving_run(q8):
    """Prompts in, tokens out, with eviction whenever a sequence is long: the cache follows a
    plain record of the tokens that are left."""
    nh, nkv, hd, page, batch = 8, 2, 64, 16, 3
    gen = torch.Generator("cuda").manual_seed(100)
    width, pages = 40, 3 * 40
    geo = q8.Q8Geometry(nh, nkv, hd, page, width, pages, "int8")
    cache = q8.PagedQ8Cache(geo, batch)
    tables = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32).view(batch, width)
    tables = tables.contiguous()
    w = torch.zeros((batch, width), device="cuda")
    prompt = [37, 250, 401]
    kept = [[], [], []]  # (k, v) [NKV, HD] of the tokens left, fp16
    cu = [0, 37, 287, 688]
    k, v = randn(gen, 688, nkv, hd), randn(gen, 688, nkv, hd)
    for b in range(batch):
        kept[b] = [(k[i], v[i]) for i in range(cu[b], cu[b + 1])]
    lens = torch.zeros(batch, **I32)
    cache.append(k, v, tables, lens, cu_new=ints(*cu), max_new=401)
    lens = ints(*prompt)
    q = randn(gen, 688, nh, hd)
    o = cache.prefill(q, ints(*cu), 401, lens, tables)
    check_attention(cache, tables, prompt, q, cu, o)
    last = [q[cu[b + 1] - 20:cu[b + 1]] for b in range(batch)]
    cache.prefill(torch.cat(last), ints(0, 20, 40, 60), 20, lens, tables, weights=w, decay=0.0)
    for step in range(40):
        if step % 13 == 5:
            before = [n for n in lens.tolist()]
            host = w.cpu()
            tables, lens, w, gone = cache.evict(w, lens, tables, keep=14, sink_pages=1,
                                                recent_pages=2)
            for b, n in enumerate(before):
                if not int(gone[b]):
                    continue
                ids = torch.arange(width, dtype=torch.int32).view(1, -1)
                stay = ref.evict(host[b:b + 1], [n], ids, page, 14, 1, 2)[0][0, :14].tolist()
                kept[b] = [x for p in stay for x in kept[b][p * page:(p + 1) * page]] + \
                    kept[b][n // page * page:]
        k, v, q = (randn(gen, batch, h, hd) for h in (nkv, nkv, nh))
        cache.append(k, v, tables, lens)
        lens = lens + 1
        for b in range(batch):
            kept[b].append((k[b], v[b]))
        window, sinks = ((60, 4) if step % 3 == 0 else (None, 0))
        o = cache.decode(q, lens, tables, window=window, sinks=sinks, weights=w, decay=0.9)
        now = lens.tolist()
        assert now == [len(x) for x in kept]
        check_attention(cache, tables, now, q, [0, 1, 2, 3], o, window=window, sinks=sinks)
    # what the cache holds is what is left of the tokens, block by block
    for b, n in enumerate(lens.tolist()):
        for i, (code, scale, tail) in enumerate(((cache.k_code, cache.k_scale, cache.k_tail),
                                                 (cache.v_code, cache.v_scale, cache.v_tail))):
            x = torch.stack([t[i] for t in kept[b]])
            full = n // page
            y, s = ref.quantise(x[:full * page].view(full, page, nkv, hd).transpose(1, 2), "int8")
            at = tables[b, :full].long()
            got = code[at].transpose(2, 3) if i else code[at]
            assert torch.equal(got, ref.code_bytes(y, "int8"))
            assert torch.equal(scale[at], s.float())
            assert torch.equal(tail[b, :, :n - full * page], x[full * page:].transpose(0, 1))


# ---------------------------------------------------------------- streams, graphs, places

def test_graph_replays(q8):
    """A step (append, decode with weights, evict in place) captured once and replayed, against
    the eager calls on a twin; eager work in between."""
    nh, nkv, hd, page, batch, width = 10, 2, 128, 16, 5, 24
    gen = torch.Generator("cuda").manual_seed(110)

    def start():
        cache, tables, seq = make(q8, nh, nkv, hd, page, "e4m3", [300, 20, 15, 370, 160], seed=111,
                                  width=width, spare=5 * width)
        free = torch.arange(batch * width, **I32).view(batch, width) % cache.geo.num_pages
        return cache, torch.where(tables < 0, free, tables).contiguous(), seq, torch.zeros(
            (batch, width), device="cuda")

    a, b = start(), start()
    k, v, q = (torch.zeros((batch, h, hd), dtype=torch.float16, device="cuda")
               for h in (nkv, nkv, nh))
    outs = [torch.zeros((batch, nh, hd), dtype=torch.float16, device="cuda") for _ in range(2)]
    gone = torch.zeros(batch, **I32)

    def step(s, out):
        cache, tables, seq, w = s
        cache.append(k, v, tables, seq)
        seq.add_(1)
        cache.decode(q, seq, tables, weights=w, out=out)
        cache.evict(w, seq, tables, keep=20, sink_pages=1, recent_pages=1,
                    out=(tables, seq, w, gone))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # warm up on a third
        step(start(), outs[0])
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(a, outs[0])
    for i in range(40):
        for t in (k, v, q):
            t.copy_(randn(gen, *t.shape))
        graph.replay()
        step(b, outs[1])
        torch.cuda.synchronize()
        assert torch.equal(outs[0], outs[1]), i
        assert torch.equal(a[1], b[1]) and torch.equal(a[2], b[2]) and torch.equal(a[3], b[3])
    for x, y in zip(a[0].pool(), b[0].pool()):
        assert torch.equal(x, y)


def test_replays_of_a_prompt_in_slices(q8):
    """Captured once, replayed with other lengths, offsets and queries; the rows behind the last
    sequence, and queries past max_q, are left as they are."""
    lens, m = [9000, 4000, 300], 60
    cache, tables, seq = make(q8, 40, 8, 128, 32, "int8", lens, seed=125)
    gen = torch.Generator("cuda").manual_seed(126)
    q = randn(gen, 3 * m + 7, 40, 128)
    cu = ints(0, m, 2 * m, 3 * m)
    size = q8.lib().jacq_q8_attend_workspace_size(cache.geo.ref, 3, 3 * m + 7, m, 0)
    assert size > 0  # slices
    out = torch.full((3 * m + 7, 40, 128), 7.0, dtype=torch.float16, device="cuda")
    cache.prefill(q, cu, m, seq, tables, out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.prefill(q, cu, m, seq, tables, out=out)
    for now, at in ((lens, [0, m, 2 * m, 3 * m]), ([8000, 65, 300], [0, 10, 70, 71]),
                    ([0, 4000, 1], [5, 5, 66, 67]), (lens, [0, m + 4, m + 5, 3 * m])):
        q.copy_(randn(gen, *q.shape))
        seq.copy_(ints(*now))
        cu.copy_(ints(*at))
        out.fill_(7.0)
        graph.replay()
        want = torch.full_like(out, 7.0)
        cache.prefill(q, cu, m, seq, tables, out=want)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        assert bool((out[:at[0]] == 7.0).all()) and bool((out[at[3]:] == 7.0).all())
        for b in range(3):  # a query past max_q is left alone, and the others count from the end
            count = at[b + 1] - at[b]
            assert bool((out[at[b] + min(count, m):at[b + 1]] == 7.0).all())
            if count <= m and now[b]:
                rows = slice(at[b], at[b + 1])
                check_attention(cache.sequence_view(b), tables[b:b + 1], now[b:b + 1], q[rows],
                                [0, count], out[rows])


def test_calls_of_several_threads(q8):
    import threading
    lens = [3000, 5000]
    cache, tables, seq = make(q8, 8, 2, 128, 32, "int8", lens, seed=127)
    gen = torch.Generator("cuda").manual_seed(128)
    q = [randn(gen, 2, 8, 128) for _ in range(4)]
    want = [cache.decode(x, seq, tables) for x in q]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got = cache.decode(q[i], seq, tables)
                torch.cuda.current_stream().synchronize()
                if not torch.equal(got, want[i]):
                    bad.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_another_stream_and_a_shared_workspace(q8):
    lens = [4000, 9000]
    cache, tables, seq = make(q8, 8, 2, 128, 32, "int8", lens, seed=120)
    gen = torch.Generator("cuda").manual_seed(121)
    q = [randn(gen, 2, 8, 128) for _ in range(2)]
    want = [cache.decode(x, seq, tables) for x in q]
    size = q8.lib().jacq_q8_attend_workspace_size(cache.geo.ref, 2, 2, 1, 0)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    ws.random_(0, 255)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    graphs, outs = [], []
    for x in q:  # two graphs over one workspace, replayed one after another
        o = torch.empty_like(want[0])
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            cache.decode(x, seq, tables, out=o, workspace=ws)
        graphs.append(g)
        outs.append(o)
    for _ in range(3):
        for g, o, x in zip(graphs, outs, want):
            o.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(o, x)
    with torch.cuda.stream(side):
        got = cache.decode(q[0], seq, tables)
    side.synchronize()
    assert torch.equal(got, want[0])


def test_offsets_past_32_bits(q8):
    """Pages behind 4 GiB of codes."""
    nh, nkv, hd, page = 8, 8, 128, 64
    pages = (5 << 30) // (nkv * hd * page)
    geo = q8.Q8Geometry(nh, nkv, hd, page, 6, pages, "int8")
    t = {"k_code": torch.empty((pages, nkv, page, hd), dtype=torch.uint8, device="cuda"),
         "v_code": torch.empty((pages, nkv, hd, page), dtype=torch.uint8, device="cuda"),
         "k_scale": torch.zeros((pages, nkv), device="cuda"),
         "v_scale": torch.zeros((pages, nkv), device="cuda"),
         "k_tail": torch.zeros((1, nkv, page, hd), dtype=torch.float16, device="cuda")}
    t["v_tail"] = t["k_tail"].clone()
    cache = q8.PagedQ8Cache.from_tensors(geo, t)
    tables = ints(*(pages - 1 - 7 * i for i in range(6))).view(1, 6)
    gen = torch.Generator("cuda").manual_seed(130)
    n = 6 * 64 - 5
    k, v, q = randn(gen, n, nkv, hd), randn(gen, n, nkv, hd), randn(gen, n, nh, hd)
    cache.append(k, v, tables, ints(0), cu_new=ints(0, n))
    y, _ = ref.quantise(k[:64].transpose(0, 1), "int8")
    assert torch.equal(cache.k_code[pages - 1], ref.code_bytes(y, "int8"))
    got = cache.prefill(q, ints(0, n), n, ints(n), tables)
    check_attention(cache, tables, [n], q, [0, n], got)
    got = cache.decode(q[-1:], ints(n), tables)
    check_attention(cache, tables, [n], q[-1:], [0, 1], got)


def test_bounds_past_32_bits(q8):
    big = 1 << 33
    lens, gen = [70, 3], torch.Generator("cuda").manual_seed(0)
    cache, tables, n = make(q8, 4, 2, 64, 16, "int8", lens)
    other = q8.PagedQ8Cache(cache.geo, 2)
    k, v = randn(gen, 7, 2, 64), randn(gen, 7, 2, 64)
    for c in (cache, other):
        c.append(k, v, tables, torch.zeros_like(n), cu_new=ints(0, 5, 7),
                 max_new=big if c is cache else 5)
    assert torch.equal(cache.k_tail[0, :, :5], other.k_tail[0, :, :5])
    n, q = ints(5, 2), randn(gen, 7, 4, 64)
    assert torch.equal(cache.prefill(q, ints(0, 5, 7), big, n, tables, window=big, sinks=big),
                       other.prefill(q, ints(0, 5, 7), 5, n, tables))
    w = torch.ones(2, cache.geo.max_pages_per_seq, device="cuda")
    n = ints(*lens)
    got = cache.evict(w, n, tables, keep=2 * big, sink_pages=big, recent_pages=big)
    assert all(torch.equal(a, b) for a, b in zip(got, (tables, n, w, torch.zeros_like(n))))


def test_lengths_past_the_table_are_clamped(q8):
    cache, tables, _ = make(q8, 4, 2, 64, 16, "int8", [160, 160], seed=140)
    gen = torch.Generator("cuda").manual_seed(141)
    q = randn(gen, 2, 4, 64)
    got = cache.decode(q, ints(1 << 30, -9), tables)
    assert torch.equal(got[0], cache.decode(q, ints(160, 0), tables)[0])
    assert not got[1].any()


@pytest.mark.parametrize("seed", range(24))
def test_random_calls(q8, seed):
    """Any mix of lengths, queries, windows and heads: cut and uncut, few rows and many."""
    rng = random.Random(1000 + seed)
    nh, nkv, hd = rng.choice(HEADS)
    page, codes = rng.choice((16, 32, 64)), rng.choice(("int8", "e4m3"))
    dtype = rng.choice((torch.float16, torch.bfloat16))
    batch = rng.choice((1, 2, 5, 20, 70))
    most = rng.choice((40, 300, 3000, 12000)) // (1 if batch < 20 else 4)
    lens = [rng.randint(0, most) if rng.random() < 0.8 else rng.randint(0, 3) for _ in range(batch)]
    width = None if rng.random() < 0.5 else -(-max(lens + [1]) // page) + rng.choice((1, 500))
    cache, tables, seq = make(q8, nh, nkv, hd, page, codes, lens, seed=seed, dtype=dtype,
                              width=width)
    spoil(cache, tables, lens)
    gen = torch.Generator("cuda").manual_seed(seed)
    kw = {}
    if rng.random() < 0.5:
        kw = {"window": rng.randint(1, 2 * most), "sinks": rng.choice((0, 1, 5, 100))}
    for top in (1, rng.randint(2, 9), rng.randint(10, 200)):
        m = [min(n, rng.randint(0, top)) for n in lens] if top > 1 else [1] * batch
        cu = [0]
        for x in m:
            cu.append(cu[-1] + x)
        q = randn(gen, cu[-1], nh, hd, dtype=dtype, scale=1.5)
        lse = torch.zeros((cu[-1], nh), device="cuda")
        if top == 1:
            out = cache.decode(q, seq, tables, lse=lse, **kw)
        else:
            out = cache.prefill(q, ints(*cu), max(m + [1]), seq, tables, lse=lse, **kw)
        check_attention(cache, tables, lens, q, cu, out, lse, **kw)
        if top <= 9:
            w = torch.full((batch, cache.geo.max_pages_per_seq), 3.0, device="cuda")
            if top == 1:
                again = cache.decode(q, seq, tables, weights=w, decay=0.0, **kw)
            else:
                again = cache.prefill(q, ints(*cu), max(m + [1]), seq, tables, weights=w,
                                      decay=0.0, **kw)
            check_attention(cache, tables, lens, q, cu, again, weights=w, **kw)


def test_many_sequences(q8):
    rng = random.Random(3)
    lens = [rng.choice((0, 1, 30, 64, 200)) for _ in range(700)]
    cache, tables, seq = make(q8, 4, 1, 64, 16, "int8", lens, seed=150, width=100)
    gen = torch.Generator("cuda").manual_seed(151)
    q = randn(gen, 700, 4, 64)
    got = cache.decode(q, seq, tables)
    check_attention(cache, tables, lens, q, list(range(701)), got)


@pytest.mark.parametrize("batch,heads", [(65, (10, 2, 128)), (1100, (4, 2, 64)), (2500, (8, 1, 64))])
def test_many_sequences_under_a_wide_table(q8, batch, heads):
    """A cut that a kernel of its own plans: one round of 1024 sequences and more."""
    rng = random.Random(batch)
    lens = [rng.choice((0, 1, 30, 64, 200)) for _ in range(batch)]
    lens[batch // 2], lens[-1] = 9000, 3001
    cache, tables, seq = make(q8, *heads, 32, "int8", lens, seed=151)
    gen = torch.Generator("cuda").manual_seed(152)
    for m in (1, 2):
        cu = [0]
        for n in lens:
            cu.append(cu[-1] + min(n, m) if m > 1 else cu[-1] + 1)
        q = randn(gen, cu[-1], heads[0], heads[2])
        w = torch.ones((batch, cache.geo.max_pages_per_seq), device="cuda")
        for window, sinks in ((None, 0), (70, 5)):
            names = dict(window=window, sinks=sinks)
            got = (cache.decode(q, seq, tables, weights=w, decay=0.0, **names) if m == 1 else
                   cache.prefill(q, ints(*cu), m, seq, tables, weights=w, decay=0.0, **names))
            some = sorted(rng.sample(range(batch), 60) + [0, batch // 2, batch - 1])
            for b in some:
                rows = slice(cu[b], cu[b + 1])
                check_attention(cache.sequence_view(b), tables[b:b + 1], lens[b:b + 1], q[rows],
                                [0, cu[b + 1] - cu[b]], got[rows], weights=w[b:b + 1], **names)
