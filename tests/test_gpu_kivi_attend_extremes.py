"""Extremes of the int4 cache's attention of chunks, through both of its kernels: sequences without tokens
at a pass's end, queries and scales near the ends of their types, scores that are not finite,
values as large as fp16's."""
from __future__ import annotations

import ctypes
import random

import pytest

torch = pytest.importorskip("torch")

from tests import kivi_attend_ref as ref  # noqa: E402
from tests.test_gpu_kivi_attend import check, ints, is_prompt, kivi, make, offsets, randn  # noqa: E402,F401
from tests.test_gpu_kivi_attend_edges import SIZES, call  # noqa: E402

pytestmark = pytest.mark.gpu
POOL = ("k_code", "k_scale", "k_zero", "v_code", "v_scale", "v_zero")


@pytest.fixture
def pass_bytes(kivi):  # noqa: F811
    fn = kivi.lib().jacq_kivi_test_pass_bytes
    fn.argtypes, fn.restype = [ctypes.c_int64], None
    yield fn
    fn(0)


@pytest.mark.parametrize("batch,per_pass", [(6, 10), (6, 20), (6, 40), (70, 20), (70, 40)])
def test_sequences_without_tokens_at_the_end_of_a_pass(kivi, pass_bytes, batch, per_pass):  # noqa: F811
    """They have no tiles, so their place among the tiles is the next sequence's, or behind the last pass."""
    nh, nkv, hd, m = 40, 8, 128, 400
    lens = [640, 0, 640, 640, 640] + [0] * (batch - 5)
    cache, tables, seq = make(kivi, nh, nkv, hd, 32, 32, lens, seed=batch, width=608 // 32)
    cu = offsets([m] * 5 + [7] * (batch - 5))  # 7: more than what the kernel for few queries takes
    gen = torch.Generator("cuda").manual_seed(per_pass)
    q = randn(gen, cu[-1], nh, hd)
    pass_bytes(per_pass * 4 * 64 * hd * nkv)  # 10 tiles a sequence: the last pass is full
    assert is_prompt(kivi, cache, cu[-1], m)
    for causal in (True, False):
        out = torch.full((cu[-1], nh, hd), 7.0, dtype=torch.float16, device="cuda")
        lse = torch.full((cu[-1], nh), 7.0, device="cuda")
        (cache.prefill if causal else cache.cross)(q, ints(*cu), m, seq, tables, out=out, lse=lse)
        check(cache, tables, lens, q, cu, out, lse, causal=causal)
        for b, n in enumerate(lens):
            if n == 0:
                assert not out[cu[b]:cu[b + 1]].any(), f"sequence {b}"
                assert bool((lse[cu[b]:cu[b + 1]] == -torch.inf).all()), f"sequence {b}"


@pytest.mark.parametrize("heads,m,prompt", SIZES)
def test_subnormal_queries_and_scales(kivi, heads, m, prompt):  # noqa: F811
    """All scores are next to 0, so the output is a mean of the values that a query sees."""
    nh, nkv, hd = heads
    lens = [300, 222]
    cache, tables, seq, q, cu, most = call(kivi, *heads, 16, lens, m, prompt, seed=11)
    gen = torch.Generator("cuda").manual_seed(5)
    bits = torch.randint(1, 4, q.shape, generator=gen, device="cuda", dtype=torch.int16)  # x 2^-133
    bits[..., ::2] |= -2 ** 15  # negative ones
    tiny = bits.view(torch.bfloat16)
    one = torch.ones_like(tiny)
    for x, scale in ((tiny, 1 / 128), (tiny, 2.0 ** -60), (one, 1e-42), (one * 2.0 ** 100, 1e-42),
                     (q, 1e-42), (q.to(torch.bfloat16), 2.0 ** -149)):
        for window, sinks in ((None, 0), (40, 3)):
            got = cache.prefill(x, ints(*cu), most, seq, tables, window=window, sinks=sinks, scale=scale)
            check(cache, tables, lens, x, cu, got, None, window, sinks, scale=scale)
        got = cache.cross(x, ints(*cu), most, seq, tables, scale=scale)
        check(cache, tables, lens, x, cu, got, causal=False, scale=scale)


@pytest.mark.parametrize("heads,m,prompt", SIZES)
def test_keys_of_0_under_a_scale_beyond_fp32(kivi, heads, m, prompt):  # noqa: F811
    """The row's magnitude x the scale is no fp32 number, but the scores are 0."""
    lens = [60, 50]
    cache, tables, seq, q, cu, most = call(kivi, *heads, 16, lens, m, prompt, seed=14)
    x = q.to(torch.bfloat16) * 2.0 ** 100
    for b, n in enumerate(lens):
        cache.k_scr[b, :, :n] = 0.0
    got = cache.prefill(x, ints(*cu), most, seq, tables, scale=2.0 ** 60)
    check(cache, tables, lens, x, cu, got, scale=2.0 ** 60)


@pytest.mark.parametrize("heads,m,prompt", SIZES)
def test_rows_whose_scores_are_all_minus_infinity(kivi, heads, m, prompt):  # noqa: F811
    """0 / 0 by the definition, so NaN, with lse -inf; only a query that sees nothing gives 0."""
    nh, nkv, hd = heads
    lens = [3000, 300, 57, 1]  # cut into slices, whole
    cache, tables, seq, q, cu, most = call(kivi, *heads, 16, lens, m, prompt, seed=12)
    q[..., 5] = 1.0
    assert bool((seq[3] < most).all())  # queries of the last that see nothing
    last = [lens[0], 290, 50, 1]  # tokens of each, from the first on, whose keys have an infinity
    for b, n in enumerate(lens):
        old = ref.old_tokens(cache.geo, n)
        for t in range(0, min(old, last[b]), ref.GROUP):
            cache.k_zero[tables[b, t // 16].long(), :, 5] = -torch.inf
        cache.k_scr[b, :, :max(0, last[b] - old), 5] = -torch.inf
    for causal, window, sinks in ((True, None, 0), (True, 4, 0), (True, 4, 40), (False, None, 0)):
        lse = torch.empty(cu[-1], nh, device="cuda")
        if causal:
            got = cache.prefill(q, ints(*cu), most, seq, tables, window=window, sinks=sinks, lse=lse)
        else:
            got = cache.cross(q, ints(*cu), most, seq, tables, lse=lse)
        for b, n in enumerate(lens):
            what = f"sequence {b}, causal {causal}, window {window}, sinks {sinks}"
            lack = max(0, m - n) if causal else 0
            rows = slice(cu[b] + lack, cu[b + 1])
            assert not got[cu[b]:cu[b] + lack].any(), what
            assert bool((lse[cu[b]:cu[b] + lack] == -torch.inf).all()), what
            r = ref.attend(q[rows], *ref.held_values(cache, tables, b, n), window, sinks, causal)
            none = r["lse"] == -torch.inf
            assert bool(none.any()) if b in (0, 3) else bool((~none).any()), what
            want = torch.where(none[..., None], torch.nan, r["o"])
            r["size"] = torch.where(r["size"].isinf(), 30.0, r["size"])  # of the scores that are finite
            ref.assert_within(got[rows], want, ref.tolerance(r, hd, got.dtype), what)
            assert torch.equal(lse[rows] == -torch.inf, none), what


@pytest.mark.parametrize("heads,m,prompt", SIZES)
def test_a_mean_of_the_largest_values_is_finite(kivi, heads, m, prompt):  # noqa: F811
    """The weights of 30 tokens are rounded up by a 2^-11th, the first's not, so their sum is more than the
    rounded ones' is divided by; what it gives may not pass fp16, as no mean of fp16 values does."""
    nh, nkv, hd = heads
    for lens, groups in (([31], 0), ([31 + 2048], 64)):  # in the residual window; and behind groups that
        cache, tables, seq, q, cu, most = call(kivi, *heads, 16, lens, m, prompt, seed=13)  # weigh nothing
        old = ref.old_tokens(cache.geo, lens[0])
        if groups:
            for t in range(0, old, ref.GROUP):
                at = tables[0, t // 16].long()
                cache.k_scale[at], cache.k_zero[at] = 0.0, 0.0
                cache.k_zero[at, :, 1] = -30000.0
        left = lens[0] - old
        k = torch.zeros(nkv, left, hd, dtype=torch.float16, device="cuda")
        k[:, :-31, 1] = -30000.0
        k[:, -31, 0] = 1.0
        cache.k_scr[0, :, :left] = k
        q.zero_()
        q[..., :2] = 1.0
        # weights 2^7 and 2^6.00079 = 64.035, which rounds to 64.0625
        for sign in (1, -1):
            cache.v_scr[0, :, :left] = sign * 65504.0
            got = cache.cross(q, ints(*cu), most, seq, tables, scale=0.6926)
            assert bool((got == sign * 65504.0).all())
            got = cache.cross(q, ints(*cu), most, seq, tables, scale=0.6926,
                              out=torch.empty(q.shape, device="cuda"))
            assert bool(((got * sign - 65504.0).abs() <= 65504.0 * 2.0 ** -11).all())


def test_the_queries_of_one_head_may_lie_apart(kivi):  # noqa: F811
    cache, tables, seq, q, cu, most = call(kivi, 1, 1, 64, 16, [300, 77], 5, False, seed=15)
    wide = torch.full((cu[-1], 96), float("nan"), dtype=torch.float16, device="cuda")
    x = wide[:, None, :64]
    x.copy_(q)
    assert not x.is_contiguous()
    got = cache.prefill(x, ints(*cu), most, seq, tables)
    assert torch.equal(got, cache.prefill(q, ints(*cu), most, seq, tables))
    check(cache, tables, [300, 77], q, cu, got)


def test_a_chunk_beside_the_steps_of_many_sequences_under_a_wide_table(kivi, pass_bytes):  # noqa: F811
    """max_q for every sequence would be more workgroups than a launch takes, the tiles of the table's width
    more passes than pay for prompts alone."""
    nh, nkv, hd, batch, chunk = 32, 2, 64, 2048, 8200
    rng = random.Random(3)
    lens = [rng.choice((0, 1, 20, 33, 64, 90)) for _ in range(batch)]
    m = [rng.choice((0, 1, 1, 2, 3)) for _ in lens]
    lens[700], m[700] = 400, chunk  # most of them before the first token
    lens[1500], m[1500] = 700, 1
    cache, tables, seq = make(kivi, nh, nkv, hd, 16, 32, lens, seed=1, width=2048)
    cu = offsets(m)
    pass_bytes(1 << 28)
    assert is_prompt(kivi, cache, cu[-1], chunk)
    gen = torch.Generator("cuda").manual_seed(1)
    q = randn(gen, cu[-1], nh, hd)
    some = [b for b in range(batch) if b % 29 == 0 or b in (699, 700, 701, 1500, batch - 1)]
    for window, sinks in ((None, 0), (50, 3)):
        lse = torch.full((cu[-1], nh), 7.0, device="cuda")
        got = cache.prefill(q, ints(*cu), chunk, seq, tables, window=window, sinks=sinks, lse=lse)
        assert not bool((lse == 7.0).all(-1).any())  # every row is written
        for b in some:
            rows = slice(cu[b], cu[b + 1])
            part = kivi.PagedKiviCache.from_tensors(cache.geo, {
                **dict(zip(POOL, cache.pool()[:6])), "k_scr": cache.k_scr[b:b + 1],
                "v_scr": cache.v_scr[b:b + 1]})
            check(part, tables[b:b + 1], lens[b:b + 1], q[rows], [0, m[b]], got[rows], lse[rows], window,
                  sinks)
