"""Chunks of queries, cross attention and read-back over the int4 cache on the GPU, against their
definition in 64 bits (tests/kivi_attend_ref.py)."""
from __future__ import annotations

import random

import pytest

torch = pytest.importorskip("torch")

from tests import kivi_attend_ref as ref  # noqa: E402

pytestmark = pytest.mark.gpu
I32 = {"dtype": torch.int32, "device": "cuda"}


@pytest.fixture(scope="module")
def kivi():
    from jacq_amd import kivi as m
    assert torch.cuda.is_available(), "GPU tests need a GPU"
    m.lib()
    return m


def ints(*x):
    return torch.tensor(x, **I32)


def randn(gen, *shape, dtype=torch.float16):
    return torch.randn(shape, generator=gen, device="cuda").to(dtype)


def offsets(m):
    cu = [0]
    for x in m:
        cu.append(cu[-1] + x)
    return cu


def make(kivi, nh, nkv, hd, page, residual, lens, seed=0, spare=3, width=None):
    """A cache whose sequences hold `lens` random tokens, written by its own append, in shuffled
    pages.  What no token of a sequence is in holds NaN, infinities and stray codes."""
    gen = torch.Generator("cuda").manual_seed(seed)
    per = ref.GROUP // page
    old = [max(0, n - residual) // ref.GROUP for n in lens]
    need = [n * per for n in old]
    # a table has to address all but the residual window, a begun group of it too
    width = max([per, *(-(-max(0, n - residual) // ref.GROUP) * per for n in lens)]) \
        if width is None else width
    pages = sum(need) + spare
    perm = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    tables = torch.full((len(lens), width), -1, **I32)
    at = 0
    for b, k in enumerate(need):
        tables[b, :k] = perm[at:at + k]
        at += k
    geo = kivi.KiviGeometry(nh, nkv, hd, page, ref.GROUP, residual, width, pages)
    cache = kivi.PagedKiviCache(geo, len(lens))
    for t in (cache.k_scale, cache.v_scale, cache.k_scr):
        t.fill_(float("nan"))
    for t in (cache.k_zero, cache.v_zero, cache.v_scr):
        t.fill_(float("inf"))
    cache.k_code.fill_(0x7F)
    cache.v_code.fill_(0xFF)
    for b, n in enumerate(lens):
        if n:
            k = randn(gen, 1, n, nkv, hd)
            k[..., 3] *= 5
            cache.sequence_view(b).append(k, randn(gen, 1, n, nkv, hd), tables[b:b + 1],
                                          torch.zeros(1, **I32))
            left = n - ref.old_tokens(geo, n)
            cache.k_scr[b, :, left:] = float("nan")
            cache.v_scr[b, :, left:] = float("inf")
    return cache, tables, ints(*lens)


def check(cache, tables, lens, q, cu, got, lse=None, window=None, sinks=0, causal=True, scale=None):
    """Every sequence's rows of `got` against the reference over what the cache holds."""
    for b, n in enumerate(lens):
        rows = slice(cu[b], cu[b + 1])
        m = cu[b + 1] - cu[b]
        if m == 0:
            continue
        k, v = ref.held_values(cache, tables, b, n)
        lack = max(0, m - n) if causal else 0  # queries before the first token see nothing
        what = (f"sequence {b} of {n} tokens, {m} queries, window {window}, sinks {sinks}, "
                f"causal {causal}")
        assert not got[rows][:lack].any(), what
        r = ref.attend(q[rows][lack:], k, v, window, sinks, causal, scale)
        hd = cache.geo.head_dim
        ref.assert_within(got[rows][lack:], r["o"], ref.tolerance(r, hd, got.dtype), what)
        if lse is not None:
            assert bool((lse[rows][:lack] == -torch.inf).all()), what
            ref.assert_within(lse[rows][lack:], r["lse"], ref.score_error(r, hd) + 2.0 ** -22
                              * (1 + r["lse"].abs().nan_to_num(posinf=0)), what + " lse")


HEADS = [(32, 4, 64), (14, 2, 64), (40, 8, 128), (5, 1, 128), (16, 1, 64), (3, 3, 128)]
LENS = [1, 31, 32, 33, 64, 95, 128, 160, 161, 250, 333, 700]


@pytest.mark.parametrize("page", [16, 32])
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_a_query_or_a_few_of_every_sequence(kivi, heads, page, dtype):
    rng = random.Random(heads[0] * page)
    nh, nkv, hd = heads
    for residual in (32, 128):
        cache, tables, seq = make(kivi, nh, nkv, hd, page, residual, [0, *LENS], seed=page)
        lens = [0, *LENS]
        gen = torch.Generator("cuda").manual_seed(residual)
        for m in ([1] * len(lens), [rng.randint(0, 7) for _ in lens], [3] * len(lens)):
            cu = offsets(m)
            q = randn(gen, cu[-1], nh, hd, dtype=dtype)
            for window, sinks in ((None, 0), (40, 0), (7, 3), (100, 33)):
                lse = torch.empty(cu[-1], nh, device="cuda")
                got = cache.prefill(q, ints(*cu), max(m), seq, tables, window=window, sinks=sinks,
                                    lse=lse)
                assert got.dtype == dtype
                check(cache, tables, lens, q, cu, got, lse, window, sinks)
            got = cache.cross(q, ints(*cu), max(m), seq, tables, out=torch.empty(
                cu[-1], nh, hd, device="cuda"))
            check(cache, tables, lens, q, cu, got, causal=False)


def is_prompt(kivi, cache, total, max_q):
    """Whether the prompts' kernel runs a call, not the one for few queries."""
    return bool(kivi.lib().jacq_kivi_test_is_prompt(cache.geo.ref, cache.batch, total, max_q))


@pytest.mark.parametrize("heads", [(14, 2, 64), (40, 8, 128), (4, 4, 64), (8, 1, 128)])
@pytest.mark.parametrize("page", [16, 32])
@pytest.mark.parametrize("prompt", [False, True])
def test_prompts_and_chunks(kivi, heads, page, prompt):
    """Under a wide table these are prompts; under a narrow one of a few heads' they are not."""
    nh, nkv, hd = heads
    lens = [0, 1, 70, 333, 700, 1500]
    width = 262080 // page if prompt else None
    cache, tables, seq = make(kivi, nh, nkv, hd, page, 64, lens, seed=hd, width=width)
    assert is_prompt(kivi, cache, sum(lens), 1500) == (prompt or nh > 8)
    gen = torch.Generator("cuda").manual_seed(page)
    for m in (lens, [0, 0, 0, 0, 0, 1500], [1, 1, 65, 200, 128, 513], [2, 130, 1, 0, 700, 64]):
        cu = offsets(m)
        q = randn(gen, cu[-1], nh, hd)
        for window, sinks in ((None, 0), (150, 5), (33, 0)):
            lse = torch.empty(cu[-1], nh, device="cuda")
            got = cache.prefill(q, ints(*cu), max(m), seq, tables, window=window, sinks=sinks,
                                lse=lse)
            check(cache, tables, lens, q, cu, got, lse, window, sinks)
        lse = torch.empty(cu[-1], nh, device="cuda")
        got = cache.cross(q, ints(*cu), max(m), seq, tables, lse=lse)
        check(cache, tables, lens, q, cu, got, lse, causal=False)


@pytest.mark.parametrize("page", [16, 32])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads", [(14, 2, 64), (40, 8, 128), (3, 3, 64), (1, 1, 128)])
def test_read_back_is_the_definition_rounded_once(kivi, heads, page, dtype):
    nh, nkv, hd = heads
    lens = [0, 1, 31, 64, 65, 160, 333, 700]
    cache, tables, seq = make(kivi, nh, nkv, hd, page, 64, lens, seed=hd + page)
    for starts in ([0] * 8, [0, 1, 30, 64, 33, 17, 100, 699], [0, 0, 31, 1, 64, 159, 330, 31]):
        total = sum(n - s for n, s in zip(lens, starts))
        for most in (total, total + 5, max(0, total - 40)):
            k, v = cache.read(ints(*starts), seq, tables, most, dtype=dtype)
            assert k.shape == v.shape == (most, nkv, hd) and k.dtype == dtype
            at = 0
            for b, n in enumerate(lens):
                want_k, want_v, _ = ref.exact_values(cache, tables, b, n)
                for got, want in ((k, want_k), (v, want_v)):
                    want = want[:, starts[b]:].transpose(0, 1)
                    part = got[at:at + n - starts[b]]
                    want = want[:part.shape[0]]
                    if dtype == torch.float16:
                        assert torch.equal(part, ref.to_half(want))
                    else:  # bf16: of the fp32 sum
                        step = ref.HALF_STEP[dtype] * (1 + 2.0 ** -14)
                        assert bool(((part.double() - want).abs() <= step * want.abs()).all())
                at += n - starts[b]
