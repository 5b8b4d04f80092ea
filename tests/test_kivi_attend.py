"""Refusals and host arithmetic of the int4 cache's attention of chunks and read-back, without a
GPU."""
from __future__ import annotations

import copy
import pickle

import pytest

torch = pytest.importorskip("torch")

from jacq_amd import kivi  # noqa: E402
from tests import kivi_attend_ref as ref  # noqa: E402

EINVAL, ENOMEM = 1, 3
GOOD = dict(num_heads=8, num_kv_heads=2, head_dim=64, page_size=16, residual=64,
            max_pages_per_seq=8, num_pages=16)
FIELDS = ("Q", "CU_Q", "SEQ_LENS", "BLOCK_TABLES", "O", "LSE", "q_stride", "q_dtype", "o_dtype",
          "batch", "total_q", "max_q", "window", "sinks", "causal", "scale")
ARGS = dict(zip(FIELDS, (0x10000, 0x20000, 0x30000, 0x40000, 0x50000, 0, 8 * 64, 0, 0, 2, 10, 5, 0, 0,
                         1, 0.125)))
POOL = tuple(0x100000 * (i + 1) for i in range(8))


def error(rc, code, text):
    assert rc == code and text in kivi.last_error(), (rc, kivi.last_error())


def attend(ws=0, ws_bytes=0, pool=POOL, geo=None, **kw):
    """Aligned host addresses that no call may reach: every call here is refused before it launches
    anything, or has nothing to launch."""
    g = kivi.KiviGeometry(**{**GOOD, **(geo or {})})
    args = kivi._ATTEND.pack(*{**ARGS, **kw}.values())
    return kivi.lib().jacq_kivi_attend(g.ref, kivi._POOL.pack(*pool), args, ws, ws_bytes, None)


@pytest.mark.parametrize("kw,text", [
    (dict(batch=-1), "batch"), (dict(batch=65536), "batch"), (dict(q_dtype=2), "fp16 or bf16"),
    (dict(o_dtype=1), "queries' type"), (dict(total_q=-1), "negative"), (dict(max_q=-1), "negative"),
    (dict(CU_Q=0), "one query"), (dict(window=-1), "negative"), (dict(sinks=-1), "negative"),
    (dict(causal=2), "causal"), (dict(causal=0, window=5), "no window"),
    (dict(causal=0, sinks=5), "no window"), (dict(scale=float("nan")), "finite"),
    (dict(scale=float("inf")), "finite"), (dict(scale=0.0), "positive"), (dict(scale=-0.5), "positive"),
    (dict(q_stride=500), "stride"), (dict(q_stride=516), "stride"), (dict(Q=0), "null"),
    (dict(O=0), "null"), (dict(SEQ_LENS=0), "null"), (dict(BLOCK_TABLES=0), "null"),
    (dict(Q=0x10008), "16-byte"), (dict(O=0x50008), "16-byte"), (dict(LSE=0x60002), "4-byte"),
    (dict(CU_Q=0x20001), "4-byte"), (dict(total_q=1 << 30, max_q=1 << 30), "too many")])
def test_attend_refusals(kw, text):
    error(attend(**kw), EINVAL, text)


@pytest.mark.parametrize("geo,text", [
    (dict(num_heads=9), "multiple"), (dict(num_heads=34), "<= 16"), (dict(head_dim=96), "head_dim"),
    (dict(page_size=64), "page_size"), (dict(residual=16), "residual"), (dict(num_pages=0), "num_pages"),
    (dict(max_pages_per_seq=-1), "max_pages"), (dict(max_pages_per_seq=1 << 20), "addresses")])
def test_geometries_are_the_caches(geo, text):
    error(attend(geo=geo), EINVAL, text)


def test_pools_are_checked():
    for i in range(8):
        error(attend(pool=POOL[:i] + (0,) + POOL[i + 1:]), EINVAL, "null")
        error(attend(pool=POOL[:i] + (POOL[i] + 8,) + POOL[i + 1:]), EINVAL, "16-byte")


def test_a_small_workspace_is_refused():
    geo = dict(max_pages_per_seq=1024)
    g = kivi.KiviGeometry(**{**GOOD, **geo})
    need = kivi.lib().jacq_kivi_attend_workspace_size(g.ref, 2, 10, 5)
    assert need > 0
    error(attend(geo=geo), ENOMEM, str(need))
    error(attend(ws=0x70000, ws_bytes=need - 1, geo=geo), ENOMEM, str(need))
    error(attend(ws=0x70008, ws_bytes=need, geo=geo), EINVAL, "16-byte")


def test_calls_with_nothing_to_do_launch_nothing():
    for kw in (dict(batch=0), dict(total_q=0), dict(max_q=0)):
        assert attend(Q=0, O=0, SEQ_LENS=0, BLOCK_TABLES=0, **kw) == 0
    assert kivi.lib().jacq_kivi_attend_workspace_size(kivi.KiviGeometry(**GOOD).ref, 0, 5, 5) == 0


def read(batch=2, total=10, dtype=0, starts=0x10000, ends=0x20000, tables=0x30000, k=0x40000,
         v=0x50000, pool=POOL, geo=None):
    g = kivi.KiviGeometry(**{**GOOD, **(geo or {})})
    return kivi.lib().jacq_kivi_read(g.ref, kivi._POOL.pack(*pool), starts, ends, tables, batch, total,
                                     k, v, dtype, None)


@pytest.mark.parametrize("kw,text", [
    (dict(batch=-1), "batch"), (dict(total=-1), "negative"), (dict(dtype=3), "fp16, bf16 or fp32"),
    (dict(dtype=-1), "fp16, bf16 or fp32"), (dict(starts=0), "null"), (dict(ends=0), "null"),
    (dict(tables=0), "null"), (dict(k=0), "null"), (dict(v=0), "null"), (dict(k=0x40008), "16-byte"),
    (dict(v=0x50008), "16-byte"), (dict(starts=0x10002), "4-byte"), (dict(ends=0x20001), "4-byte"),
    (dict(total=1 << 30), "too many"), (dict(geo=dict(head_dim=32)), "head_dim"),
    (dict(pool=(0,) * 8), "null")])
def test_read_refusals(kw, text):
    error(read(**kw), EINVAL, text)


def test_reads_of_nothing_launch_nothing():
    assert read(batch=0) == 0 and read(total=0, k=0, v=0) == 0


# ---- the Python surface ----

def cpu_cache():
    return kivi.PagedKiviCache(kivi.KiviGeometry(**GOOD), 2, device="cpu")


LENS = torch.tensor([5, 9], dtype=torch.int32)
TABLES = torch.zeros((2, 8), dtype=torch.int32)
CU = torch.tensor([0, 1, 3], dtype=torch.int32)


def q(tokens=3, dtype=torch.float16):
    return torch.zeros((tokens, 8, 64), dtype=dtype)


@pytest.mark.parametrize("kw,text", [
    (dict(q=torch.zeros(3, 7, 64)), "Q must be"), (dict(q=torch.zeros(3, 8 * 64)), "Q must be"),
    (dict(q=q(dtype=torch.float32)), "fp16 or bf16"),
    (dict(q=q().transpose(0, 1).contiguous().transpose(0, 1)), "side by side"),
    (dict(q=q(1).expand(3, 8, 64)), "one before"),
    (dict(seq_lens=LENS.long()), "int32"), (dict(seq_lens=LENS[:1]), "SEQ_LENS"),
    (dict(seq_lens=LENS.repeat_interleave(2)[::2]), "contiguous"),
    (dict(block_tables=TABLES[:, :7]), "BLOCK_TABLES"), (dict(block_tables=TABLES.long()), "int32"),
    (dict(cu_q=CU[:2]), "CU_Q"), (dict(cu_q=CU.long()), "int32"), (dict(cu_q=None), "per sequence"),
    (dict(cu_q=None, q=q(2), max_q=2), "MAX_Q"), (dict(max_q=-1), "MAX_Q"),
    (dict(scale=0.0), "SCALE"), (dict(scale=float("inf")), "SCALE"), (dict(scale=float("nan")), "SCALE"),
    (dict(out=torch.zeros(3, 8, 64, dtype=torch.bfloat16)), "O must be"),
    (dict(out=torch.zeros(2, 8, 64)), "O dim"), (dict(lse=torch.zeros(3, 7)), "LSE"),
    (dict(lse=torch.zeros(3, 8, dtype=torch.float16)), "LSE"),
    (dict(q=torch.zeros(3, 8, 64, dtype=torch.float16, device="meta")), "device"),
    (dict(), "GPU device")])
@pytest.mark.parametrize("call", ["prefill", "cross"])
def test_python_refusals(call, kw, text):
    args = {**dict(q=q(), cu_q=CU, max_q=2, seq_lens=LENS, block_tables=TABLES), **kw}
    with pytest.raises(kivi.KiviCheckError, match=text):
        getattr(cpu_cache(), call)(**args)


@pytest.mark.parametrize("kw,text", [(dict(window=0), "WINDOW"), (dict(window=-3), "WINDOW"),
                                     (dict(sinks=-1), "SINKS")])
def test_window_refusals(kw, text):
    with pytest.raises(kivi.KiviCheckError, match=text):
        cpu_cache().prefill(q(), CU, 2, LENS, TABLES, **kw)


@pytest.mark.parametrize("kw,text", [
    (dict(starts=LENS[:1]), "STARTS"), (dict(starts=LENS.long()), "int32"), (dict(total=-1), "TOTAL"),
    (dict(dtype=torch.float64), "fp16, bf16 or fp32"), (dict(ends=LENS.long()), "int32"),
    (dict(block_tables=TABLES[:1]), "BLOCK_TABLES"), (dict(), "GPU device")])
def test_python_read_refusals(kw, text):
    args = {**dict(starts=LENS * 0, ends=LENS, block_tables=TABLES, total=14), **kw}
    with pytest.raises(kivi.KiviCheckError, match=text):
        cpu_cache().read(**args)


POOL_ATTRS = ("k_code", "k_scale", "k_zero", "v_code", "v_scale", "v_zero", "k_scr", "v_scr")


def test_a_cache_of_other_tensors_than_its_geometrys_is_not_taken():
    for name in POOL_ATTRS:
        cache = cpu_cache()
        t = getattr(cache, name)
        cache._record()
        for other in (t[:-1], t.double(), torch.cat((t, t), -1)[..., :t.shape[-1]]):
            setattr(cache, name, other)
            with pytest.raises(kivi.KiviCheckError, match="must be contiguous"):
                cache.prefill(q(), CU, 2, LENS, TABLES)
        setattr(cache, name, t)
        cache._record()


def test_calls_take_the_tensors_that_a_cache_holds_now():
    cache = cpu_cache()

    def held(c):
        return kivi._POOL.unpack(c._record()[0])

    for name in POOL_ATTRS:
        held(cache)
        setattr(cache, name, getattr(cache, name).clone())
        assert held(cache) == tuple(t.data_ptr() for t in cache.pool())
        getattr(cache, name).data = getattr(cache, name).clone()
        assert held(cache) == tuple(t.data_ptr() for t in cache.pool())
    for make, shared in ((copy.copy, True), (copy.deepcopy, False),
                         (lambda c: pickle.loads(pickle.dumps(c)), False)):
        other = make(cache)
        assert other.geo == cache.geo and other.batch == 2
        assert held(other) == tuple(t.data_ptr() for t in other.pool())
        assert (held(other) == held(cache)) == shared
    assert held(cache.sequence_view(1))[6] == cache.k_scr[1].data_ptr()


@pytest.mark.parametrize("batch,total,most", [
    (65535, 2 ** 31 - 1, 2 ** 31 - 1), (65535, 2 ** 31 - 1, 10), (1, 2 ** 31 - 1, 2 ** 31 - 1),
    (65535, 100000, 50000), (300, 100000, 20000)])
def test_workspaces_of_the_largest_calls_have_a_size(batch, total, most):
    """Whether the call is refused or not: no product of its sizes passes 64 bits."""
    for heads in ((65536, 65536, 128), (65536, 4096, 128), (40, 8, 128), (16, 1, 64)):
        for pages in (0, 8000, 16000):
            geo = kivi.KiviGeometry(*heads, 16, 32, 32, pages, 100)
            size = kivi.lib().jacq_kivi_attend_workspace_size(geo.ref, batch, total, most)
            # parts of 1 GiB, the tiles of a pass of 2 GiB and, behind it, of a sequence's end
            assert size <= 2 ** 32 + 4096 * 64 * heads[2] * 4 * heads[1]


# ---- the reference itself ----

def test_the_reference_is_the_caches_definition():
    """Against the loops of the definition, on a small cache."""
    geo = kivi.KiviGeometry(**{**GOOD, "residual": 32})
    gen = torch.Generator().manual_seed(0)
    cache = kivi.PagedKiviCache(geo, 1, device="cpu")
    for t in cache.pool():
        t.copy_(torch.randint(0, 256, t.shape, generator=gen) if t.dtype == torch.uint8
                else torch.randn(t.shape, generator=gen))
    tables = torch.randperm(16, generator=gen)[:8].to(torch.int32)[None]
    n, page, hd = 75, 16, 64
    k, v, there = ref.exact_values(cache, tables, 0, n)
    assert bool(there.all()) and k.shape == v.shape == (2, n, hd)
    for t in (0, 15, 16, 31, 32, 63 - 32, 40, 74):
        for h in range(2):
            for d in (0, 1, 33, 63):
                if t >= 32:
                    want = cache.k_scr[0, h, t - 32, d], cache.v_scr[0, h, t - 32, d]
                else:
                    p, first = int(tables[0, t // page]), int(tables[0, t // 32 * 32 // page])
                    ck, cv = (int(x[p, h, t % page, d // 2]) >> 4 * (d % 2) & 15
                              for x in (cache.k_code, cache.v_code))
                    want = (ck * cache.k_scale[first, h, d].double() + cache.k_zero[first, h, d].double(),
                            cv * cache.v_scale[p, h, t % page, d // 32].double()
                            + cache.v_zero[p, h, t % page, d // 32].double())
                assert float(k[h, t, d]) == float(want[0]) and float(v[h, t, d]) == float(want[1])
    q = torch.randn((5, 8, hd), generator=gen)
    for causal, window, sinks in ((True, None, 0), (True, 9, 2), (False, None, 0)):
        r = ref.attend(q, k, v, window, sinks, causal)
        for i in range(5):
            for head in (0, 3, 7):
                pos = n - 5 + i
                seen = [j for j in range(n) if not causal or (j <= pos and (
                    window is None or j < sinks or j > pos - window))]
                x = (k[head // 4, seen] @ q[i, head].double()) / 8
                o = torch.softmax(x, 0) @ v[head // 4, seen]
                assert float((o - r["o"][i, head]).abs().max()) < 1e-12
                assert abs(float(torch.logsumexp(x, 0) - r["lse"][i, head])) < 1e-12
